"""Draws from exponentiated returns against the definition in 64 bits (oracle/ref_learn.py).

An index has to be the oracle's: the numbers u are random, and the chance that one lies within the kernels' rounding
(below 2^-40 of the mass) of a border between two samples is below 1e-7 over all of these tests.  A weight is rounded to
float32 once (2^-24 relative); the fp64 exponentials behind it are good to 1e-13 at the largest distance that can be drawn
(kappa (Rmax - R) < 44, times 2^-53, a few of them)."""
import numpy as np
import pytest

from oracle import ref_learn

pytestmark = pytest.mark.gpu

TYPES = ["float64", "float32", "float16", "bfloat16"]
WEIGHT_RTOL = 2.0 ** -24 * (1 + 1e-5) + 1e-13

FILTERS = [
    dict(),
    dict(top_k=1),
    dict(top_k=7),
    dict(top_p=0.5),
    dict(min_p=0.3),
    dict(top_k=40, top_p=0.9, min_p=0.02),
    dict(top_k=1 << 20, top_p=0.999, min_p=1e-6),
]


def _draw(R, u, **kw):
    from trajopt_amd.device import draw_from_returns
    return draw_from_returns(R, u, **kw)


def _check(R, u, kappa=1.0, top_k=0, top_p=1.0, min_p=0.0, got=None):
    """R, u: CUDA tensors (rows, K), (rows, D); parameters numbers or CUDA tensors."""
    index, weight = got if got is not None else _draw(R, u, kappa=kappa, top_k=top_k, top_p=top_p, min_p=min_p)
    assert index.shape == weight.shape == u.shape and str(index.dtype) == "torch.int64" and str(weight.dtype) == "torch.float32"
    Rn, un = R.double().cpu().numpy(), u.double().cpu().numpy()
    index, weight = index.cpu().numpy(), weight.cpu().numpy()
    one = lambda v, b: v.cpu().numpy()[b] if hasattr(v, "cpu") else v  # noqa: E731
    for b in range(Rn.shape[0]):
        i, w = ref_learn.draw(Rn[b], un[b], one(kappa, b), one(top_k, b), one(top_p, b), one(min_p, b))
        assert np.array_equal(index[b], i), (b, np.flatnonzero(index[b] != i)[:5], index[b][index[b] != i][:5], i[index[b] != i][:5])
        assert np.all(np.abs(weight[b] - w) <= WEIGHT_RTOL * w + 1e-45), (b, np.abs(weight[b] - w).max())


def _returns(rows, K, dtype, seed, spread=2.0, masked=0.0):
    import torch
    rng = np.random.RandomState(seed)
    R = torch.tensor(-20.0 + spread * rng.normal(size=(rows, K)), device="cuda").to(getattr(torch, dtype))
    if masked:
        bad = torch.tensor([np.nan, -np.inf, np.inf, 0.0], dtype=R.dtype, device="cuda")
        bad[3] = torch.finfo(R.dtype).min
        at = torch.tensor(rng.uniform(size=(rows, K)) < masked, device="cuda")
        R = torch.where(at, bad[torch.tensor(rng.randint(0, 4, size=(rows, K)), device="cuda")], R)
    return R


def _numbers(rows, D, seed):
    import torch
    return torch.tensor(np.random.RandomState(1000 + seed).uniform(size=(rows, D)), device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("f", range(len(FILTERS)))
@pytest.mark.parametrize("rows,K,D", [(1, 1, 1), (3, 2, 3), (5, 63, 2), (1, 64, 9), (4, 65, 1), (2, 511, 70), (2, 513, 3), (1, 4099, 20)])
def test_draws(dtype, f, rows, K, D):
    R, u = _returns(rows, K, dtype, K + f), _numbers(rows, D, K)
    _check(R, u, kappa=1.5, **FILTERS[f])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,K", [(2, 255), (2, 257), (2, 1023), (2, 1025), (2, 2047), (2, 2049), (3, 4097), (2, 8191), (2, 8193), (2, 16383),
                                    (2, 16385), (1, 32769), (2, 65535), (1, 65537), (1, 131071), (1, 524291)])
def test_long_rows(dtype, rows, K):
    R = _returns(rows, K, dtype, K, masked=0.05)
    _check(R, _numbers(rows, 5, K), kappa=0.7, top_k=K // 3, top_p=0.8)
    _check(R, _numbers(rows, 33, K), kappa=1.1, top_p=0.97, min_p=1e-4)
    _check(R, _numbers(rows, 2, K), kappa=3.0, top_k=50)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kappa", [0.0, 1e-3, 25.0, 300.0, 1e6])
def test_temperatures(dtype, kappa):
    """From uniform (kappa 0) to the best sample alone."""
    for K in (50, 3000, 40000):
        R, u = _returns(2, K, dtype, K), _numbers(2, 11, K)
        _check(R, u, kappa=kappa)
        _check(R, u, kappa=kappa, top_k=K // 2, top_p=0.6)
        _check(R, u, kappa=kappa, min_p=0.2, top_p=0.9)


@pytest.mark.parametrize("K", [10, 700, 5000, 70000])
@pytest.mark.parametrize("levels", [1, 2, 5])
def test_ties_go_to_the_lowest_index(K, levels):
    """Few different returns: every border lies among equal samples."""
    import torch
    rng = np.random.RandomState(K + levels)
    R = torch.tensor(rng.randint(0, levels, size=(2, K)).astype(np.float32) * 0.25, device="cuda")
    if levels > 1:
        R = torch.where(R == 0, torch.tensor([0.0, -0.0], device="cuda").repeat(K)[:K], R)      # both zeros are one value
    u = _numbers(2, 17, K)
    for f in (dict(top_k=K // 2), dict(top_k=3), dict(top_p=0.37), dict(top_p=0.9, top_k=(2 * K) // 3), dict(min_p=0.9), dict(min_p=1.0)):
        _check(R, u, kappa=2.0, **f)
    half = R.to(torch.bfloat16)
    _check(half, u, kappa=0.0, top_k=K // 3, top_p=0.5)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_a_mask_empties(dtype):
    import torch
    for K in (5, 600, 9000, 66000):
        R = _returns(6, K, dtype, K, masked=0.3)
        R[0] = float("nan")
        R[1] = -float("inf")
        R[2] = torch.finfo(R.dtype).min                     # finite: every sample weighs the same
        R[3] = float("-inf")
        R[3, K - 1] = -3.0                                   # one sample left
        R[4] = torch.finfo(R.dtype).min
        R[4, K // 2] = 1.0
        u = _numbers(6, 4, K)
        for f in (dict(), dict(top_k=3), dict(top_p=0.5), dict(top_k=5, top_p=0.9, min_p=0.1)):
            _check(R, u, kappa=1.0, **f)
        index, weight = _draw(R, u)
        assert (index[:2] == -1).all() and (weight[:2] == 0).all() and (index[3] == K - 1).all() and (index[4] == K // 2).all()


def test_range_of_the_type():
    """Returns as far apart as the type allows, and neighbours one rounding apart."""
    import torch
    for dtype in (torch.float64, torch.float32):
        big = torch.finfo(dtype).max
        R = torch.tensor([[-big, big, 0.0, big, -big, 1.0, torch.finfo(dtype).tiny / 4]], dtype=dtype, device="cuda")
        u = torch.linspace(0, 0.99, 23, dtype=torch.float64, device="cuda").reshape(1, -1)
        for f in (dict(), dict(top_k=1), dict(top_k=3), dict(top_p=0.5)):
            _check(R, u, kappa=1.0, **f)
            _check(R / 4, u, kappa=0.0, **f)
        one = torch.ones(1, 1000, dtype=dtype, device="cuda")
        eps = torch.finfo(dtype).eps
        close = one + eps * torch.arange(1000, device="cuda", dtype=dtype)[torch.randperm(1000, generator=torch.Generator().manual_seed(1)).cuda()]
        for K in (1000, 64000):
            _check(close.repeat(1, K // 1000), u, kappa=1.0, top_k=K // 3 + 1, top_p=0.7)


@pytest.mark.parametrize("dtype", ["float64", "float32"])
@pytest.mark.parametrize("K", [200, 1000, 9000, 17000, 70000])
def test_ranges_that_overflow(K, dtype):
    """Both ends of the type in one row (their distance is infinite, the bins' quotient zero), ranges so small that the quotient is
    infinite, and rows whose lowest values a look at every fourth sample misses."""
    import torch
    t = getattr(torch, dtype)
    rng = np.random.RandomState(K)
    big, small = torch.finfo(t).max, torch.finfo(t).tiny * torch.finfo(t).eps
    u = _numbers(3, 7, K)
    filters = (dict(), dict(top_k=K // 3), dict(top_p=0.6), dict(top_k=K // 2, top_p=0.7), dict(top_k=20))
    ends = torch.tensor(rng.choice([-big, -big / 2, 0.0, big / 3, big], size=(3, K)), device="cuda", dtype=t)
    for f in filters:
        _check(ends, u, kappa=0.0, **f)
    denormal = torch.tensor(rng.randint(0, 5, size=(3, K)) * small, device="cuda", dtype=t)
    for f in filters:
        _check(denormal, u, kappa=0.3, **f)
    low = _returns(3, K, dtype, K)
    at = torch.arange(K, device="cuda")
    low = torch.where((at % 4 != 0) & (at % 5 == 1), torch.full_like(low, -big / 4), low)
    for f in filters + (dict(top_k=K - 3), dict(top_p=0.999)):
        _check(low, u, kappa=0.0, **f)
        _check(low, u, kappa=0.9, **f)


@pytest.mark.parametrize("K", [7, 64, 300, 1000, 9000, 17000, 70000])
@pytest.mark.parametrize("kappa", [3e-308, 1e-308, 5e-309, 1e-310])
def test_distances_beyond_the_range_of_fp64(K, kappa):
    """Returns whose distance fp64 does not hold, at temperatures that tell them apart all the same; against 80-bit numbers."""
    import torch
    rng = np.random.RandomState(K)
    big = np.finfo(np.float64).max
    R = rng.uniform(-1.0, 1.0, size=K) * big
    R[rng.randint(K)] = big
    R[0] = -big
    u = rng.uniform(size=33)
    for top_k, min_p in ((0, 0.0), (K // 2 + 1, 0.0), (0, 0.2)):
        x = R.astype(np.longdouble)
        w = np.exp(-np.longdouble(kappa) * (x.max() - x))
        if top_k:
            w[np.argsort(-R, kind="stable")[top_k:]] = 0
        w[w < min_p] = 0
        upto = np.cumsum(w)
        want = np.searchsorted(upto, u.astype(np.longdouble) * upto[-1], side="right")
        index, weight = _draw(torch.tensor(R[None], device="cuda"), torch.tensor(u[None], device="cuda"), kappa=kappa, top_k=top_k, min_p=min_p)
        assert np.array_equal(index.cpu().numpy()[0], want), (top_k, min_p)
        share = (w[want] / upto[-1]).astype(np.float64)
        assert np.all(np.abs(weight.cpu().numpy()[0] - share) <= WEIGHT_RTOL * share)


def test_numbers_at_the_ends():
    import torch
    for K in (40, 5000, 80000):
        R = _returns(1, K, "float32", K)
        R[0, 0] = -1000.0                                    # weighs nothing: u = 0 must not pick it
        R[0, K - 1] = float("-inf")
        u = torch.tensor([[0.0, 1 - 2.0 ** -53, 1.0, 2.0, -1.0, float("nan"), float("inf"), -float("inf")]], dtype=torch.float64, device="cuda")
        index, weight = _draw(R, u, kappa=2.0, top_p=0.99)
        w = ref_learn.kept_weights(R[0].double().cpu().numpy(), 2.0, 0, 0.99)
        first, last = np.flatnonzero(w * 2.0 ** 40 > 1)[[0, -1]]
        assert index.cpu().tolist()[0] == [first, last, last, last, first, first, last, first]


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dtype):
    import torch
    for rows, K in ((3, 50), (4, 3001), (2, 20000), (2, 70001)):
        u = _numbers(rows, 6, K)
        wide = _returns(rows, K + 7, dtype, K)
        _check(wide[:, 3:K + 3], u, kappa=1.0, top_k=20, top_p=0.9)           # rows at every alignment
        tall = _returns(K, rows, dtype, K)
        _check(tall.t(), u, kappa=1.0, top_p=0.8)                              # samples a row apart
        _check(wide[:, ::2][:, :K // 2], u, kappa=1.0, min_p=0.05)
        _check(wide[:1, :K].expand(rows, K), u, kappa=1.0, top_p=0.8)          # one row for all
    R, u = _returns(1, 999, dtype, 5), _numbers(1, 3, 5)
    index, weight = _draw(R[0], u[0], kappa=0.5)
    assert index.shape == (3,)
    _check(R, u, kappa=0.5, got=(index[None], weight[None]))
    index, weight = _draw(R, u.float(), kappa=0.5)
    _check(R, u.float().double(), kappa=0.5, got=(index, weight))


@pytest.mark.parametrize("K", [30, 500, 6000, 70000])
def test_parameters_per_row(K):
    import torch
    rows = 12
    rng = np.random.RandomState(K)
    R, u = _returns(rows, K, "float32", K, masked=0.02), _numbers(rows, 5, K)
    kappa = torch.tensor(np.exp(rng.uniform(-2, 3, rows)), device="cuda")
    top_k = torch.tensor(rng.randint(0, K, rows), device="cuda")
    top_p = torch.tensor(rng.uniform(0.05, 1.0, rows), device="cuda")
    min_p = torch.tensor(rng.uniform(0.0, 0.2, rows), device="cuda")
    top_p[3] = 1.0
    top_k[4] = 0
    top_k[5] = K + 100
    _check(R, u, kappa=kappa, top_k=top_k, top_p=top_p, min_p=min_p)
    _check(R, u, kappa=kappa, top_k=5, top_p=top_p, min_p=0.0)
    # values no call could pass as numbers leave their row without samples (a negative top_k: with all)
    kappa[0], kappa[1], kappa[2] = -1.0, float("nan"), float("inf")
    top_p[6], top_p[7], min_p[8], min_p[9], top_k[10] = 0.0, float("nan"), 1.5, float("nan"), -3
    index, _ = _draw(R, u, kappa=kappa, top_k=top_k, top_p=top_p, min_p=min_p)
    assert (index[[0, 1, 2, 6, 7, 8, 9]] == -1).all() and (index[[3, 4, 5, 10, 11]] >= 0).all()
    index32, _ = _draw(R, u, kappa=kappa.float().double(), top_k=top_k.int(), top_p=top_p, min_p=min_p)
    assert index32.shape == index.shape


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float64"])
@pytest.mark.parametrize("K", [30, 500, 6000, 20000, 70000])
def test_parameters_per_row_outside_their_range(K, dtype):
    """Every parameter alone, on either side of its range: its row has no samples (a negative top_k: all), the rows beside it
    are drawn from as ever."""
    import torch
    inf, nan = float("inf"), float("nan")
    bad = [("kappa", v) for v in (-1.0, -inf, inf, nan)] + [("top_p", v) for v in (1.5, inf, 1.0 + 2.0 ** -52, 0.0, -0.5, -inf, nan)] + \
          [("min_p", v) for v in (-0.1, -inf, -5e-324, 1.0 + 2.0 ** -52, inf, nan)]
    rows = 2 * len(bad) + 2
    R = _returns(rows, K, dtype, K, masked=0.02)
    for D in (1, 9):
        u = _numbers(rows, D, K + D)
        for usual in (dict(kappa=0.8, top_k=0, top_p=0.9, min_p=0.01), dict(kappa=0.8, top_k=K // 3, top_p=1.0, min_p=0.0)):
            of = {name: torch.full((rows,), usual[name], dtype=torch.int64 if name == "top_k" else torch.float64, device="cuda") for name in usual}
            for i, (name, value) in enumerate(bad):
                of[name][2 * i + 1] = value
            of["top_k"][rows - 1] = -3
            index, weight = _draw(R, u, **of)
            for i, (name, value) in enumerate(bad):
                assert (index[2 * i + 1] == -1).all() and (weight[2 * i + 1] == 0).all(), (name, value)
            _check(R[::2], u[::2], got=(index[::2], weight[::2]), **usual)
            _check(R[-1:], u[-1:], got=(index[-1:], weight[-1:]), **dict(usual, top_k=0))


def test_many_rows_and_many_draws():
    R, u = _returns(700, 130, "float32", 1), _numbers(700, 1, 1)
    _check(R, u, kappa=2.0, top_k=64, top_p=0.95, min_p=0.01)
    R, u = _returns(3, 200, "float64", 2), _numbers(3, 5000, 2)
    _check(R, u, kappa=0.3)
    R, u = _returns(2, 9000, "float32", 3), _numbers(2, 2000, 3)
    _check(R, u, kappa=0.5, top_p=0.9)
    R, u = _returns(1, 100000, "bfloat16", 4), _numbers(1, 600, 4)
    _check(R, u, kappa=0.5, top_p=0.9, top_k=60000)


def test_many_small_rows():
    """More rows than a grid's second dimension holds; compared with the two-sample formula in closed form."""
    import torch
    R, u = _returns(70001, 2, "float32", 5), _numbers(70001, 1, 5)
    index, weight = _draw(R, u, kappa=0.8)
    w = torch.exp(0.8 * (R.double() - R.double().amax(1, keepdim=True)))
    want = (u[:, 0] * w.sum(1) >= w[:, 0]).long()
    assert torch.equal(index[:, 0], want)
    share = w.gather(1, index) / w.sum(1, keepdim=True)
    assert ((weight.double() - share).abs() <= WEIGHT_RTOL * share).all()
    for D in (8, 9, 100):                                    # rows that one wave finishes, few draws and many
        for K in (3, 64, 65, 128, 129):
            _check(_returns(4, K, "float64", K + D, masked=0.2), _numbers(4, D, K + D), kappa=1.0, top_k=K // 2 + 1, top_p=0.8, min_p=0.01)


def test_more_rows_than_one_grid_holds():
    """2^26 + 5 rows of one sample, a wave each: 2^32 threads are more than a grid can have.  Rows with a NaN stay empty."""
    import torch
    rows = (1 << 26) + 5
    R = torch.zeros(rows, 1, dtype=torch.bfloat16, device="cuda")
    bad = [0, 12345, (1 << 26) - 2, (1 << 26) - 1, 1 << 26, rows - 2]
    R[bad] = float("nan")
    index, weight = _draw(R, torch.full((rows, 1), 0.3, dtype=torch.float64, device="cuda"))
    assert (index[bad] == -1).all() and (weight[bad] == 0).all()
    assert (index.count_nonzero(), weight.count_nonzero()) == (len(bad), rows - len(bad))
    assert (weight.max(), index.min(), index.max()) == (1, -1, 0)


def test_more_draws_than_one_workgroup_takes():
    for K, D, dtype in ((300, 16385, "float64"), (3000, 33000, "float32"), (9000, 40000, "bfloat16"), (20000, 8192, "float32"), (20000, 8193, "float32")):
        _check(_returns(2, K, dtype, K, masked=0.1), _numbers(2, D, K), kappa=0.7, top_p=0.99)


def test_more_draws_of_a_long_row_than_one_grid_holds():
    """2^26 + 5 draws, a wave each, from a row with two samples."""
    import torch
    D, K = (1 << 26) + 5, 40000
    R = torch.full((1, K), float("-inf"), device="cuda")
    R[0, 77] = R[0, 39999] = 3.0
    u = torch.full((1, D), 0.25, dtype=torch.float64, device="cuda")
    u[0, 1::2] = 0.75
    u[0, [0, (1 << 26) - 2, (1 << 26) - 1, 1 << 26, D - 1]] = 0.5
    index, weight = _draw(R, u)
    assert torch.equal(index, torch.where(u < 0.5, 77, 39999)) and (weight == 0.5).all()


def test_negated_views():
    """A view that torch negates lazily: its memory holds the other sign."""
    import torch
    z = torch.complex(torch.zeros(2, 50, device="cuda"), _returns(2, 50, "float32", 3))
    u = _numbers(2, 4, 3)
    lazy = z.conj().imag
    assert lazy.is_neg()
    with pytest.raises(ValueError, match="negated"):
        _draw(lazy, u)
    _check(lazy.resolve_neg(), u, kappa=0.5)
    half = torch.complex(torch.zeros_like(u), -u).conj().imag                 # as u, and as a row's parameter
    assert half.is_neg() and torch.equal(half.resolve_neg(), u)
    want = _draw(z.imag, u, top_p=u[:, 0].contiguous())
    got = _draw(z.imag, half, top_p=half[:, 0])
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_longest_row(dtype):
    """The largest K there is: every index up to 2^24 - 1 is reached by its own chunk, and one sample more is refused."""
    import torch
    from trajopt_amd._lib import MppiError
    K = 1 << 24
    R = _returns(1, K, dtype, 1)
    _check(R, _numbers(1, 7, 1), kappa=0.6, top_k=K // 5, top_p=0.9)
    one = torch.full((1, K), float("-inf"), dtype=R.dtype, device="cuda")
    for at in (0, K // 2 + 12345, K - 1):
        one.fill_(float("-inf"))
        one[0, at] = 2.0
        assert _draw(one, _numbers(1, 2, 1), top_p=0.5)[0].tolist() == [[at, at]]
    with pytest.raises(MppiError):
        _draw(torch.zeros(1, K + 1, dtype=R.dtype, device="cuda"), _numbers(1, 1, 1))


@pytest.mark.parametrize("rows,K,dtype", [(39, 20001, "float32"), (40, 20001, "float32"), (40, 20001, "bfloat16"), (41, 16385, "float16"), (32, 16385, "bfloat16"),
                                          (64, 32768, "float32"), (63, 32768, "float32"), (128, 65536, "bfloat16"), (129, 65535, "float16"), (33, 16384, "float64")])
def test_many_long_rows(rows, K, dtype):
    """As many rows as are taken by one workgroup each, or one less."""
    R, u = _returns(rows, K, dtype, rows, masked=0.02), _numbers(rows, 2, rows)
    for f in (dict(), dict(top_k=300), dict(top_k=5000, top_p=0.8), dict(top_p=0.9, min_p=0.02)):
        _check(R, u, kappa=0.8, **f)


@pytest.mark.parametrize("D", [1, 8, 9, 30])
@pytest.mark.parametrize("step", [0.0, 0.01, 0.5])
@pytest.mark.parametrize("dtype", TYPES)
def test_draws_of_long_rows(dtype, step, D):
    """Few and many samples near the border (returns rounded to multiples of a step share values), with either border, both of
    them, and neither."""
    K = 70001
    R = _returns(3, K, dtype, D, masked=0.01)
    if step:
        R = ((R.double() / step).round() * step).to(R.dtype)
    u = _numbers(3, D, D)
    for f in (dict(top_k=1), dict(top_k=900), dict(top_p=0.9), dict(top_k=5000, top_p=0.6), dict(top_k=30000, top_p=0.99, min_p=0.01),
              dict(top_k=K - 1), dict(min_p=0.2)):
        _check(R, u, kappa=0.9, **f)


def test_offsets_beyond_32_bits():
    """Rows, and samples of a row, further apart than 2^31 elements; and more than 2^31 samples in one call, of rows that one workgroup holds
    and of rows in chunks (their lists lie as far apart)."""
    import torch
    far = 1 << 31
    flat = torch.full((far + (1 << 20),), float("-inf"), dtype=torch.bfloat16, device="cuda")
    for shape, strides in (((3, 50), (far // 2 + 7, 1)), ((3, 5000), (far // 2 + 7, 1)), ((2, 70001), (far + 11, 1)), ((2, 300), (5, far // 299)),
                           ((2, 6000), (7, far // 5999)), ((2, 70001), (3, far // 70000))):
        R = flat.as_strided(shape, strides)
        R.copy_(_returns(*shape, "bfloat16", shape[1]))
        _check(R, _numbers(shape[0], 5, shape[1]), kappa=0.8, top_k=shape[1] // 2, top_p=0.9)
        R.fill_(float("-inf"))
    del flat, R
    for rows, K in ((40000, 65000), (33000, 70000)):
        R = torch.full((rows, K), float("-inf"), dtype=torch.bfloat16, device="cuda")
        first, gap = torch.arange(rows, device="cuda") * 7919 % (K - 200), torch.arange(rows, device="cuda") % 199 + 1
        R.scatter_(1, torch.stack((first, first + gap), 1), 2.0)         # two samples of the same weight
        u = torch.tensor([[0.25, 0.75]], dtype=torch.float64, device="cuda").repeat(rows, 1)
        index, weight = _draw(R, u, top_p=0.9)
        assert torch.equal(index, torch.stack((first, first + gap), 1)) and (weight == 0.5).all()
        index, weight = _draw(R, u, top_p=0.4)
        assert torch.equal(index, torch.stack((first, first), 1)) and (weight == 1).all()
        del R


def test_nothing_to_do():
    import torch
    R, u = _returns(2, 10, "float32", 0), _numbers(2, 0, 0)
    assert _draw(R, u)[0].shape == (2, 0)
    assert _draw(R[:0], _numbers(0, 4, 0))[0].shape == (0, 4)
    with pytest.raises(RuntimeError):
        _draw(R[:, :0], _numbers(2, 1, 0))
    assert torch.cuda.current_device() == 0


def test_rows_behind_the_last_are_left_alone():
    """The library writes rows x D values and nothing else."""
    import ctypes
    import torch
    from trajopt_amd import _lib as L
    for K in (40, 5000, 70000):
        R, u = _returns(3, K, "float32", 1), _numbers(3, 2, 1)
        index = torch.full((12,), 77, dtype=torch.int64, device="cuda")
        weight = torch.full((12,), 7.0, device="cuda")
        f = L.DrawFilterC(kappa=1.0, top_k=5, top_p=0.9, min_p=0.0)
        torch.cuda.synchronize()
        index2, weight2 = _draw(R, u, kappa=1.0, top_k=5, top_p=0.9)
        need = ctypes.c_size_t()
        L.check(L.lib().mppi_draw_workspace(L.F32, 3, K, ctypes.byref(need)))
        ws = torch.full((need.value + 64,), 0x5a, dtype=torch.uint8, device="cuda")
        L.check(L.lib().mppi_draw_from_returns(0, R.data_ptr(), L.F32, 3, K, K, 1, u.data_ptr(), 2, ctypes.byref(f), index[3:].data_ptr(),
                                               weight[3:].data_ptr(), ws.data_ptr() if need.value else None, need.value,
                                               torch.cuda.current_stream().cuda_stream))
        assert (ws[need.value:] == 0x5a).all()
        torch.cuda.synchronize()
        assert (index[:3] == 77).all() and (index[9:] == 77).all() and (weight[:3] == 7).all() and (weight[9:] == 7).all()
        assert torch.equal(index[3:9].reshape(3, 2), index2) and torch.equal(weight[3:9].reshape(3, 2), weight2)
        assert ctypes.sizeof(f) == 64


@pytest.mark.parametrize("D", [2, 9])
@pytest.mark.parametrize("K", [40, 3000, 100000])
def test_captured_and_replayed(K, D):
    """Two graphs and eager calls in turn; every replay against the eager result of its own inputs."""
    import torch
    R, u = _returns(2, K, "float32", K), _numbers(2, D, K)
    _draw(R, u, kappa=1.0, top_k=30, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    ins = [(R.clone(), u.clone()), (R.flip(1).contiguous(), u.clone())]
    with torch.cuda.stream(side):
        for r, v in ins:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(_draw(r, v, kappa=1.0, top_k=30, top_p=0.9))
            graphs.append(g)
    torch.cuda.synchronize()
    for turn in range(4):
        for (r, v), g, out in zip(ins, graphs, outs):
            v.copy_(_numbers(2, D, 50 + turn))
            r.copy_(_returns(2, K, "float32", 90 + turn))
            g.replay()
            want = _draw(r, v, kappa=1.0, top_k=30, top_p=0.9)
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        _check(ins[0][0], ins[0][1], kappa=1.0, top_k=30, top_p=0.9, got=outs[0])


def test_two_streams_at_once_and_repeated_calls():
    """Same bits every time, whatever runs beside it."""
    import torch
    sets = [(_returns(1, K, "float32", K), _numbers(1, 8, K)) for K in (100000, 90001, 70000, 300)]
    want = [_draw(R, u, kappa=0.5, top_k=5000, top_p=0.9) for R, u in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[] for _ in sets]
    for _ in range(5):
        for k, (R, u) in enumerate(sets):
            with torch.cuda.stream(streams[k]):
                got[k].append(_draw(R, u, kappa=0.5, top_k=5000, top_p=0.9))
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        for g in gs:
            assert torch.equal(w[0], g[0]) and torch.equal(w[1], g[1])


def test_shares_of_many_draws():
    """The frequencies of 200 000 draws are the weights (five standard deviations of a binomial count)."""
    import torch
    R = _returns(1, 6, "float32", 8, spread=0.7)
    n = 200000
    index, weight = _draw(R, torch.rand(1, n, dtype=torch.float64, device="cuda", generator=torch.Generator("cuda").manual_seed(3)), kappa=1.0)
    share = torch.bincount(index[0], minlength=6).double().cpu().numpy() / n
    w = ref_learn.kept_weights(R[0].double().cpu().numpy(), 1.0)
    w /= w.sum()
    assert np.all(np.abs(share - w) < 5 * np.sqrt(w * (1 - w) / n))

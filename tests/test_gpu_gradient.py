"""Gradient norm and clipping against the definition in 64 bits (oracle/ref_learn.py).

Tolerances.  The norm: fp64 sums of fp64 squares (below 1e-12 relative at these sizes), rounded to float32 once, 2^-24.
A clipped fp32 entry: one rounding of an fp64 product, 2^-24 relative.  A clipped 16-bit entry: the product is rounded to fp32
first (2^-24), then to the type: eps / 2 relative, or half the smallest subnormal step of the type."""
import numpy as np
import pytest

from oracle import ref_learn

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]


def _tensors(sizes, dtype, seed, scale=1.0):
    import torch
    rng = np.random.RandomState(seed)
    return [torch.tensor(scale * rng.normal(size=n) * 10.0 ** rng.uniform(-3, 0), device="cuda").to(getattr(torch, dtype)) for n in sizes]


def _numpy(tensors):
    return [t.double().cpu().numpy() for t in tensors]


def _close(t, want):
    import torch
    f = torch.finfo(t.dtype)
    step = float(f.tiny) * float(f.eps)
    extra = 0.0 if t.dtype == torch.float32 else 2.0 ** -24
    got = t.double().cpu().numpy()
    assert np.all(np.abs(got - want) <= (f.eps / 2 + extra) * 1.0000001 * np.abs(want) + step / 2), np.abs(got - want).max()


def _check(grads, max_norm, kind="l2", inplace=True):
    import torch
    from trajopt_amd.device import clip_gradients, gradient_norm
    before = _numpy(grads)
    kept = [g.clone() for g in grads]
    want_norm, want = ref_learn.clip(before, max_norm, kind)
    n0 = gradient_norm(grads, norm=kind)
    outs = grads if inplace else [torch.full_like(g, 3.0) for g in grads]
    n1 = clip_gradients(grads, max_norm, norm=kind, out=None if inplace else outs)
    assert n0.shape == () and n0.dtype == torch.float32 and torch.equal(n0, n1)
    with np.errstate(over="ignore"):
        rounded = float(np.float32(want_norm))       # a norm beyond fp32 (3e38 in four entries: 4.1e38 > 3.403e38) is reported as infinite
    assert float(n1) == rounded or abs(float(n1) - want_norm) <= (2.0 ** -24 + 1e-12) * want_norm
    for o, w, g, k in zip(outs, want, grads, kept):
        if want_norm > max_norm:
            _close(o, w.reshape(o.shape))
        else:
            assert torch.equal(o, k)
        if not inplace:
            assert torch.equal(g, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["l2", "max"])
@pytest.mark.parametrize("inplace", [True, False])
@pytest.mark.parametrize("sizes", [(1,), (3,), (1, 1), (7, 0, 9), (64,), (1792, 128, 16384, 128, 128, 1), (16383,), (16384,), (16385, 1, 40000),
                                   (100003, 5, 262145)])
def test_clip(dtype, kind, inplace, sizes):
    grads = _tensors(sizes, dtype, sum(sizes))
    norm = ref_learn.norm(_numpy(grads), kind)
    for max_norm in (norm * 0.3, norm * 2.0):
        _check([g.clone() for g in grads], max_norm, kind, inplace)


def test_clipping_to_nothing_and_to_no_bound():
    import torch
    from trajopt_amd.device import clip_gradients
    grads = _tensors((100, 3), "float32", 1)
    keep = [g.clone() for g in grads]
    clip_gradients(grads, float("inf"))
    assert all(torch.equal(g, k) for g, k in zip(grads, keep))
    clip_gradients(grads, 0.0)
    assert all((g == 0).all() for g in grads)
    assert float(clip_gradients(grads, 1.0)) == 0.0 and all((g == 0).all() for g in grads)


@pytest.mark.parametrize("kind", ["l2", "max"])
@pytest.mark.parametrize("n", [2, 127, 128, 129, 167, 168, 169, 300, 335, 336, 337, 1200])
def test_many_tensors_of_mixed_types(n, kind):
    rng = np.random.RandomState(n)
    grads = []
    for i in range(n):
        grads += _tensors((int(rng.choice([0, 1, 5, 129, 700, 20000], p=[.05, .2, .25, .25, .23, .02])),), TYPES[rng.randint(3)], i)
    norm = ref_learn.norm(_numpy(grads), kind)
    _check(grads, norm * 0.5, kind, inplace=bool(n % 2))


@pytest.mark.parametrize("dtype", TYPES)
def test_every_alignment(dtype):
    """Views at every offset from a 16-byte line, packed back to back, and outputs aligned otherwise than their inputs."""
    import torch
    flat = _tensors((60000,), dtype, 3)[0]
    out = torch.full((60010,), 9.0, device="cuda", dtype=flat.dtype)
    at, grads, outs = 0, [], []
    for n in (1, 2, 3, 5, 8, 13, 17, 33, 1001, 4099, 17003, 20001):
        grads.append(flat[at:at + n])
        outs.append(out[at + 5:at + 5 + n])
        at += n
    from trajopt_amd.device import clip_gradients
    norm, want = ref_learn.clip(_numpy(grads), 0.25)
    assert norm > 0.25
    clip_gradients(grads, 0.25, out=outs)
    for o, w in zip(outs, want):
        _close(o, w)
    assert (out[:5] == 9.0).all() and (out[5 + at:] == 9.0).all()            # nothing beside the outputs
    rest = flat[at:].clone()
    _check(grads, 0.25)
    assert torch.equal(flat[at:], rest)


def test_layouts():
    """Permuted dense tensors are taken as they lie; slices and expanded gradients are refused."""
    import torch
    from trajopt_amd.device import clip_gradients, gradient_norm
    g = torch.randn(6, 5, 4, device="cuda", generator=torch.Generator("cuda").manual_seed(0))
    _check([g.permute(2, 0, 1), g.clone().t() if g.dim() == 2 else g.clone()], 0.5)
    with pytest.raises(ValueError):
        clip_gradients([g[:, :3]], 1.0)
    with pytest.raises(ValueError):
        gradient_norm([torch.ones(1, device="cuda").expand(10)])
    # the gradient of a broadcast input is expanded by autograd: it has to be made dense first
    x = torch.randn(10, device="cuda", requires_grad=True)
    x.sum().backward()
    dense = x.grad.contiguous() if not x.grad.is_contiguous() else x.grad.clone()
    assert abs(float(gradient_norm([dense])) - np.sqrt(10.0)) < 1e-6


def test_large_and_small_magnitudes():
    """Squares that fp32 cannot hold, and subnormal gradients."""
    import torch
    for scale in (1e30, 1e-38, 3e38):
        g = [torch.tensor([1.0, -0.25, 0.5, 0.75], device="cuda") * scale]
        norm = ref_learn.norm(_numpy(g))
        _check(g, norm * 1e-3 if scale > 1 else norm * 0.5)
    # the norm itself beyond fp32: reported as infinite, the gradients still clipped
    from trajopt_amd.device import clip_gradients
    g = [torch.full((100,), 3e38, device="cuda")]
    assert float(clip_gradients(g, 1.0)) == float("inf")
    assert torch.allclose(g[0], torch.full_like(g[0], 0.1))
    # a scale below fp32's range
    for n in (300, 200000):
        g = [torch.full((n,), 3e38, device="cuda").to(torch.bfloat16), torch.full((n,), 1e30, device="cuda")]
        _check(g, 1e-7)
    for dtype in (torch.float16, torch.bfloat16):
        g = [torch.full((4096,), torch.finfo(dtype).max / 2, dtype=dtype, device="cuda")]
        _check(g, 1.0)
        g = [torch.full((64,), torch.finfo(dtype).tiny * 4, dtype=dtype, device="cuda")]
        _check(g, float(torch.finfo(dtype).tiny) * 3.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("kind", ["l2", "max"])
@pytest.mark.parametrize("n", [50, 70000])
def test_a_norm_that_is_not_finite_changes_nothing(dtype, bad, kind, n):
    import torch
    from trajopt_amd.device import clip_gradients
    grads = _tensors((n, 33, n + 1), dtype, 4)
    grads[1][20] = bad
    keep = [g.clone() for g in grads]
    outs = [torch.zeros_like(g) for g in grads]
    norm = clip_gradients(grads, 0.01, norm=kind, out=outs)
    assert torch.isnan(norm) if np.isnan(bad) else torch.isinf(norm)
    clip_gradients(grads, 0.01, norm=kind)
    for a in (grads, outs):
        for g, k in zip(a, keep):
            assert torch.equal(g.view(torch.int32 if dtype == "float32" else torch.int16), k.view(torch.int32 if dtype == "float32" else torch.int16))


def test_nothing_but_empty_tensors():
    import torch
    from trajopt_amd.device import clip_gradients, gradient_norm
    e = [torch.zeros(0, device="cuda"), torch.zeros(0, device="cuda", dtype=torch.bfloat16)]
    assert float(gradient_norm(e)) == 0.0 and float(clip_gradients(e, 1.0)) == 0.0
    assert float(gradient_norm(e, norm="max")) == 0.0


def test_same_bits_every_time_and_on_other_streams():
    import torch
    from trajopt_amd.device import clip_gradients
    sets = [_tensors((n, 1000, 77), "bfloat16", n) for n in (300000, 50000, 10)]
    want = []
    for g in sets:
        out = [torch.empty_like(x) for x in g]
        want.append((clip_gradients(g, 0.1, out=out), out))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(4):
        for g, s, w in zip(sets, streams, want):
            with torch.cuda.stream(s):
                out = [torch.empty_like(x) for x in g]
                got.append((clip_gradients(g, 0.1, out=out), out, w))
    torch.cuda.synchronize()
    for norm, out, w in got:
        assert torch.equal(norm, w[0]) and all(torch.equal(a, b) for a, b in zip(out, w[1]))


@pytest.mark.parametrize("sizes", [((5000, 128, 300), (200000, 128, 300)), ((700,) * 170, (4001,) * 400)])
def test_captured_and_replayed(sizes):
    """Two graphs over different gradients, with eager calls between the replays; few tensors, and more than travel in arguments."""
    import torch
    from trajopt_amd.device import clip_gradients
    base = [_tensors(s, "float32", len(s)) for s in sizes]
    live = [[g.clone() for g in b] for b in base]
    clip_gradients([g.clone() for g in base[0]], 0.1)
    torch.cuda.synchronize()
    graphs, norms = [], []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for l in live:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                norms.append(clip_gradients(l, 0.1))
            graphs.append(graph)
    torch.cuda.synchronize()
    for turn in range(4):
        for b, l, graph, norm in zip(base, live, graphs, norms):
            for x, y in zip(l, b):
                x.copy_(y * (1.0 + turn))
            eager = [x.clone() for x in l]
            graph.replay()
            want = clip_gradients(eager, 0.1)
            torch.cuda.synchronize()
            assert torch.equal(norm, want) and all(torch.equal(x, y) for x, y in zip(l, eager))
            assert abs(ref_learn.norm(_numpy(l)) - 0.1) < 1e-7


def test_refusals():
    import torch
    from trajopt_amd._lib import MppiError
    from trajopt_amd.device import clip_gradients, gradient_norm
    g = torch.ones(100, device="cuda")
    with pytest.raises(ValueError):
        gradient_norm([])
    with pytest.raises(ValueError):
        gradient_norm([g], norm="l3")
    with pytest.raises(TypeError):
        gradient_norm([g.cpu()])
    with pytest.raises(TypeError):
        gradient_norm([g.double()])
    with pytest.raises(TypeError):
        gradient_norm([g.long()])
    for bad in (-1.0, float("nan")):
        with pytest.raises(MppiError):
            clip_gradients([g], bad)
    with pytest.raises(MppiError):
        clip_gradients([g, g], 1.0)                               # the same tensor twice
    with pytest.raises(MppiError):
        clip_gradients([g[:60], g[50:]], 1.0)
    with pytest.raises(MppiError):
        clip_gradients([g[:50]], 1.0, out=[g[20:70]])
    with pytest.raises(MppiError):
        clip_gradients([g[:50], g[50:]], 1.0, out=[g[50:], g[:50]])
    with pytest.raises(ValueError):
        clip_gradients([g], 1.0, out=[g, g])
    with pytest.raises(ValueError):
        clip_gradients([g], 1.0, out=[torch.ones(99, device="cuda")])
    with pytest.raises(ValueError):
        clip_gradients([g], 1.0, out=[g.half()])
    assert abs(float(gradient_norm([g, g])) - np.sqrt(200.0)) < 1e-5      # reading twice is no harm: counted twice
    assert (g == 1).all()


def test_negated_views_are_refused():
    """A view that torch negates lazily: its memory holds the other sign."""
    import torch
    from trajopt_amd.device import clip_gradients, gradient_norm
    lazy = torch.complex(torch.zeros(1, device="cuda"), torch.ones(1, device="cuda")).conj().imag
    assert lazy.is_neg()
    with pytest.raises(ValueError, match="negated"):
        gradient_norm([lazy])
    with pytest.raises(ValueError, match="negated"):
        clip_gradients([torch.ones(1, device="cuda")], 1.0, out=[lazy])


@pytest.mark.parametrize("kind", ["l2", "max"])
def test_one_tensor_beyond_32_bits(kind):
    """More than 2^31 entries in one tensor (and 2^32 bytes): entries at its ends and near 2^31, zeros between them."""
    import torch
    from trajopt_amd.device import clip_gradients, gradient_norm
    n = (1 << 31) + 12345
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 1, (1 << 30) + 3, (1 << 31) - 1, 1 << 31, (1 << 31) + 1, n - 2, n - 1], device="cuda")
    values = torch.tensor([3.0, -4.0, 2.0, 6.0, -1.0, 5.0, 8.0, -7.0], dtype=torch.bfloat16, device="cuda")
    g[at] = values
    small = torch.full((100,), 0.5, device="cuda")
    both = [g, small]
    want_norm, want = ref_learn.clip([values.double().cpu().numpy(), small.double().cpu().numpy()], 2.0, kind)
    assert want_norm > 2.0
    norm = gradient_norm(both, norm=kind)
    assert abs(float(norm) - want_norm) <= (2.0 ** -24 + 1e-12) * want_norm
    assert torch.equal(clip_gradients(both, 2.0, norm=kind), norm)
    _close(g[at], want[0])
    _close(small, want[1])
    g[at] = 0
    assert not g.any()

"""Refusals of the draw and gradient entry points, and the oracle they are tested against (no GPU: nothing is launched)."""
import ctypes as C

import numpy as np
import pytest

from oracle import ref_learn


def _draw(**kw):
    from trajopt_amd import _lib as L
    a = dict(device=0, R=0x1000, dtype=L.F32, rows=2, K=10, rs=10, cs=1, u=0x2000, D=1, kappa=1.0, top_k=0, top_p=1.0, min_p=0.0,
             index=0x3000, filter=True, ws=None, ws_bytes=0)
    a.update(kw)
    f = L.DrawFilterC(kappa=a["kappa"], top_k=a["top_k"], top_p=a["top_p"], min_p=a["min_p"])
    return L.lib().mppi_draw_from_returns(a["device"], a["R"], a["dtype"], a["rows"], a["K"], a["rs"], a["cs"], a["u"], a["D"],
                                          C.byref(f) if a["filter"] else None, a["index"], None, a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(filter=False), -1), (dict(K=0), -1), (dict(K=-4), -1), (dict(rows=-1), -1), (dict(D=-1), -1), (dict(rs=-1), -1), (dict(cs=-2), -1),
    (dict(dtype=4), -1), (dict(dtype=-1), -1), (dict(K=(1 << 24) + 1), -6), (dict(R=None), -1), (dict(u=None), -1), (dict(index=None), -1),
    (dict(kappa=-0.5), -1), (dict(kappa=float("nan")), -1), (dict(kappa=float("inf")), -1), (dict(top_k=-1), -1), (dict(top_p=0.0), -1),
    (dict(top_p=1.5), -1), (dict(top_p=float("nan")), -1), (dict(min_p=-0.1), -1), (dict(min_p=1.1), -1), (dict(min_p=float("nan")), -1),
    (dict(K=100000), -1), (dict(K=100000, ws=0x10000, ws_bytes=4096), -1), (dict(K=100000, ws=0x10010, ws_bytes=1 << 40), -1),
    (dict(rows=0), 0), (dict(D=0), 0), (dict(rows=0, R=None, index=None, u=None), 0)])
def test_draw_refuses(kw, code):
    from trajopt_amd import _lib as L
    assert _draw(**kw) == code
    if code:
        assert L.lib().mppi_last_error()


def _clip(grads, out, sizes, types, norm_type=0, max_norm=1.0, norm=0x100, ws=0x10000, ws_bytes=1 << 20):
    from trajopt_amd import _lib as L
    n = len(sizes)
    g = (C.c_void_p * n)(*grads) if grads is not None else None
    o = (C.c_void_p * n)(*out) if out is not None else None
    return L.lib().mppi_clip_gradients(0, n, g, o, (C.c_int64 * n)(*sizes), (C.c_int32 * n)(*types), norm_type, max_norm, norm, ws, ws_bytes, None)


@pytest.mark.parametrize("args,kw", [
    (([0x1000], [0x1000], [4], [1]), {}),                                  # fp64
    (([0x1000], [0x1000], [4], [9]), {}),
    (([0x1000], [0x1000], [-4], [0]), {}),
    (([0x1000], [0x1000], [4], [0]), dict(norm_type=2)),
    (([0x1000], [0x1000], [4], [0]), dict(max_norm=-1.0)),
    (([0x1000], [0x1000], [4], [0]), dict(max_norm=float("nan"))),
    (([0x1000], [0x1000], [4], [0]), dict(norm=None)),
    (([0x1000], [0x1000], [4], [0]), dict(ws=None)),
    (([0x1000], [0x1000], [4], [0]), dict(ws_bytes=4)),
    (([0x1000], [0x1000], [4], [0]), dict(ws=0x10004)),
    (([None], [0x1000], [4], [0]), {}),
    (([0x1000], [None], [4], [0]), {}),
    ((None, [0x1000], [4], [0]), {}),
    (([0x1000], None, [4], [0]), {}),
    (([0x1002], [0x1002], [4], [0]), {}),                                  # not a multiple of four
    (([0x1001], [0x1001], [4], [3]), {}),
    (([0x1000, 0x1000], [0x1000, 0x1000], [4, 4], [0, 0]), {}),            # twice the same
    (([0x1000, 0x1008], [0x1000, 0x1008], [4, 4], [0, 0]), {}),            # overlapping
    (([0x1000], [0x1008], [4], [0]), {}),                                  # output over its input's end
    (([0x1000, 0x2000], [0x2000, 0x1000], [4, 4], [0, 0]), {}),            # outputs over the other's input
    (([0x1000, 0x2000], [0x3000, 0x3004], [4, 4], [0, 0]), {}),            # outputs over each other
    (([0x1000], [0x1000], [(1 << 40) + 1], [0]), {}),
])
def test_clip_refuses(args, kw):
    from trajopt_amd import _lib as L
    assert _clip(*args, **kw) in (-1, -6)
    assert L.lib().mppi_last_error()


def test_workspace_query():
    from trajopt_amd import _lib as L
    need = C.c_size_t()
    for dtype, most in ((L.F32, 32768), (L.F64, 16384), (L.F16, 65536), (L.BF16, 65536)):
        assert L.lib().mppi_draw_workspace(dtype, 1000, most, C.byref(need)) == 0 and need.value == 0
        assert L.lib().mppi_draw_workspace(dtype, 3, most + 1, C.byref(need)) == 0
        assert 3 * (most + 1) * 8 <= need.value < 3 * (most + 1) * 14 + 100000
    for bad in ((L.F32, -1, 5), (L.F32, 1, 0), (9, 1, 5), (L.F32, 1, (1 << 24) + 1)):
        assert L.lib().mppi_draw_workspace(*bad, C.byref(need)) < 0
    assert L.lib().mppi_draw_workspace(L.F32, 1, 5, None) == -1
    assert L.lib().mppi_gradient_workspace(-1, C.byref(need)) == -1 and L.lib().mppi_gradient_workspace(1, None) == -1
    for n in (0, 1, 168, 169, 100000):         # partial sums of 1024 workgroups, and a table entry of 24 bytes where they do not travel
        assert L.lib().mppi_gradient_workspace(n, C.byref(need)) == 0 and need.value == 1024 * 8 + (24 * n if n > 168 else 0)


def test_python_refusals():
    import torch
    from trajopt_amd.device import clip_gradients, draw_from_returns, gradient_norm
    R, u = torch.zeros(4), torch.zeros(1, dtype=torch.float64)
    with pytest.raises(TypeError):
        draw_from_returns(R, u)                 # host tensors: there is no CPU form
    with pytest.raises(TypeError):
        draw_from_returns(np.zeros(4), np.zeros(1))
    with pytest.raises(TypeError):
        gradient_norm([R])
    with pytest.raises(TypeError):
        clip_gradients([None], 1.0)
    with pytest.raises(ValueError):
        clip_gradients([], 1.0)


def test_tensors_that_autograd_follows_are_refused():
    """There are no derivatives: what would drop a graph without a word is refused before anything is launched (tensors
    without memory, so that no GPU is needed)."""
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode
    from trajopt_amd.device import clip_gradients, draw_from_returns, gradient_norm
    with FakeTensorMode():
        x = torch.empty(3, 4, device="cuda")
        leaf = torch.empty(3, 4, device="cuda", requires_grad=True)
        row = torch.empty(3, dtype=torch.float64, device="cuda", requires_grad=True)
        u = torch.empty(3, 1, device="cuda", dtype=torch.float64)
        for call in (lambda: draw_from_returns(leaf, u), lambda: draw_from_returns(leaf * 2.0, u), lambda: draw_from_returns(x, u, kappa=row),
                     lambda: draw_from_returns(x, u, top_p=row), lambda: draw_from_returns(x, u, min_p=row),
                     lambda: gradient_norm([x, leaf]), lambda: gradient_norm(leaf * 2.0), lambda: clip_gradients([leaf], 1.0),
                     lambda: clip_gradients([leaf * 2.0], 1.0), lambda: clip_gradients([x], 1.0, out=[leaf])):
            with pytest.raises(RuntimeError, match="no derivative"):
                call()


def test_numbers_of_a_drawn_step_are_checked_without_a_device():
    """What train_step(draw=...) asks before it touches anything: the argument's form, and whether a draw takes its numbers."""
    from trajopt.algos.mppi import MPPI
    from trajopt_amd._lib import MppiError
    from trajopt_amd.device import check_draw
    check_draw(8, 5.0)
    check_draw(1 << 24, 0.0, 1 << 40, 1.0, 1.0)
    for bad in ((0, 1.0), ((1 << 24) + 1, 1.0), (8, -1.0), (8, float("nan")), (8, 1.0, -1), (8, 1.0, 0, 0.0), (8, 1.0, 0, 1.1), (8, 1.0, 0, float("nan")),
                (8, 1.0, 0, 1.0, -0.5), (8, 1.0, 0, 1.0, 1.5)):
        with pytest.raises(MppiError):
            check_draw(*bad)
    with pytest.raises(TypeError):
        check_draw(8, 1.0, 2.5)
    for u in (0.25, np.float32(0.25), np.array([0.25]), [0.25]):
        assert MPPI._draw_arguments(dict(u=u), 0, 1)["u"] == 0.25
    for u in ([], [0.1, 0.2], float("nan"), float("inf"), "x"):
        with pytest.raises(ValueError):
            MPPI._draw_arguments(dict(u=u), 0, 1)


def test_top_k_beyond_64_bits():
    """Not its lowest 64 bits, which would keep 5 samples, or none of a filter."""
    from trajopt_amd.device import DevicePlanner, check_draw
    check_draw(8, 1.0, 2 ** 63 - 1)
    for k in (2 ** 64 + 5, 2 ** 64, 2 ** 63, -2 ** 63 - 1):
        with pytest.raises(OverflowError):
            check_draw(8, 1.0, k)
        p = DevicePlanner.__new__(DevicePlanner)              # (no device behind it: nothing may be called)
        p.P, p._h = 1, None
        with pytest.raises(OverflowError):
            p.draw(0.5, top_k=k)


def test_oracle_draws():
    R = np.array([1.0, 3.0, np.nan, 2.0, 3.0, -np.inf])
    assert np.allclose(ref_learn.kept_weights(R, 1.0), [np.exp(-2), 1, 0, np.exp(-1), 1, 0])
    assert np.array_equal(ref_learn.kept_weights(R, 1.0, top_k=1) > 0, [0, 1, 0, 0, 0, 0])         # ties: the lower index
    assert np.array_equal(ref_learn.kept_weights(R, 1.0, top_k=3) > 0, [0, 1, 0, 1, 1, 0])
    assert np.array_equal(ref_learn.kept_weights(R, 1.0, top_p=0.3) > 0, [0, 1, 0, 0, 0, 0])
    assert np.array_equal(ref_learn.kept_weights(R, 1.0, top_p=0.5) > 0, [0, 1, 0, 0, 1, 0])       # the one that crosses it is kept
    assert np.array_equal(ref_learn.kept_weights(R, 1.0, min_p=0.3) > 0, [0, 1, 0, 1, 1, 0])
    i, w = ref_learn.draw(R, [0.0, 0.99, 1.0, np.nan], 0.0)
    assert i.tolist() == [0, 4, 4, 0] and np.allclose(w, 0.25)
    assert ref_learn.draw([np.nan], [0.5])[0].tolist() == [-1]


def test_oracle_clip():
    n, c = ref_learn.clip([[3.0], [4.0]], 1.0)
    assert n == 5.0 and np.allclose(np.concatenate(c), [0.6, 0.8])
    n, c = ref_learn.clip([[3.0], [np.inf]], 1.0, "max")
    assert n == np.inf and np.array_equal(np.concatenate(c), [3.0, np.inf])

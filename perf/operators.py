"""Cases of the framework's draw and gradient operators, with their plain forms in elementary torch operations.

`draw_from_returns` picks samples of a planner by their exponentiated returns (kappa = 1 / temperature, top-k, top-p,
min-p) from given uniform numbers; `gradient_norm` and `clip_gradients` work on the gradients of many tensors.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}


# ---- cases ------------------------------------------------------------------------------------------------------------
def _draw_case(name, rows, K, D, dtype, kappa, top_k, top_p, min_p, spread, per_row=False, masked=0.0):
    return {"name": name, "op": "draw", "rows": rows, "K": K, "D": D, "dtype": dtype, "kappa": kappa, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "spread": spread, "per_row": per_row, "masked": masked}


def _clip_case(name, op, tensors, total, dtype, norm, max_norm, layout):
    return {"name": name, "op": op, "tensors": tensors, "total": total, "dtype": dtype, "norm": norm, "max_norm": max_norm,
            "layout": layout}


def listed():
    return [
        # one planning step of the example scripts: 40 samples, elites of 10, applied at every control step
        _draw_case("draw_script", 1, 40, 1, "f64", 25.0, 10, 1.0, 0.0, 1.5),
        # one planning step of the benchmark's planner: 4096 samples, nucleus
        _draw_case("draw_step", 1, 4096, 1, "f32", 25.0, 0, 0.95, 0.0, 0.3),
        # 1024 planners in one handle, each with its own temperature and filters
        _draw_case("draw_planners", 1024, 512, 1, "f32", 2.0, 64, 0.95, 0.01, 2.0, per_row=True),
        # resampling: as many draws as samples, no filter
        _draw_case("draw_resample", 64, 200, 200, "f32", 1.0, 0, 1.0, 0.0, 2.0),
        # one planner with the largest sample count of the benchmark tools
        _draw_case("draw_long", 1, 524288, 1, "f32", 4.0, 1024, 0.99, 0.0, 1.5),
        # many long rows of 16-bit scores, an odd length, a tenth of them masked
        _draw_case("draw_wide", 192, 65535, 4, "bf16", 1.0, 50, 0.9, 0.05, 2.0, masked=0.1),
        # fp64 planners, a broad nucleus, many draws from each
        _draw_case("draw_double", 16, 262144, 64, "f64", 0.5, 0, 0.9, 0.0, 3.0),
        # one step of the critic: its six tensors, the smallest call of a training loop
        _clip_case("clip_critic", "clip", 6, 18561, "f32", "l2", 1.0, "critic"),
        # an ensemble of 64 critics stepped together: 384 small tensors
        _clip_case("clip_ensemble", "clip", 384, 64 * 18561, "f32", "l2", 1.0, "critic"),
        # 16-bit gradients of odd sizes packed back to back, largest entry as the norm
        _clip_case("clip_ragged", "clip", 150, 5000011, "f16", "max", 0.5, "packed"),
        # a large model's bf16 gradients
        _clip_case("clip_large", "clip", 200, 1 << 27, "bf16", "l2", 1.0, "aligned"),
        # the norm alone (logged, or checked for infinities) of large fp32 gradients
        _clip_case("norm_large", "norm", 12, 1 << 28, "f32", "l2", 0.0, "aligned"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.6:
        dtype = rng.choice(["f64", "f32", "f16", "bf16"])
        K = _log_uniform(rng, 1, 524288)
        rows = _log_uniform(rng, 1, max(1, min(1024, (1 << 25) // (K * SIZE[dtype]))))
        D = _log_uniform(rng, 1, 256)
        top_k = rng.choice([0, _log_uniform(rng, 1, K)])
        top_p = rng.choice([1.0, round(rng.uniform(0.05, 0.999), 3)])
        min_p = rng.choice([0.0, round(math.exp(rng.uniform(math.log(1e-4), math.log(0.5))), 5)])
        return _draw_case("", rows, K, D, dtype, round(math.exp(rng.uniform(math.log(0.2), math.log(25.0))), 3), top_k, top_p,
                          min_p, round(rng.uniform(0.2, 4.0), 3), per_row=rng.random() < 0.4,
                          masked=rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.5), 3)]))
    op = rng.choice(["clip", "clip", "norm"])
    layout = rng.choice(["critic", "packed", "aligned"])
    tensors = _log_uniform(rng, 1, 400)
    total = _log_uniform(rng, tensors, 1 << 26)
    if layout == "critic":
        tensors = 6 * (1 + tensors // 6)
        total = tensors // 6 * 18561
    return _clip_case("", op, tensors, total, rng.choice(["f32", "f16", "bf16"]), rng.choice(["l2", "l2", "max"]),
                      0.0 if op == "norm" else round(math.exp(rng.uniform(math.log(0.1), math.log(100.0))), 3), layout)


def _sizes(case):
    """Element counts of the tensors of a gradient case."""
    n, total = case["tensors"], case["total"]
    if case["layout"] == "critic":
        return [14 * 128, 128, 128 * 128, 128, 128, 1] * (n // 6)
    share = np.random.RandomState(n).gamma(0.7, size=n) + 1e-3
    sizes = 1 + np.floor((total - n) * share / share.sum()).astype(np.int64)
    sizes[-1] += total - sizes.sum()
    return [int(s) for s in sizes]


def work(case):
    if case["op"] == "draw":
        values, draws = case["rows"] * case["K"], case["rows"] * case["D"]
        return {"bytes": values * SIZE[case["dtype"]] + draws * (8 + 8 + 4), "flops": 4 * values}
    once = case["total"] * SIZE[case["dtype"]]
    return {"bytes": once * (1 if case["op"] == "norm" else 2) + 4, "flops": case["total"] * (2 if case["op"] == "norm" else 3)}


# ---- inputs -----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if case["op"] == "draw":
        return _prepare_draw(case, gen)
    return _prepare_gradients(case, gen)


def _prepare_draw(case, gen):
    rows, K, D, dtype = case["rows"], case["K"], case["D"], TYPES[case["dtype"]]
    R = torch.randn(rows, K, generator=gen, device="cuda", dtype=torch.float64) * case["spread"] - 20.0
    R = R.to(dtype)
    if case["masked"]:
        # diverged rollouts and masked entries: NaN, -inf, +inf and the type's lowest value; and a planner that lost all
        at = torch.rand(rows, K, generator=gen, device="cuda")
        kinds = torch.tensor([math.nan, -math.inf, math.inf, torch.finfo(dtype).min], device="cuda", dtype=dtype)
        which = torch.randint(0, 4, (rows, K), generator=gen, device="cuda")
        R = torch.where(at < case["masked"], kinds[which], R)
        if rows > 1:
            R[rows // 2] = -math.inf
    u = torch.rand(rows, D, generator=gen, device="cuda", dtype=torch.float64)
    kappa, top_k, top_p, min_p = case["kappa"], case["top_k"], case["top_p"], case["min_p"]
    if case["per_row"]:
        # every planner its own: temperature within a factor of two, filters off on some of them
        kappa = kappa * torch.exp2(torch.rand(rows, generator=gen, device="cuda", dtype=torch.float64) * 2 - 1)
        on = torch.rand(3, rows, generator=gen, device="cuda") < 0.8
        top_k = torch.where(on[0], top_k, 0)
        top_p = torch.where(on[1], torch.tensor(top_p, device="cuda", dtype=torch.float64), 1.0)
        min_p = torch.where(on[2], torch.tensor(min_p, device="cuda", dtype=torch.float64), 0.0)
    return {"op": "draw", "R": R, "u": u, "kappa": kappa, "top_k": top_k, "top_p": top_p, "min_p": min_p}


def _prepare_gradients(case, gen):
    dtype, sizes = TYPES[case["dtype"]], _sizes(case)
    # "aligned": every tensor starts on 256 bytes; otherwise one behind the other, wherever that is
    step = 256 // SIZE[case["dtype"]] if case["layout"] == "aligned" else 1
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // step) * step
    # layers differ in scale by orders of magnitude, which a few powers of two over the buffer stand for
    flat = torch.randn(at, generator=gen, device="cuda", dtype=torch.float32)
    scale = torch.exp2(torch.randint(-6, 1, (max(1, at // 4096 + 1),), generator=gen, device="cuda").float()) * 0.1
    flat = (flat * scale.repeat_interleave(4096)[:at]).to(dtype)
    out = torch.zeros(at, device="cuda", dtype=dtype)
    grads = [flat[s:s + n] for s, n in zip(starts, sizes)]
    outs = [out[s:s + n] for s, n in zip(starts, sizes)]
    return {"op": case["op"], "grads": grads, "outs": outs, "out": out, "norm": case["norm"], "max_norm": case["max_norm"]}


# ---- one pass ---------------------------------------------------------------------------------------------------------
def run(state):
    if state["op"] == "draw":
        args = (state["R"], state["u"], state["kappa"], state["top_k"], state["top_p"], state["min_p"])
        if own:
            from trajopt_amd.device import draw_from_returns
            return draw_from_returns(*args)
        return _plain_draw(*args)
    if state["op"] == "norm":
        if own:
            from trajopt_amd.device import gradient_norm
            return gradient_norm(state["grads"], norm=state["norm"])
        return _plain_norm(state["grads"], state["norm"]).float()
    if own:
        from trajopt_amd.device import clip_gradients
        norm = clip_gradients(state["grads"], state["max_norm"], norm=state["norm"], out=state["outs"])
    else:
        norm = _plain_clip(state["grads"], state["max_norm"], state["norm"], state["outs"])
    return {"norm": norm, "grads": state["out"]}


def _plain_draw(R, u, kappa, top_k, top_p, min_p):
    rows, K = R.shape
    column = lambda v: v.reshape(rows, 1) if isinstance(v, torch.Tensor) else v  # noqa: E731
    kappa, top_k, top_p, min_p = column(kappa), column(top_k), column(top_p), column(min_p)
    R = R.double()                                   # neighbours of a border are told apart in 64 bits
    fine = torch.isfinite(R)
    R = torch.where(fine, R, -math.inf)
    best = R.amax(1, keepdim=True)
    w = torch.where(fine, torch.exp(kappa * (R - torch.where(torch.isfinite(best), best, 0.0))), 0.0)
    order = torch.sort(R, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(K, device=R.device).reshape(1, K)
    limit = torch.where(top_k > 0, top_k, K) if isinstance(top_k, torch.Tensor) else (top_k if top_k > 0 else K)
    ws = torch.where(rank < limit, ws, 0.0)
    upto = torch.cumsum(ws, 1)
    before = torch.cat((torch.zeros_like(upto[:, :1]), upto[:, :-1]), 1)
    keep = (before < top_p * upto[:, -1:]) & (ws >= min_p)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0.0))
    upto = torch.cumsum(kept, 1)
    mass = upto[:, -1:]
    index = torch.searchsorted(upto, u * mass, right=True).clamp_(max=K - 1)
    some = mass > 0
    weight = torch.where(some, kept.gather(1, index) / mass, 0.0)
    return torch.where(some, index, -1), weight.float()


def _plain_norm(grads, norm):
    if norm == "max":
        return torch.stack([g.float().abs().amax() for g in grads]).amax()
    return torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads]).sum().sqrt()


def _plain_clip(grads, max_norm, norm, outs):
    total = _plain_norm(grads, norm)
    s = torch.where((total > max_norm) & torch.isfinite(total), max_norm / total, 1.0)
    list(map(lambda o, g: o.copy_(g.float() * s), outs, grads))
    return total.float()


# ---- the definition, in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "draw":
        return _exact_draw(state)
    grads = [g.cpu().double().numpy() for g in state["grads"]]
    if case["norm"] == "max":
        total = max(float(np.max(np.abs(g))) for g in grads)
    else:
        total = math.sqrt(math.fsum(float(np.dot(g, g)) for g in grads))
    if case["op"] == "norm":
        return np.float64(total)
    s = case["max_norm"] / total if total > case["max_norm"] else 1.0
    out = np.zeros(state["out"].numel())
    base = state["out"].data_ptr()
    for g, o in zip(grads, state["outs"]):
        at = (o.data_ptr() - base) // o.element_size()
        out[at:at + g.size] = g * s
    return {"norm": np.float64(total), "grads": out}


def _exact_draw(state):
    R, u = state["R"].double().cpu().numpy(), state["u"].cpu().numpy()
    rows, K = R.shape
    own_of = lambda v: v.cpu().numpy() if isinstance(v, torch.Tensor) else np.full(rows, v)  # noqa: E731
    kappa, top_k, top_p, min_p = (own_of(state[n]) for n in ("kappa", "top_k", "top_p", "min_p"))
    index, weight = np.full(u.shape, -1, dtype=np.int64), np.zeros(u.shape)
    for b in range(rows):
        at = np.flatnonzero(np.isfinite(R[b]))
        if not len(at):
            continue
        at = at[np.argsort(-R[b, at], kind="stable")]
        if top_k[b] > 0:
            at = at[:int(top_k[b])]
        w = np.exp(kappa[b] * (R[b, at] - R[b, at[0]]))
        upto = np.cumsum(w, dtype=np.longdouble)
        w_left = w[(np.concatenate(([0], upto[:-1])) < top_p[b] * upto[-1]) & (w >= min_p[b])]
        left = at[:len(w_left)]                      # both conditions end at one place of the descending order
        back = np.argsort(left)
        left, w_left = left[back], w_left[back]
        upto = np.cumsum(w_left, dtype=np.longdouble)
        pick = np.minimum(np.searchsorted(upto, u[b] * upto[-1], side="right"), len(left) - 1)
        index[b], weight[b] = left[pick], w_left[pick] / np.float64(upto[-1])
    return index, weight

"""Draws and clipping where a user meets them: the planner applies a drawn sequence (mppi_draw, MPPI.train_step), the
critic trains with clipped gradients (Critic.clip_gradients), and both together as the actor-critic script runs them."""
import numpy as np
import pytest

from oracle import ref_learn, ref_mppi

pytestmark = pytest.mark.gpu
FILTER = [np.ones(7), 0.25, 0.8, 0.0]
WEIGHT_RTOL = 2.0 ** -24 * (1 + 1e-5) + 1e-13         # one rounding to float32 (tests/test_gpu_draw.py)


@pytest.fixture(scope="module")
def dm():
    from trajopt_amd.device import DeviceModel
    return DeviceModel.get("reacher_7dof")


def _p(dm, K, H, dtype="f32", **kw):
    from trajopt_amd.device import DevicePlanner
    kw.setdefault("kappa", 25.0)
    return DevicePlanner(dm, K, H, dtype=dtype, sigma=FILTER[0], betas=FILTER[1:], **kw)


def _applied(base, eps, dtype):
    """base + eps in the rollouts' type."""
    t = np.float32 if dtype == "f32" else np.float64
    return (base.astype(t) + eps.astype(t)).astype(np.float64)


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("K", [1, 40, 300, 4096, 40000])
def test_draw_applies_one_sample(dm, dtype, K):
    H = 5
    rng = np.random.RandomState(K)
    raw, base = rng.normal(size=(K, H, 7)), rng.normal(size=(H, 7)) * 0.2
    eps = ref_mppi.filter_noise(raw.copy(), FILTER)
    p = _p(dm, K, H, dtype, kappa=2.0)
    for f in (dict(), dict(top_k=10), dict(top_p=0.5), dict(top_k=64, top_p=0.9, min_p=0.05)):
        u = rng.uniform()
        p.set_start_state(np.full(7, -0.1), np.zeros(7), np.zeros(3), 0)
        p.set_base_actions(base)
        p.upload_noise(raw)
        p.draw(u, **f)
        k, w = p.drawn()
        R = p.returns()
        want_k, want_w = ref_learn.draw(R, [u], 2.0, **f)
        assert k == want_k[0] and abs(w - want_w[0]) <= WEIGHT_RTOL * want_w[0]
        assert np.array_equal(p.act_sequence(), _applied(base, eps[k], dtype))
    # the drawn sequence is the base of the next rollouts
    seq = p.act_sequence()
    p.rollout()
    again = _p(dm, K, H, dtype, kappa=2.0)
    again.set_start_state(np.full(7, -0.1), np.zeros(7), np.zeros(3), 0)
    again.set_base_actions(seq)
    again.upload_noise(raw)
    again.rollout()
    assert np.array_equal(p.returns(), again.returns())
    p.close()
    again.close()


@pytest.mark.parametrize("dtype", ["f32", "f64"])
def test_batched_planners_draw_each_for_itself(dm, dtype):
    P, K, H = 5, 200, 4
    rng = np.random.RandomState(3)
    raw, base, u = rng.normal(size=(P, K, H, 7)), rng.normal(size=(P, H, 7)) * 0.2, rng.uniform(size=P)
    p = _p(dm, K, H, dtype, kappa=1.0, planners=P)
    qp = rng.uniform(-0.3, 0.0, size=(P, 7))
    qp[3] = np.nan                                            # every rollout of this one diverges
    p.set_start_state(qp, np.zeros((P, 7)), np.zeros((P, 3)), 0)
    p.set_base_actions(base)
    p.upload_noise(raw)
    p.draw(u, top_k=50, top_p=0.8)
    k, w = p.drawn()
    R, seq = p.returns(), p.act_sequence()
    for b in range(P):
        want_k, want_w = ref_learn.draw(R[b], [u[b]], 1.0, 50, 0.8)
        assert k[b] == want_k[0] and abs(w[b] - want_w[0]) <= WEIGHT_RTOL * max(want_w[0], 1e-30)
        if b == 3:
            assert k[b] == -1 and w[b] == 0 and np.array_equal(seq[b], base[b])      # left as it was
        else:
            assert np.array_equal(seq[b], _applied(base[b], ref_mppi.filter_noise(raw[b].copy(), FILTER)[k[b]], dtype))
    p.close()


def test_draw_of_explicit_actions_and_between_iterations(dm):
    K, H = 64, 6
    rng = np.random.RandomState(4)
    act = rng.normal(size=(K, H, 7))
    p = _p(dm, K, H, "f64", kappa=0.5)
    p.set_start_state(np.zeros(7), np.zeros(7), np.zeros(3), 0)
    p.upload_actions(act)
    p.draw(0.4)
    k, _ = p.drawn()
    assert k == ref_learn.draw(p.returns(), [0.4], 0.5)[0][0] and np.array_equal(p.act_sequence(), act[k])
    # iterate, draw, iterate again: the captured iteration goes on from the drawn sequence
    raw = rng.normal(size=(K, H, 7))
    eps = ref_mppi.filter_noise(raw.copy(), FILTER)
    p.upload_noise(raw)
    p.iterate(1)
    base = p.act_sequence()
    p.draw(0.7, top_k=5)
    k, _ = p.drawn()
    assert np.array_equal(p.act_sequence(), base + eps[k])
    p.iterate(1)
    R = p.returns()
    assert np.abs(p.act_sequence() - ref_mppi.update(base + eps[k] + eps, R, 0.5)).max() < 1e-12
    p.close()


def test_draws_with_a_critic_and_from_several_host_threads(dm):
    """The critic's values belong to the returns that a draw weighs; planners of their own in threads of their own draw while others
    capture their graphs, and give what they give one after the other."""
    import threading
    rng = np.random.RandomState(2)
    W = [rng.normal(size=s).astype(np.float32) * 0.3 for s in ((128, 14), (128,), (128, 128), (128,), (1, 128), (1,))]
    u = rng.uniform(size=(4, 6))

    def run(i, out):
        K, H, dtype = [(700, 6, "f32"), (64, 9, "f64"), (4096, 5, "f32"), (40000, 4, "f32")][i]
        seen = []
        for life in range(2):
            p = _p(dm, K, H, dtype, kappa=3.0)
            p.set_start_state(np.full(7, 0.1 * i), np.zeros(7), np.array([0.1, 0.0, 0.1]), 0)
            p.set_base_actions(np.zeros((H, 7)))
            if life == 0:
                p.set_critic(14, W)
            for t in range(6):
                p.generate_noise(5 + t)
                p.iterate(t % 3)
                p.draw(u[i, t], top_k=(0, 20)[t % 2], top_p=(1.0, 0.8)[t % 2])
                k, w = p.drawn()
                R = p.returns()
                want_k, want_w = ref_learn.draw(R, [u[i, t]], 3.0, top_k=(0, 20)[t % 2], top_p=(1.0, 0.8)[t % 2])
                assert k == want_k[0] and abs(w - want_w[0]) <= WEIGHT_RTOL * want_w[0]
                seen.append(np.r_[p.act_sequence().ravel(), R])
                p.advance()
            p.close()
        out[i] = seen

    serial, threaded = {}, {}
    for i in range(4):
        run(i, serial)
    assert not np.array_equal(serial[0][0], serial[0][6])          # with and without the critic
    threads = [threading.Thread(target=run, args=(i, threaded)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(4):
        assert i in threaded and all(np.array_equal(a, b) for a, b in zip(serial[i], threaded[i])), i


def test_draw_refusals(dm):
    from trajopt_amd._lib import MppiError
    p = _p(dm, 16, 3)
    p.set_start_state(np.zeros(7), np.zeros(7), np.zeros(3), 0)
    p.generate_noise(1)
    with pytest.raises(MppiError):
        p.drawn()                                             # nothing drawn yet
    seq = p.act_sequence()
    for bad in (dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.1), dict(min_p=-0.1), dict(min_p=2.0), dict(top_p=float("nan"))):
        with pytest.raises(MppiError):
            p.draw(0.5, **bad)
    with pytest.raises(TypeError):
        p.draw(0.5, top_k=2.5)
    with pytest.raises(ValueError):
        p.draw([0.5, 0.5])
    assert np.array_equal(p.act_sequence(), seq)
    p.close()
    p = _p(dm, 16, 3, k_offset=16)                            # a shard: its samples are not all there are
    p.set_start_state(np.zeros(7), np.zeros(7), np.zeros(3), 0)
    p.generate_noise(1)
    with pytest.raises(MppiError):
        p.draw(0.5)
    p.close()
    p = _p(dm, 16, 3, reward_type="tracking")                 # no reference
    with pytest.raises(MppiError):
        p.draw(0.5)
    p.close()


def test_a_failed_draw_has_no_outcome(dm):
    """A draw on a capturing stream fails (it has to wait for the stream) behind its allocations: there is nothing to be read then, and
    the next one is as if it had been the first."""
    import ctypes
    from trajopt_amd import _lib as L
    hip = L.lib()                                             # (the runtime's functions through the library that links it)
    outcome = []
    for fails in (False, True):
        p = _p(dm, 64, 4, "f64", kappa=2.0)
        p.set_start_state(np.zeros(7), np.zeros(7), np.zeros(3), 0)
        p.set_base_actions(np.zeros((4, 7)))
        p.generate_noise(1)
        p.rollout()
        p.synchronize()
        if fails:
            s, g = ctypes.c_void_p(), ctypes.c_void_p()
            assert hip.hipStreamCreate(ctypes.byref(s)) == 0 and hip.hipStreamBeginCapture(s, 2) == 0
            with pytest.raises(L.MppiError, match="error -2"):
                p.draw(0.5, stream=s)
            hip.hipStreamEndCapture(s, ctypes.byref(g))       # (no capture is left: the wait has ended it)
            assert hip.hipStreamDestroy(s) == 0
            hip.hipGetLastError()
            with pytest.raises(L.MppiError, match="no draw"):
                p.drawn()
        p.draw(0.5)
        outcome.append((p.drawn(), p.act_sequence()))
        with pytest.raises(L.MppiError):
            p.draw(0.5, top_p=2.0)                            # a refused draw leaves the last one's outcome
        assert p.drawn() == outcome[-1][0]
        p.close()
    assert outcome[0][0] == outcome[1][0] and np.array_equal(outcome[0][1], outcome[1][1])


def test_no_shard_draws(dm):
    """The first shard of a caller-made exchange has offset 0 like a whole planner; that its statistics go out tells it from one."""
    import torch
    from trajopt_amd._lib import MppiError
    K, H = 64, 4
    shards = [_p(dm, K, H, "f64", k_offset=r * K) for r in range(2)]
    for s in shards:
        s.set_start_state(np.zeros(7), np.zeros(7), np.zeros(3), 0)
        s.set_base_actions(np.zeros((H, 7)))
        s.generate_noise(3)
    for begin in (lambda p: p.partials_ptr(), lambda p: p.local_partials()):
        for s in shards:
            begin(s)
            with pytest.raises(MppiError, match="every sample"):
                s.draw(0.5)
            s.synchronize()
    gathered = torch.from_numpy(np.stack([s.partials() for s in shards])).cuda()
    torch.cuda.synchronize()
    for s in shards:
        s.merge(gathered.data_ptr(), 2)
        seq = s.act_sequence()
        with pytest.raises(MppiError, match="every sample"):
            s.draw(0.5)
        assert np.array_equal(s.act_sequence(), seq)
        s.close()
    # a world of one rank: the same calls, and all samples there are
    p = _p(dm, K, H, "f64")
    p.set_start_state(np.zeros(7), np.zeros(7), np.zeros(3), 0)
    p.set_base_actions(np.zeros((H, 7)))
    p.generate_noise(3)
    p.local_partials()
    p.merge(p.partials_ptr()[0], 1)
    p.draw(0.5)
    assert p.drawn()[0] == ref_learn.draw(p.returns(), [0.5], 25.0)[0][0]
    p.close()


def test_a_group_of_one_rank_draws(dm):
    """After mppi_comm_init with one rank the planner still owns every sample: drawn steps and iterations in turn, as without."""
    from trajopt_amd.device import DevicePlanner
    out = []
    for grouped in (False, True):
        p = _p(dm, 128, 5, "f64", kappa=2.0)
        p.set_start_state(np.zeros(7), np.zeros(7), np.zeros(3), 0)
        p.set_base_actions(np.zeros((5, 7)))
        if grouped:
            p.comm_init(DevicePlanner.comm_unique_id(), 0, 1)
        p.generate_noise(4)
        p.draw(0.3, top_k=30)
        first = p.drawn(), p.act_sequence()
        assert first[0][0] == ref_learn.draw(p.returns(), [0.3], 2.0, 30)[0][0]
        p.iterate(1)
        p.draw(0.8, top_p=0.7)
        out.append((first, p.drawn(), p.act_sequence()))
        p.close()
    for (a, b) in ((out[0][0], out[1][0]), (out[0][1:], out[1][1:])):
        assert a[0] == b[0] and np.array_equal(a[1], b[1])


def _agent(noise, dtype="f64", **kw):
    from trajopt.algos.mppi import MPPI
    from trajopt.envs.utils import get_environment
    e = get_environment('reacher_7dof')
    e.reset_model(seed=None, goal=(0.0, 0.0, 0.0))
    return MPPI(e, H=8, paths_per_cpu=50, num_cpu=1, kappa=5.0, gamma=1.0, mean=np.zeros(7), filter_coefs=FILTER, default_act='mean',
                seed=11, noise=noise, dtype=dtype, **kw)


@pytest.mark.parametrize("niter", [1, 3])
def test_train_step_with_a_draw(oracle_sim, niter):
    """Host noise, fp64: every step against the oracle -- niter - 1 updates, the draw from the device's returns, the
    real environment's step with the drawn sequence's first action."""
    ag = _agent('host')
    for t in range(6):
        s0, seq = ag.sol_state[-1], ag.act_sequence.copy()
        u = 0.05 + 0.15 * t
        np.random.seed(99)
        assert ag.train_step(niter=niter, draw=dict(u=u, top_k=20, top_p=0.9)) == []
        eps = ref_mppi.filter_noise(ref_mppi.all_raw_normals(11 + t, 50, 1, 8, 7), FILTER)
        for _ in range(niter - 1):
            R = oracle_sim.rollout(s0["qp"], s0["qv"], np.zeros(3), t, seq + eps)
            seq = ref_mppi.update(seq + eps, R, 5.0)
        R = oracle_sim.rollout(s0["qp"], s0["qv"], np.zeros(3), t, seq + eps)
        R_dev = ag._planner.returns()
        assert np.abs(R_dev - R).max() < 1e-8
        k, _ = ag._planner.drawn()
        assert k == ref_learn.draw(R_dev, [u], 5.0, 20, 0.9)[0][0]
        seq = seq + eps[k]
        q, v, _, r, _ = oracle_sim.env_step(s0["qp"], s0["qv"], np.zeros(3), seq[0], t)
        assert np.abs(ag.sol_state[-1]["qp"] - q).max() < 1e-8 and abs(ag.sol_reward[-1] - r) < 1e-8
        assert np.abs(ag.act_sequence - ref_mppi.shift(seq, "mean", np.zeros(7))).max() < 1e-8


@pytest.mark.parametrize("noise", ["host", "philox"])
def test_drawn_steps_leave_the_other_steps_alone(noise):
    """Drawn and ordinary steps in turn; a twin that sends its state again before every step does the same; and a step
    without a draw equals the one of an agent that has never heard of draws."""
    a, b = _agent(noise), _agent(noise)
    for t in range(8):
        draw = dict(top_k=10) if t % 3 == 1 else None
        a.train_step(niter=2, draw=draw)
        b._dev_state = b._dev_seq = None                     # everything is sent again
        b.train_step(niter=2, draw=draw)
        assert np.array_equal(a.act_sequence, b.act_sequence) and np.array_equal(a.sol_state[-1]["qp"], b.sol_state[-1]["qp"])
    c, d = _agent(noise), _agent(noise)
    for _ in range(3):
        c.train_step(niter=2)
        d.train_step(niter=2, draw=None)
    assert np.array_equal(c.act_sequence, d.act_sequence)


def test_train_step_draw_refusals():
    ag = _agent('philox')
    with pytest.raises(ValueError):
        ag.train_step(draw=dict(topk=3))
    with pytest.raises(ValueError):
        ag.train_step(niter=0, draw=dict(top_k=3))
    with pytest.raises(ValueError):
        ag.train_step(critic=lambda x: x[:, :1], draw=dict(top_k=3))      # rollouts scored on the host
    assert len(ag.sol_state) == 1
    u = [ag._draw_arguments({}, 5, 1)["u"], ag._draw_arguments({}, 5, 1)["u"], ag._draw_arguments({}, 6, 1)["u"]]
    assert u[0] == u[1] != u[2] and 0.0 <= u[0] < 1.0


BAD_DRAWS = [dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.5), dict(top_p=float("nan")), dict(min_p=-0.1), dict(min_p=2.0), dict(u=[0.1, 0.2]),
             dict(u=[]), dict(u=float("nan")), dict(u=float("inf")), dict(u="x"), dict(top_k=2.5), dict(top_k="x"), dict(min_p=None), dict(topk=3)]


@pytest.mark.parametrize("noise", ["host", "philox"])
def test_a_refused_drawn_step_changes_nothing(noise):
    """Every refusal of train_step(draw=...) comes before noise, numpy's generator, act_sequence or the device is touched: an agent with
    refused calls between its steps goes on as one without."""
    from trajopt_amd._lib import MppiError
    a, b = _agent(noise), _agent(noise)
    for t in range(3):
        for ag in (a, b):
            np.random.seed(5)
            ag.train_step(niter=2, draw=dict(top_k=10) if t == 1 else None)
        np.random.seed(77)
        before = np.random.get_state()[1].copy()
        seq, ahead, device = a.act_sequence.copy(), a._ahead, a._planner.act_sequence()
        for bad in BAD_DRAWS:
            with pytest.raises((MppiError, ValueError, TypeError)):
                a.train_step(niter=2, draw=bad)
        a.kappa = -1.0                                         # an update takes it, a draw does not
        with pytest.raises(MppiError):
            a.train_step(niter=2, draw={})
        a.kappa = b.kappa
        assert np.array_equal(np.random.get_state()[1], before) and a._ahead is ahead and len(a.sol_state) == t + 2
        assert np.array_equal(a.act_sequence, seq) and np.array_equal(a._planner.act_sequence(), device)
    for ag in (a, b):
        ag.train_step(niter=2, draw=dict(u=np.array([0.25]), min_p=0.01))
    assert np.array_equal(a.act_sequence, b.act_sequence) and np.array_equal(a.sol_state[-1]["qp"], b.sol_state[-1]["qp"])


def test_critic_gradients_clipped_on_the_way_to_the_optimizer():
    """A temporal-difference step of the critic on the GPU: gradients against differences of the loss, their norm and the
    clipped values against the definition, and the step an SGD makes with them."""
    import torch
    from trajopt.models.critic_nets import Critic
    torch.manual_seed(1)
    critic = Critic(input_dim=14, inner_layer=128).cuda()
    gen = torch.Generator().manual_seed(2)
    x, y = torch.randn(64, 14, generator=gen).cuda(), (100.0 * torch.randn(64, 1, generator=gen)).cuda()
    loss = torch.nn.functional.mse_loss(critic(x), y)
    loss.backward()
    grads = [p.grad.double().cpu().numpy() for p in critic.parameters()]
    # central differences in float64 of the same network, along each parameter's own gradient
    twin = Critic(input_dim=14, inner_layer=128).double()
    twin.load_state_dict({k: v.double().cpu() for k, v in critic.state_dict().items()})
    for p, g in zip(twin.parameters(), grads):
        direction = torch.tensor(g / np.linalg.norm(g))
        h, values = 1e-5, []
        for sign in (1.0, -1.0):
            with torch.no_grad():
                p.add_(sign * h * direction)
                values.append(float(torch.nn.functional.mse_loss(twin(x.double().cpu()), y.double().cpu())))
                p.sub_(sign * h * direction)
        slope = (values[0] - values[1]) / (2 * h)
        # fp32 backward: a few hundred roundings of 2^-24 in sums over 64 samples and 128 units; differences: h^2 of a smooth loss
        assert abs(slope - np.linalg.norm(g)) < 1e-4 * np.linalg.norm(g) + 1e-6
    want_norm, want = ref_learn.clip(grads, 1.0)
    assert want_norm > 1.0
    norm = critic.clip_gradients(1.0)
    assert abs(float(norm) - want_norm) <= (2.0 ** -24 + 1e-12) * want_norm
    before = [p.detach().clone() for p in critic.parameters()]
    for p, w in zip(critic.parameters(), want):
        got = p.grad.double().cpu().numpy()
        assert np.all(np.abs(got - w) <= 2.0 ** -24 * 1.0000001 * np.abs(w) + 2.0 ** -150)
    torch.optim.SGD(critic.parameters(), lr=0.5).step()
    moved = np.sqrt(sum(float(((p.detach() - b).double() ** 2).sum()) for p, b in zip(critic.parameters(), before)))
    # a step of length 0.5: each of 18 561 entries rounds by up to 2^-25 of a parameter below 1
    assert abs(moved - 0.5) < np.sqrt(18561) * 2.0 ** -24
    with pytest.raises(ValueError):
        Critic().clip_gradients(1.0)                          # no gradients yet
    cpu = Critic()
    cpu(torch.zeros(1, 14)).sum().backward()
    with pytest.raises(TypeError):
        cpu.clip_gradients(1.0)                               # there is no CPU form


def test_clipping_tells_autograd_that_it_wrote():
    """Values saved for a backward pass and then clipped in place are noticed, as with any in-place operation of torch."""
    import torch
    from trajopt_amd.device import clip_gradients
    x = torch.randn(50, device="cuda", requires_grad=True)
    y = x * 2.0
    z = (y * y).sum()
    clip_gradients([y.detach()], 1e-3)
    with pytest.raises(RuntimeError):
        z.backward()


def test_no_graph_is_dropped_in_silence():
    """Autograd's tensors are refused while it records and taken while it does not; nothing is written by a refused call, and
    tensors that stand for others (vmap, forward mode, without memory) are refused as well."""
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode
    from trajopt_amd.device import clip_gradients, draw_from_returns, gradient_norm
    leaf = torch.randn(40, device="cuda", requires_grad=True)
    u = torch.tensor([0.1, 0.9], device="cuda", dtype=torch.float64)
    keep, plain = leaf.detach().clone(), torch.ones(40, device="cuda")
    for call in (lambda: draw_from_returns(leaf, u), lambda: gradient_norm([leaf]), lambda: clip_gradients([leaf * 1.0], 0.1),
                 lambda: clip_gradients([leaf], 0.1), lambda: clip_gradients([plain], 0.1, out=[leaf])):
        with pytest.raises(RuntimeError, match="no derivative"):
            call()
    assert torch.equal(leaf, keep) and (plain == 1).all()
    with torch.no_grad():
        a, b = draw_from_returns(leaf, u), draw_from_returns(keep, u)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and not a[1].requires_grad
        assert torch.equal(gradient_norm([leaf]), gradient_norm([keep]))
        version = leaf._version
        clip_gradients([leaf], 0.1)
        clip_gradients([keep], 0.1)
        assert torch.equal(leaf, keep) and leaf._version > version
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(plain, torch.ones_like(plain))
        for call in (lambda: draw_from_returns(dual, u), lambda: gradient_norm([dual]), lambda: clip_gradients([dual], 0.1)):
            with pytest.raises(RuntimeError, match="no derivative"):
                call()
    for call in (lambda x: draw_from_returns(x, u)[1], lambda x: gradient_norm([x]), lambda x: clip_gradients([x], 0.1)):
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(plain.reshape(4, 10))
        with pytest.raises(RuntimeError), FakeTensorMode():
            call(torch.ones(40, device="cuda"))
    assert (plain == 1).all()


def test_critic_clips_gradients_that_have_a_graph_of_their_own():
    import torch
    from trajopt.models.critic_nets import Critic
    torch.manual_seed(3)
    critic = Critic(input_dim=14, inner_layer=128).cuda()
    (critic(torch.randn(8, 14, device="cuda")) ** 2).sum().backward(create_graph=True)
    grads = [p.grad for p in critic.parameters()]
    assert any(g.requires_grad for g in grads)
    want_norm, want = ref_learn.clip([g.detach().double().cpu().numpy() for g in grads], 0.01)
    assert want_norm > 0.01
    norm = critic.clip_gradients(0.01)
    assert not norm.requires_grad and abs(float(norm) - want_norm) <= (2.0 ** -24 + 1e-12) * want_norm
    for g, w in zip(grads, want):
        assert np.all(np.abs(g.detach().double().cpu().numpy() - w) <= 2.0 ** -24 * 1.0000001 * np.abs(w) + 2.0 ** -150)
    for p in critic.parameters():
        p.grad = None                                         # (a graph that holds its own leaves)


def test_epochs_of_drawn_steps_and_clipped_training():
    """The whole loop: drawn steps fill the replay buffer, the critic trains on the GPU with clipped gradients, the next
    epoch's rollouts end in the trained critic's value."""
    import torch
    from trajopt.models.critic_nets import Critic
    from trajopt.utils import ReplayBuffer
    torch.manual_seed(0)
    critic = Critic(num_iters=8, input_dim=14, inner_layer=128, batch_size=16, gamma=0.9).cuda()
    optimizer = torch.optim.Adam(critic.parameters(), lr=1e-2)
    replay = ReplayBuffer(max_size=1000)
    for epoch in range(2):
        ag = _agent('philox', 'f32')
        for _ in range(12):
            ag.train_step(critic=critic, niter=2, goal=np.zeros(3), dim=14, draw=dict(top_k=8, top_p=0.9))
            k, w = ag._planner.drawn()
            R = ag._planner.returns()
            assert 0 <= k < 50 and R[k] >= np.sort(R)[-8] and 0 < w <= 1
        samples = critic.compress_agent(ag, dim=14)
        assert len(samples) == 12
        replay.concatenate(samples)
        before = critic.linear2.weight.detach().clone()
        for _ in range(critic.num_iters):
            batch = replay.get_minibatch(size=min(critic.batch_size, len(replay.buffer)))
            state = torch.tensor(np.array([d.state for d in batch]), dtype=torch.float32, device="cuda")
            reward = torch.tensor([float(d.reward) for d in batch], dtype=torch.float32, device="cuda").unsqueeze(1)
            loss = torch.nn.functional.mse_loss(critic(state), reward)
            optimizer.zero_grad()
            loss.backward()
            raw = [p.grad.double().cpu().numpy() for p in critic.parameters()]
            want_norm, want = ref_learn.clip(raw, 0.5)
            norm = critic.clip_gradients(0.5)
            assert abs(float(norm) - want_norm) <= (2.0 ** -24 + 1e-12) * want_norm
            for p, w in zip(critic.parameters(), want):
                assert np.all(np.abs(p.grad.double().cpu().numpy() - w) <= 2.0 ** -24 * 1.0000001 * np.abs(w) + 2.0 ** -150)
            optimizer.step()
        assert not torch.equal(before, critic.linear2.weight.detach())


def test_example_actor_critic_script_with_draws_and_clipping():
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "actor_critic_reacher.py")
    spec = importlib.util.spec_from_file_location("actor_critic_reacher", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    results = mod.main(["--epochs", "2", "--steps", "20", "--iters", "10", "--draw", "8", "--device", "cuda", "--clip", "1.0"])
    assert len(results) == 2 and all(np.isfinite(r[3]) for r in results)
    with pytest.raises(SystemExit):
        mod.main(["--clip", "1.0"])


def test_results_in_inference_mode():
    """Tensors made inside are inference tensors, tensors made outside are not, and either kind may be clipped or drawn from."""
    import torch
    from trajopt_amd.device import clip_gradients, draw_from_returns
    R, u, g = torch.randn(2, 9, device="cuda"), torch.rand(2, 3, device="cuda", dtype=torch.float64), torch.ones(16, device="cuda")
    want = draw_from_returns(R, u)
    assert not want[0].is_inference() and not want[1].requires_grad
    with torch.inference_mode():
        got = draw_from_returns(R + 0.0, u)
        norm = clip_gradients([g * 1.0], 1.0)
        clip_gradients([g], 2.0)
    assert got[0].is_inference() and norm.is_inference() and float(norm) == 4.0
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert (g == 0.5).all()

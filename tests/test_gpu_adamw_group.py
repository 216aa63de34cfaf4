"""GPU: pde_amd.optim.GroupedAdamW, grad_norm and clip_grad_norm_ against float64 numpy (adamw_formulas.py).

Tolerances, with h = 2^-24 the half step of float32.  m: g - m, 1 - b1, their product and the sum are rounded once each, a
clipped g twice more: |dm| <= h (|m'| + 4 (1 - b1) (|g| + |m|)).  v: both of its terms are positive and take at most 6
roundings each, the sum one: |dv| <= 8 h v'.  p: the decayed weight takes 2 roundings, the sum one, the update U takes dm / m, half of
dv / v and at most 10 more: |dp| <= h (|p'| + 2 |p| + 16 |U|) + step |dm| / denom.  A 16-bit weight adds half its own step,
finfo.eps / 2 of its value (of a float16 below 2^-14: half of 2^-24).  8-bit moments are formed in float64 from exactly decoded ones: they
have to be equal.  The norm: float64 sums, one rounding to float32."""
import numpy as np
import pytest
import torch

import adamw_formulas as F
from pde_amd._native import _cur_stream, load_library
from pde_amd.optim import FusedAdam, GroupedAdamW, clip_grad_norm_, grad_norm

pytestmark = pytest.mark.gpu
H = 2.0 ** -24
HYPER = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2)
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SIZES = [(1,), (3, 5), (0,), (127,), (128,), (129,), (2047,), (2048,), (2049,), (70, 61), (8192,), (12345,)]


def cuda():
    return torch.device("cuda", 0)


def make(sizes, dtype, seed, scale=1.0):
    rng = np.random.default_rng(seed)
    return [torch.tensor(scale * rng.standard_normal(s), dtype=torch.float32).to(dtype).to(cuda()) for s in sizes]


def params_of(tensors):
    return [torch.nn.Parameter(t) for t in tensors]


def f64(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def half_step(dtype, x):
    if dtype == torch.float32:
        return 0.0
    return np.maximum(torch.finfo(dtype).eps / 2 * np.abs(x), 2.0 ** -25 if dtype == torch.float16 else 0.0)


class Oracle:
    """The same optimizer in float64: holds what the float32 (or 8-bit) state holds after each step."""

    def __init__(self, opt):
        self.opt, self.t = opt, [0] * len(opt._params)
        self.p = [f64(p) for p in opt._params]
        self.m = [np.zeros(p.numel()) for p in opt._params]
        self.v = [np.zeros(p.numel()) for p in opt._params]

    def step(self, grads, check=True):
        """grads: flat float64 arrays or None, before opt.step() has been taken; returns nothing, compares what the step left"""
        opt = self.opt
        factor = 1.0
        if opt.max_norm is not None:
            norm, factor = F.clip_factor([g for g in grads if g is not None], opt.max_norm)
            assert abs(float(opt.grad_norm) - norm) <= 2 * H * norm
        ms, vs = (f64(x) for x in opt.moments())
        i = 0
        for grp in opt.param_groups:
            for p in grp["params"]:
                self.one(i, p, grads[i], factor, grp, ms, vs)
                i += 1

    def one(self, i, p, g, factor, grp, ms, vs):
        opt, at = self.opt, self.opt.offsets[i]
        gm, gv = ms[at:at + p.numel()], vs[at:at + p.numel()]
        pad = slice(at + p.numel(), at + -(-p.numel() // F.BLOCK) * F.BLOCK)
        assert not ms[pad].any() and not vs[pad].any()
        got = f64(p) if opt.master is None or p.dtype == torch.float32 else f64(opt.master[at:at + p.numel()])
        if g is None:
            assert np.array_equal(got, self.p[i]) and np.array_equal(gm, self.m[i]) and np.array_equal(gv, self.v[i])
            return
        self.t[i] += 1
        b1, b2 = grp["betas"]
        lr, eps, wd, t = grp["lr"], grp["eps"], grp["weight_decay"], self.t[i]
        g = g * factor
        p1, m1, v1 = F.step(self.p[i], g, self.m[i], self.v[i], t, lr, b1, b2, eps, wd)
        bad = ~np.isfinite(p1)
        assert np.array_equal(bad, ~np.isfinite(got)), i
        dm = H * (np.abs(m1) + 4 * (1 - b1) * (np.abs(g) + np.abs(self.m[i])))
        per_m = lr / (1 - b1 ** t) / (np.sqrt(v1 / (1 - b2 ** t)) + eps)
        tol = H * (np.abs(p1) + 2 * np.abs(self.p[i]) + 16 * per_m * np.abs(m1)) + per_m * dm
        if opt.master is None or p.dtype == torch.float32:
            tol = tol + half_step(p.dtype, p1)
        else:                                                          # the 16-bit weights are the master's, rounded once
            assert torch.equal(p.detach().reshape(-1), opt.master[at:at + p.numel()].to(p.dtype))
        ok = ~bad
        assert (np.abs(got - p1)[ok] <= tol[ok]).all(), (i, np.max((np.abs(got - p1) / tol)[ok]))
        if opt.state_bits == 32:
            assert (np.abs(gm - m1)[ok] <= dm[ok]).all() and (np.abs(gv - v1)[ok] <= 8 * H * v1[ok]).all(), i
        else:
            m1, sm = F.round_flat(m1, at, t, F.M)
            v1, sv = F.round_flat(v1, at, t, F.V)
            blk = slice(at // F.BLOCK, at // F.BLOCK + len(sm))
            assert np.array_equal(opt.exp_avg_scale[blk].cpu().numpy(), sm) and np.array_equal(opt.exp_avg_sq_scale[blk].cpu().numpy(), sv), i
            assert np.array_equal(gm, m1, equal_nan=True) and np.array_equal(gv, v1, equal_nan=True), i
        self.p[i], self.m[i], self.v[i] = got, gm, gv
        assert opt.device_state[i].tolist()[0] == (t if p.numel() else 0)      # an empty parameter is in no launch


def run(opt, n_steps, seed, none_every=0):
    params = opt._params
    oracle = Oracle(opt)
    for k in range(n_steps):
        grads = make([tuple(p.shape) for p in params], torch.float32, seed + k, 0.3 / (k + 1))
        for i, p in enumerate(params):
            p.grad = None if none_every and (i + k) % none_every == 0 else torch.empty_like(p).copy_(grads[i])
        opt.step()
        flat = [None if p.grad is None else f64(torch.as_strided(p.grad, (p.numel(),), (1,))) for p in params]
        oracle.step(flat)
    return oracle


@pytest.mark.parametrize("clip", [None, 0.5, 1e6])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, False), (torch.bfloat16, True), (torch.float16, False), (torch.float16, True)])
def test_steps(dtype, master, bits, clip):
    params = params_of(make(SIZES, dtype, 1, 0.5))
    run(GroupedAdamW(params, state_bits=bits, master_weights=master, max_norm=clip, **HYPER), 3, 100)


@pytest.mark.parametrize("bits", [32, 8])
def test_missing_gradients_keep_their_own_count(bits):
    params = params_of(make(SIZES, torch.float32, 2, 0.5))
    opt = GroupedAdamW(params, state_bits=bits, max_norm=1.0, **HYPER)
    run(opt, 4, 200, none_every=3)
    assert len({tuple(r) for r in opt.device_state[:, :1].tolist()}) > 1


@pytest.mark.parametrize("bits", [32, 8])
def test_groups_types_and_more_tensors_than_one_launch_takes(bits):
    sizes = [(1 + 7 * i % 300,) for i in range(260)]
    a, b = params_of(make(sizes, torch.float32, 3)), params_of(make(SIZES, torch.bfloat16, 4))
    c = params_of(make(SIZES, torch.float16, 5) + make(SIZES, torch.float32, 6))
    opt = GroupedAdamW([dict(params=a), dict(params=b, lr=1e-3, weight_decay=0.0), dict(params=c, betas=(0.8, 0.95), eps=1e-6)],
                       state_bits=bits, master_weights=True, max_norm=3.0, **HYPER)
    assert len(opt._launches) == 5
    run(opt, 2, 300, none_every=7)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_unaligned_and_permuted_tensors(dtype, bits):
    flat = make([(9000,)], dtype, 7)[0]
    params = params_of([flat[1:1 + 513], flat[515:515 + 2050], flat[3001:3001 + 1]]) + params_of([make([(33, 65)], dtype, 8)[0].t(),
                                                                                                   make([(4, 6, 10)], dtype, 9)[0].permute(2, 0, 1)])
    before = flat.clone()
    opt = GroupedAdamW(params, state_bits=bits, **HYPER)
    oracle = Oracle(opt)
    oracle.p = [f64(torch.as_strided(p, (p.numel(),), (1,), p.storage_offset())) for p in params]
    for k in range(2):
        gflat = make([(9000,)], dtype, 70 + k)[0]
        params[0].grad, params[1].grad, params[2].grad = gflat[3:3 + 513], gflat[600:600 + 2050], gflat[5:6]
        params[3].grad = make([(65, 33)], dtype, 80 + k)[0]                     # contiguous, its parameter is not: another order
        params[4].grad = torch.empty_like(params[4]).copy_(make([(10, 4, 6)], dtype, 90 + k)[0])
        opt.step()
        order = [f64(g) for g in (params[0].grad, params[1].grad, params[2].grad, params[3].grad.t())]
        order.append(f64(torch.as_strided(params[4].grad, (240,), (1,))))
        ms, vs = (f64(x) for x in opt.moments())
        saved = params[3], params[4]
        for i, p in enumerate(params):
            view = torch.as_strided(p.detach(), (p.numel(),), (1,), p.storage_offset())
            oracle.one(i, view, order[i], 1.0, opt.param_groups[0], ms, vs)
        assert saved[0].stride() == (1, 65)
    outside = torch.ones(9000, dtype=torch.bool)
    for a, n in ((1, 513), (515, 2050), (3001, 1)):
        outside[a:a + n] = False
    assert torch.equal(flat.cpu()[outside], before.cpu()[outside])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_not_finite(bits, bad):
    params = params_of(make([(300,), (40,)], torch.float32, 10))
    opt = GroupedAdamW(params, state_bits=bits, **HYPER)
    for p, g in zip(params, make([(300,), (40,)], torch.float32, 11)):
        p.grad = g
    params[0].grad[130] = bad
    opt.step()
    assert torch.isnan(params[0]).nonzero().flatten().tolist() == [130] and torch.isfinite(params[1]).all()
    m, v = opt.moments()
    if bits == 8:                                                              # the block 128 .. 255 is one scale
        assert torch.isnan(m).nonzero().flatten().tolist() == list(range(128, 256)) == torch.isnan(v).nonzero().flatten().tolist()
    else:
        assert (~torch.isfinite(m)).nonzero().flatten().tolist() == [130]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip", [None, 1.0])
def test_skip_nonfinite_leaves_everything(bits, clip):
    params = params_of(make(SIZES, torch.bfloat16, 12))
    opt = GroupedAdamW(params, state_bits=bits, max_norm=clip, skip_nonfinite=True, master_weights=True, **HYPER)
    run(opt, 1, 400)
    before = opt.state_dict()["fused"], [p.detach().clone() for p in params]
    for bad in (float("nan"), float("inf")):
        params[5].grad[7] = bad
        opt.step()
        assert not torch.isfinite(opt.grad_norm)
        after = opt.state_dict()["fused"]
        assert all(torch.equal(before[0][k], after[k]) for k in after)
        assert all(torch.equal(a, b.detach()) for a, b in zip(before[1], params))
    oracle = Oracle(opt)
    oracle.p = [f64(opt.master[at:at + p.numel()]) for p, at in zip(params, opt.offsets)]
    ms, vs = (f64(x) for x in opt.moments())
    oracle.m = [ms[at:at + p.numel()] for p, at in zip(params, opt.offsets)]
    oracle.v = [vs[at:at + p.numel()] for p, at in zip(params, opt.offsets)]
    oracle.t = [1] * len(params)
    for p, g in zip(params, make(SIZES, torch.bfloat16, 13)):
        p.grad = g
    opt.step()
    for i in range(len(params)):
        oracle.t[i] = 1
    grads = [f64(p.grad) for p in params]
    for i, p in enumerate(params):
        if p.numel() == 0:
            continue
        ms, vs = (f64(x) for x in opt.moments())
        factor = 1.0 if clip is None else F.clip_factor(grads, clip)[1]
        oracle.one(i, p, grads[i], factor, opt.param_groups[0], ms, vs)


@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e-18, 1e18])
def test_eight_bits_over_the_range_of_float32(scale):
    """tiny and huge gradients: v runs from below float32's smallest to beyond its largest, a moment that is not zero stays not zero"""
    params = params_of(make([(1000,)], torch.float32, 14))
    opt = GroupedAdamW(params, state_bits=8, **HYPER)
    oracle = Oracle(opt)
    for k in range(3):
        params[0].grad = make([(1000,)], torch.float32, 500 + k)[0].double().mul(scale).float()
        params[0].grad[::9] *= 1e-6
        params[0].grad[5] = 0.0
        opt.step()
        oracle.step([f64(params[0].grad)])
    m, v = opt.moments()
    if scale:
        assert v[0] > 0 and v[5] == 0 and m[5] == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_eight_bit_codes_on_their_borders(dtype):
    """Gradients chosen so that 0.9 m + 0.1 g lies on the border between two codes as the element's remainder is drawn, up to the last bits of
    float64: the formula, rounded operation by operation, says which way each goes, and every code has to follow it."""
    n, t, s0 = 1 << 16, 7, 110
    rng = np.random.default_rng(5)
    tab, unit = F.table(F.M), 2.0 ** (s0 - 127)
    i = np.arange(n, dtype=np.uint64)
    u = (((i * np.uint64(F.M["place"]) + np.uint64(t * F.M["step"] % 2 ** 32)) % np.uint64(2 ** 32)) >> np.uint64(15) | np.uint64(1)).astype(np.float64) / 2 ** 17
    old = rng.integers(8, 112, n) + 128 * rng.integers(0, 2, n)                # codes; the first of each block is the largest and sets the scale
    c = rng.integers(8, 104, n)
    target = (tab[c] + (1.0 - u) * (tab[c + 1] - tab[c])) * unit * rng.choice([-1.0, 1.0], n)
    old[::128], target[::128] = 120, 1.5 * 2.0 ** 8 * unit
    scales = np.full(n // 128, s0, dtype=np.uint8)
    m0 = F.values(old, scales, F.M)
    g = torch.tensor(10.0 * target - 9.0 * m0).to(dtype).to(cuda())
    p = torch.nn.Parameter(torch.zeros(n, dtype=dtype, device=cuda()))
    p.grad = g
    opt = GroupedAdamW([p], state_bits=8, lr=0.0, weight_decay=0.0)
    sd = opt.state_dict()
    sd["fused"]["exp_avg"].copy_(torch.tensor(old.astype(np.uint8)))
    sd["fused"]["exp_avg_scale"].fill_(s0)
    sd["fused"]["device_state"].copy_(torch.tensor([[t - 1.0, 0.9 ** (t - 1), 0.999 ** (t - 1)]], dtype=torch.float64))
    opt.load_state_dict(sd)
    opt.step()
    _, m1, v1 = F.step(np.zeros(n), f64(g), m0, np.zeros(n), t)
    if dtype == torch.float32:
        near = np.abs(np.abs(m1) / np.abs(target) - 1.0) < 2.0 ** -49
        assert near.mean() > 0.2 and (np.abs(m1) < np.abs(target))[near].any() and (np.abs(m1) >= np.abs(target))[near].any()
    ms, vs = opt.moments()
    assert np.array_equal(f64(ms), F.round_flat(m1, 0, t, F.M)[0]) and np.array_equal(f64(vs), F.round_flat(v1, 0, t, F.V)[0])


def test_small_changes_are_not_lost_in_eight_bits():
    """b2 = 0.999: g^2 is 30 times v, so v grows by 3 % a step, less than half a code (6 %); rounding to nearest would stop it.  After n
    steps v is 1 + 29 (1 - 0.999^n) times what it was; a code is 12.5 % wide and the error of a step is below one code, kept from adding up by the
    even sequence: the mean over 4096 elements within 5 % (over 4096 independent errors of one code each it would be 0.2 %)."""
    params = params_of([torch.zeros(4096, device=cuda())])
    opt = GroupedAdamW(params, state_bits=8, lr=0.0, weight_decay=0.0)
    sd = opt.state_dict()
    sd["fused"]["exp_avg_sq"].fill_((15 + 0) << 3)                             # 1.0 * 2^0
    sd["fused"]["exp_avg_sq_scale"].fill_(127)
    sd["fused"]["device_state"].copy_(torch.tensor([[1000.0, 0.9 ** 1000, 0.999 ** 1000]], dtype=torch.float64))
    opt.load_state_dict(sd)
    params[0].grad = torch.full((4096,), 30.0 ** 0.5, device=cuda())
    for n in range(1, 201):
        opt.step()
        if n in (10, 50, 200):
            want = 1 + 29 * (1 - 0.999 ** n)
            got = float(opt.moments()[1].double().mean())
            assert abs(got / want - 1) < 0.05, (n, got, want)


@pytest.mark.parametrize("clip", [None, 0.7])
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_replays_like_the_eager_one(bits, clip):
    def model():
        params = params_of(make(SIZES, torch.bfloat16, 20))
        opt = GroupedAdamW(params, state_bits=bits, max_norm=clip, master_weights=True, **HYPER)
        for p, g in zip(params, make(SIZES, torch.bfloat16, 21)):
            p.grad = g
        return params, opt
    pa, a = model()
    pb, b = model()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()
    torch.cuda.current_stream().wait_stream(side)
    b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for k in range(4):
        for p, q, g in zip(pa, pb, make(SIZES, torch.bfloat16, 30 + k)):
            p.grad.copy_(g)
            q.grad.copy_(g)
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        sa, sb = a.state_dict()["fused"], b.state_dict()["fused"]
        assert all(torch.equal(sa[n], sb[n]) for n in sa) and all(torch.equal(x, y) for x, y in zip(pa, pb))
        if clip:
            assert torch.equal(a.grad_norm, b.grad_norm)


def test_two_captured_clippings_on_two_streams():
    """each has a workspace of its own"""
    sets, graphs, norms = [], [], []
    for k in range(2):
        params = params_of(make(SIZES, torch.float32, 40 + k))
        for p, g in zip(params, make(SIZES, torch.float32, 42 + k, 3.0)):
            p.grad = g
        clip_grad_norm_(params, 1e9)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norms.append(clip_grad_norm_(params, 1.0))
        sets.append(params)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for r in range(3):
        fresh = [make(SIZES, torch.float32, 50 + 2 * r + k, 3.0) for k in range(2)]
        for params, grads in zip(sets, fresh):
            for p, g in zip(params, grads):
                p.grad.copy_(g)
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for params, grads, norm in zip(sets, fresh, norms):
            want = grad_norm(grads)
            assert torch.equal(norm, want)
            assert abs(float(grad_norm([p.grad for p in params])) - 1.0) < 1e-5


@pytest.mark.parametrize("bits", [32, 8])
def test_two_optimizers_at_once(bits):
    """each on a stream of its own, clipped: nothing is shared between them"""
    def model(k):
        params = params_of(make(SIZES + [(300000,)], torch.float32, 130 + k))
        for p, g in zip(params, make(SIZES + [(300000,)], torch.float32, 140 + k)):
            p.grad = g
        return params, GroupedAdamW(params, state_bits=bits, max_norm=0.5 + k, **HYPER)
    alone, together = [model(k) for k in range(2)], [model(k) for k in range(2)]
    for _, opt in alone:
        for _ in range(5):
            opt.step()
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for (_, opt), st in zip(together, streams):
            with torch.cuda.stream(st):
                opt.step()
    torch.cuda.synchronize()
    for (pa, a), (pb, b) in zip(alone, together):
        sa, sb = a.state_dict()["fused"], b.state_dict()["fused"]
        assert all(torch.equal(sa[n], sb[n]) for n in sa) and all(torch.equal(x, y) for x, y in zip(pa, pb))
        assert torch.equal(a.grad_norm, b.grad_norm) and not a._ticket.any() and not b._ticket.any()


def test_scalars_and_empty_parameters_and_none_without_gradients():
    params = params_of([torch.tensor(0.5, device=cuda()), torch.empty(0, 3, device=cuda()), torch.ones(2, device=cuda())])
    opt = GroupedAdamW(params, max_norm=1.0, **HYPER)
    before = opt.state_dict()["fused"]
    opt.step()                                                                 # nobody has a gradient: nothing happens
    after = opt.state_dict()["fused"]
    assert all(torch.equal(before[n], after[n]) for n in before)
    run(opt, 2, 700)
    only_empty = GroupedAdamW([params[1]])
    params[1].grad = torch.empty(0, 3, device=cuda())
    only_empty.step()
    assert only_empty.moments()[0].numel() == 0 and GroupedAdamW([params[1]], state_bits=8).moments()[0].numel() == 0


def test_step_on_another_stream_and_closure():
    params = params_of(make(SIZES, torch.float32, 60))
    opt = GroupedAdamW(params, max_norm=1.0, **HYPER)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    x = make([(61,)], torch.float32, 61)[0]
    with torch.cuda.stream(s):
        def closure():
            opt.zero_grad()
            y = (params[9] @ x).square().sum()
            y.backward()
            return y
        first = opt.step(closure)
        second = opt.step(closure)
    s.synchronize()
    assert torch.isfinite(first.detach()) and torch.isfinite(second.detach()) and not torch.equal(first, second)
    assert opt.device_state[:, 0].tolist() == [2.0 if i == 9 else 0.0 for i in range(len(params))]


def test_hooks_profiler_and_scheduler():
    """what torch's wrapper of `step` serves: step hooks, the profiler's label, learning-rate schedulers"""
    params = params_of(make(SIZES, torch.float32, 62))
    opt = GroupedAdamW(params, **HYPER)
    for p, g in zip(params, make(SIZES, torch.float32, 63)):
        p.grad = g
    seen = []
    hooks = [opt.register_step_pre_hook(lambda o, a, k: seen.append("pre")), opt.register_step_post_hook(lambda o, a, k: seen.append("post"))]
    opt.step()
    assert seen == ["pre", "post"]
    for h in hooks:
        h.remove()
    opt.step()
    assert seen == ["pre", "post"] and opt.device_state[0, 0] == 2
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        opt.step()
    assert any("Optimizer.step#GroupedAdamW.step" in e.key for e in prof.key_averages())
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, gamma=0.5)
    opt.step()
    sched.step()
    assert opt.param_groups[0]["lr"] == HYPER["lr"] / 2 and opt.device_state[0, 0] == 4


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_continues(bits):
    def model():
        return params_of(make(SIZES, torch.float16, 70))
    pa, pb = model(), model()
    kw = dict(state_bits=bits, master_weights=True, max_norm=1.0)
    a, b = GroupedAdamW(pa, lr=1e-2, **kw), GroupedAdamW(pb, lr=5e-2, **kw)
    run(a, 2, 600)
    b.load_state_dict(a.state_dict())
    assert b.param_groups[0]["lr"] == 1e-2
    for p, q in zip(pa, pb):
        q.data.copy_(p.data)
    for opt, params in ((a, pa), (b, pb)):
        opt.param_groups[0]["lr"] = 2e-2                                       # read at the call
        for p, g in zip(params, make(SIZES, torch.float16, 71)):
            p.grad = g
        opt.step()
    sa, sb = a.state_dict()["fused"], b.state_dict()["fused"]
    assert all(torch.equal(sa[n], sb[n]) for n in sa) and all(torch.equal(x, y) for x, y in zip(pa, pb))
    other = GroupedAdamW(model(), state_bits=40 - bits, master_weights=True)
    with pytest.raises(ValueError, match="expected"):
        other.load_state_dict(a.state_dict())
    for foreign in (torch.optim.AdamW(model()).state_dict(), {k: v for k, v in a.state_dict().items() if k != "fused"}):
        with pytest.raises(ValueError, match="expected"):
            other.load_state_dict(foreign)
    short = GroupedAdamW(params_of(make(SIZES[:-1], torch.float16, 70)), **kw)
    with pytest.raises(ValueError):
        short.load_state_dict(a.state_dict())


def test_agrees_with_the_flat_step():
    """the same weights as one flat buffer under FusedAdam: two float32 forms of one formula, each within 24 h of the truth relative to |p| + |U|"""
    sizes = [(50, 2), (50,), (50, 50), (50,), (1, 50), (1,)]
    flat = make([(sum(int(np.prod(s)) for s in sizes),)], torch.float32, 80)[0]
    views, at = [], 0
    for s in sizes:
        views.append(torch.nn.Parameter(flat[at:at + int(np.prod(s))].view(s)))
        at += int(np.prod(s))
    mine = params_of([v.detach().clone() for v in views])
    fused = FusedAdam(views, lr=1e-3, weight_decay=1e-2, decoupled=True, flat_params=flat)
    opt = GroupedAdamW(mine, lr=1e-3, weight_decay=1e-2)
    for k in range(20):
        fused.zero_grad()
        for a, b, g in zip(views, mine, make(sizes, torch.float32, 81 + k)):
            a.grad.copy_(g)
            b.grad = g
        fused.step()
        opt.step()
    for a, b in zip(views, mine):
        assert ((a - b).abs() <= 20 * 48 * H * (a.abs() + 1e-2)).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping_before_the_step_is_clipping_inside_it(bits):
    """as they are used together: clip_grad_norm_ then step, against max_norm.  The clipped gradient is rounded to float32 once more (h of m and
    2 h of v, so at most 3 h of the update), in 8 bits a code may then fall on the other side: the weights alone are compared there, over one step"""
    n_steps = 4 if bits == 32 else 1
    a, b = params_of(make(SIZES, torch.float32, 85)), params_of(make(SIZES, torch.float32, 85))
    oa, ob = GroupedAdamW(a, state_bits=bits, **HYPER), GroupedAdamW(b, state_bits=bits, max_norm=0.5, **HYPER)
    for k in range(n_steps):
        for p, q, g in zip(a, b, make(SIZES, torch.float32, 86 + k)):
            p.grad, q.grad = g.clone(), g
        norm = clip_grad_norm_(a, 0.5)
        oa.step()
        ob.step()
        assert abs(float(norm) / float(ob.grad_norm) - 1) <= 2 * H
    for p, q in zip(a, b):
        assert ((p - q).abs() <= n_steps * (4 * H * q.abs() + 24 * H * HYPER["lr"] * 10)).all()   # |U| <= 10 lr, generously: |m| / sqrt(v) hat is near 1


def test_moments_beyond_one_launch():
    """2^33 elements go into a launch; codes and scales behind them against the same in a small buffer"""
    n, split = (1 << 33) + 1152, 1 << 33
    if torch.cuda.mem_get_info()[0] < 12 * n:
        pytest.skip("needs 103 GB")
    codes = [torch.zeros(n, dtype=torch.uint8, device=cuda()) for _ in range(2)]
    scales = [torch.zeros(n // 128, dtype=torch.uint8, device=cuda()) for _ in range(2)]
    out = [torch.full((n,), 7.0, device=cuda()) for _ in range(2)]
    places = [slice(0, 2048), slice(split - 2048, split), slice(split, n)]
    gen = torch.Generator(cuda()).manual_seed(5)
    for w in places:
        for c, s in zip(codes, scales):
            c[w] = torch.randint(0, 127, (w.stop - w.start,), generator=gen, device=cuda(), dtype=torch.uint8)
            s[w.start // 128:w.stop // 128] = torch.randint(90, 140, ((w.stop - w.start) // 128,), generator=gen, device=cuda(), dtype=torch.uint8)

    def decode(c, s, o):
        rc = load_library().pinn_adamw_moments(*(t.data_ptr() for t in (*c, *s, *o)), o[0].numel(), _cur_stream(o[0]))
        assert rc == 0
    decode(codes, scales, out)
    for w in places:
        part = slice(w.start // 128, w.stop // 128)
        want = [torch.full((w.stop - w.start,), 7.0, device=cuda()) for _ in range(2)]
        decode([c[w].clone() for c in codes], [s[part].clone() for s in scales], want)
        for o, x in zip(out, want):
            assert torch.equal(o[w], x) and x.any()
    assert all(float(o[split // 2:split // 2 + 4096].abs().max()) == 0.0 for o in out)
    del codes, scales, out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,bits", [(torch.float32, 32), (torch.bfloat16, 8)])
def test_a_tensor_beyond_32_bits(dtype, bits):
    """2^31 + 4999 elements: offsets in bytes and in elements pass 32 bits; three places are held to the formula, and the norm to the sum of a constant"""
    n = (1 << 31) + 4999
    p = torch.nn.Parameter(torch.full((n,), 0.25, dtype=dtype, device=cuda()))
    p.grad = torch.full((n,), 2.0 ** -10, dtype=dtype, device=cuda())
    opt = GroupedAdamW([p], state_bits=bits, max_norm=1.0, **HYPER)
    places = [slice(0, 1024), slice((1 << 31) - 512, (1 << 31) + 512), slice(n - 3079, n)]
    rng = np.random.default_rng(0)
    for s in places:
        p.grad[s] = torch.tensor(rng.standard_normal(s.stop - s.start) * 2.0 ** -10, device=cuda()).to(dtype)
    grads = [f64(p.grad[s]) for s in places]
    rest = n - sum(s.stop - s.start for s in places)
    norm = np.sqrt(sum((g ** 2).sum() for g in grads) + rest * 2.0 ** -20)
    opt.step()
    assert abs(float(opt.grad_norm) / norm - 1) <= 2 * H
    ms, vs = (x[:n] for x in opt.moments())
    for s, g in zip(places, grads):
        p1, m1, v1 = F.step(np.full(len(g), 0.25), g * (1.0 / (norm + 1e-6)), 0.0, 0.0, 1, HYPER["lr"], 0.9, 0.999, 1e-8, HYPER["weight_decay"])
        # |U| is at most lr / (1 - b1) (1 - b1) / sqrt((1 - b2) / (1 - b2)) = lr at the first step
        assert (np.abs(f64(p[s]) - p1) <= H * (3 * 0.26 + 24 * HYPER["lr"]) + half_step(dtype, p1)).all()
        if bits == 32:
            assert (np.abs(f64(ms[s]) - m1) <= 5 * H * np.abs(m1)).all() and (np.abs(f64(vs[s]) - v1) <= 8 * H * v1).all()
        else:
            assert s.start % F.BLOCK == 0 and (s.stop % F.BLOCK == 0 or s.stop == n)
            assert np.array_equal(f64(ms[s]), F.round_flat(m1, s.start, 1, F.M)[0]) and np.array_equal(f64(vs[s]), F.round_flat(v1, s.start, 1, F.V)[0])


# ---- the norm ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
def test_grad_norm(dtype):
    sizes = SIZES + [(100001,), (8191,), (8193,), (16, 8192)]
    ts = make(sizes, dtype, 90)
    want = np.sqrt(sum((f64(t) ** 2).sum() for t in ts))
    got = grad_norm(ts)
    assert got.dtype == torch.float32 and got.shape == () and abs(float(got) - want) <= 2 * H * want
    assert torch.equal(got, grad_norm(iter(ts)))
    one = grad_norm(ts[-1])
    assert abs(float(one) - np.linalg.norm(f64(ts[-1]))) <= 2 * H * float(one)


def test_grad_norm_of_mixed_many_strided_and_extreme():
    ts = make([(1 + i % 40,) for i in range(333)], torch.float32, 91) + make([(77, 3)], torch.bfloat16, 92) + make([(5000,)], torch.float16, 93)
    ts += [make([(64, 50)], torch.float32, 94)[0].t(), make([(64, 50)], torch.float32, 95)[0][:, ::3], make([(7,)], torch.bfloat16, 96)[0].expand(9, 7)]
    flat = make([(40000,)], torch.bfloat16, 97)[0]
    ts.append(flat[1:30002])                                                   # 2 bytes off
    want = np.sqrt(sum((f64(t) ** 2).sum() for t in ts))
    assert abs(float(grad_norm(ts)) - want) <= 2 * H * want
    big = torch.full((3000,), 1e30, device=cuda())
    assert abs(float(grad_norm(big)) / (1e30 * 3000 ** 0.5) - 1) < 1e-6        # squares beyond float32
    small = torch.full((3000,), 1e-30, device=cuda())
    assert abs(float(grad_norm(small)) / (1e-30 * 3000 ** 0.5) - 1) < 1e-6
    assert torch.isnan(grad_norm([big, torch.tensor([float("nan")], device=cuda())]))
    assert float(grad_norm(torch.empty(0, device=cuda()))) == 0.0 and float(grad_norm([])) == 0.0
    empty = params_of([torch.empty(0, device=cuda()) for _ in range(300)])
    for p in empty:
        p.grad = torch.empty(0, device=cuda())
    for _ in range(3):
        junk = [torch.full((), 7.0, device=cuda()) for _ in range(64)]         # what the allocator hands out next is not zero by chance
        del junk
        assert float(clip_grad_norm_(empty, 1.0)) == 0.0 and float(grad_norm([p.grad for p in empty])) == 0.0
    assert float(grad_norm(torch.tensor(-3.0, device=cuda()))) == 3.0


@pytest.mark.parametrize("max_norm", [0.0, 0.25, 1e9])
def test_clip_grad_norm(max_norm):
    params = params_of(make(SIZES, torch.float32, 100) + make(SIZES, torch.bfloat16, 101) + make(SIZES, torch.float16, 102) + make([(99, 20)], torch.float32, 103))
    for p in params:
        p.grad = torch.empty_like(p).copy_(make([tuple(p.shape)], torch.float32, 104)[0])
    params[-1].grad = make([(20, 99)], torch.float32, 105)[0].t()
    params[3].grad = None
    wide = make([(128, 2)], torch.float32, 106)[0]
    params[4].grad = wide[:, 0]                                                # strided, with gaps
    gap = wide[:, 1].clone()
    had = [None if p.grad is None else f64(p.grad) for p in params]
    norm, f = F.clip_factor([g for g in had if g is not None], max_norm)
    version = params[0].grad._version
    got = clip_grad_norm_(params, max_norm)
    assert abs(float(got) - norm) <= 2 * H * norm and params[0].grad._version > version
    assert torch.equal(wide[:, 1], gap)
    for p, g in zip(params, had):
        if g is None:
            assert p.grad is None
            continue
        want = g * f
        tol = 2 * H * np.abs(want) + half_step(p.dtype, want)
        assert (np.abs(f64(p.grad) - want) <= tol).all()
        if f == 1.0:
            assert np.array_equal(f64(p.grad), g)


@pytest.mark.parametrize("n_tensors,size", [(1, 1), (10, 785), (64, 256), (65, 252), (16, 1024), (1, 16385), (32, 1024), (33, 1024), (1, 32768), (1, 32769), (700, 3)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_clip_grad_norm_around_the_one_launch_form(dtype, n_tensors, size):
    """few elements take one workgroup, 32768 elements and 64 tensors are its limits"""
    params = params_of(make([(size,)] * n_tensors, dtype, 106))
    for p, g in zip(params, make([(size,)] * n_tensors, dtype, 107, 2.0)):
        p.grad = g
    had = [f64(p.grad) for p in params]
    norm, f = F.clip_factor(had, 0.5)
    assert torch.equal(grad_norm([p.grad for p in params]), clip_grad_norm_(params, 1e9))
    assert all(np.array_equal(f64(p.grad), g) for p, g in zip(params, had))
    assert abs(float(clip_grad_norm_(params, 0.5)) - norm) <= 2 * H * norm
    for p, g in zip(params, had):
        assert (np.abs(f64(p.grad) - g * f) <= 2 * H * np.abs(g * f) + half_step(p.dtype, g * f)).all()


@pytest.mark.parametrize("dtype,n_tensors,size", [(torch.bfloat16, 600, 24579), (torch.float32, 3, 5_000_003), (torch.float16, 513, 32768)])
def test_clip_grad_norm_of_many_chunks(dtype, n_tensors, size):
    """workgroups that take several chunks, and launches whose partial sums (2400 and 2052) are added up once"""
    flat = make([(n_tensors * size,)], dtype, 108)[0]
    params = [torch.nn.Parameter(t) for t in torch.empty_like(flat).view(n_tensors, size).unbind()]
    for p, g in zip(params, flat.view(n_tensors, size).unbind()):
        p.grad = g
    had = f64(flat)
    norm, f = F.clip_factor([had], 0.5)
    assert torch.equal(grad_norm([p.grad for p in params]), clip_grad_norm_(params, 1e9)) and np.array_equal(f64(flat), had)
    assert abs(float(clip_grad_norm_(params, 0.5)) - norm) <= 2 * H * norm
    want = had * f
    assert (np.abs(f64(flat) - want) <= 2 * H * np.abs(want) + half_step(dtype, want)).all()


@pytest.mark.parametrize("size", [1000, 50000])
def test_clip_grad_norm_of_norms_that_are_not_finite(size):
    for bad in (float("nan"), float("inf")):
        p = params_of(make([(size,)], torch.float32, 110))[0]
        p.grad = make([(size,)], torch.float32, 111)[0]
        p.grad[17] = bad
        before = p.grad.clone()
        with pytest.raises(RuntimeError, match="not clipped"):
            clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
        assert torch.equal(p.grad.nan_to_num(), before.nan_to_num())
        norm = clip_grad_norm_(p, 1.0)
        assert not torch.isfinite(norm)
        finite = torch.isfinite(p.grad)
        assert not finite[17] and (not finite.any() if bad != bad else (p.grad[finite] == 0).all())
    assert float(clip_grad_norm_([torch.nn.Parameter(torch.ones(3, device=cuda()))], 1.0)) == 0.0


def test_refusals():
    p = params_of(make([(100,), (100,)], torch.float32, 120))
    p[0].grad = p[1].grad = make([(100,)], torch.float32, 121)[0]
    kept = p[0].grad.clone()
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm_(p, 1e-3)
    assert torch.equal(kept, p[0].grad)
    wide = make([(100, 3)], torch.float32, 122)[0]
    before, lone = wide.clone(), p[1]
    for one, two in ((wide[:, 0], wide[:, 0]), (wide[:, 1], wide.view(-1)[1:101])):
        p[0].grad, lone.grad = one, two
        with pytest.raises(ValueError, match="share memory"):
            clip_grad_norm_(p, 1e-3)
        assert torch.equal(wide, before)
    p[0].grad, lone.grad = wide[:, 0], wide[:, 2]                                # between each other's elements: apart
    norm = float(clip_grad_norm_(p, 1e-3))
    assert abs(norm / float(before[:, ::2].norm()) - 1) < 1e-5 and torch.equal(wide[:, 1], before[:, 1])
    assert (wide[:, ::2] - before[:, ::2] * (1e-3 / norm)).abs().max() < 1e-8
    p[0].grad = p[1].grad = kept
    assert abs(float(grad_norm([p[0].grad, p[1].grad])) / (2 ** 0.5 * float(grad_norm(kept))) - 1) < 1e-6   # reading the same one twice is fine
    q = torch.nn.Parameter(torch.ones(4, 3, device=cuda()))
    q.grad = torch.ones(3, device=cuda()).expand(4, 3)
    with pytest.raises(ValueError, match="expanded"):
        clip_grad_norm_(q, 0.1)
    with pytest.raises(ValueError, match="max_norm"):
        clip_grad_norm_(p, -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip_grad_norm_(p, float("nan"))
    with pytest.raises(ValueError, match="float32, bfloat16"):
        grad_norm(torch.ones(3, device=cuda(), dtype=torch.float64))
    with pytest.raises(TypeError):
        grad_norm([1.0])
    base = torch.zeros(300, device=cuda())
    with pytest.raises(ValueError, match="share memory"):
        GroupedAdamW([torch.nn.Parameter(base[:200]), torch.nn.Parameter(base[199:])])
    with pytest.raises(ValueError, match="share memory"), pytest.warns(UserWarning, match="duplicate"):
        GroupedAdamW([p[0], p[0]])
    with pytest.raises(ValueError, match="gaps"):
        GroupedAdamW([torch.nn.Parameter(base[::2])])
    with pytest.raises(ValueError, match="float64"):
        GroupedAdamW([torch.nn.Parameter(base.double())])
    with pytest.raises(ValueError, match="share memory"):
        tied = params_of(make([(50,), (50,)], torch.float32, 122))
        opt = GroupedAdamW(tied)
        tied[1].data = tied[0].data                                            # tied only later
        tied[0].grad = torch.ones(50, device=cuda())
        with pytest.raises(ValueError, match="share memory"):
            opt.step()
        opt.step()
    opt = GroupedAdamW([torch.nn.Parameter(base)])
    with pytest.raises(ValueError, match="all parameter groups"):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.ones(2, device=cuda()))]))
    opt.param_groups[0]["lr"] = -1.0
    opt.param_groups[0]["params"][0].grad = torch.ones(300, device=cuda())
    with pytest.raises(ValueError, match="lr"):
        opt.step()
    assert not base.any() and opt.device_state[0, 0] == 0


# ---- inside the training of a net --------------------------------------------------------------------------------
def pinn(graph, **options):
    from pde_amd import scripts
    torch.manual_seed(7)
    cls = scripts.for_script("5kdv/sw51-adamw.py").PhysicsInformedNN
    lb, ub = np.array([-10.0, -2.0]), np.array([10.0, 2.0])
    m = cls([2, 50, 50, 50, 50, 1], lb, ub)
    rng = np.random.default_rng(3)
    x0 = rng.uniform(lb[0], ub[0], (50, 1))
    with torch.no_grad():
        for p in m.dnn.parameters():
            p.copy_(torch.tensor(rng.standard_normal(tuple(p.shape)) * 0.15))
    m.set_training_data(x0, np.exp(-x0 ** 2), rng.uniform(lb[1], ub[1], (50, 1)), lb + (ub - lb) * rng.random((2000, 2)))
    m.use_hip_graph = graph
    for k, v in options.items():
        setattr(m, k, v)
    return m


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("bits,clip", [(32, None), (32, 1e-2), (8, 1e-2)])
def test_training_a_net(bits, clip, graph):
    """`adam_impl = "grouped"`: 20 steps, then one more whose update is held to the formula with the net's own gradients; without
    clipping and in float32 the weights follow FusedAdam's within the 1e-4 that float32 sums in another order leave after such a run."""
    m = pinn(graph, adam_impl="grouped", adam_state_bits=bits, max_grad_norm=clip)
    m.train(20, LBFGS_max_iter=0)
    opt = m.optimizer_Adam
    assert opt.device_state[:, 0].tolist() == [20.0] * 10 and opt.state_bits == bits
    if clip is None:
        other = pinn(graph)
        other.train(20, LBFGS_max_iter=0)
        a, b = m.dnn.flat_theta().double(), other.dnn.flat_theta().double()
        assert float((a - b).norm() / b.norm()) < 1e-4
    oracle = Oracle(opt)
    ms, vs = (f64(x) for x in opt.moments())
    oracle.m = [ms[at:at + p.numel()] for p, at in zip(opt._params, opt.offsets)]
    oracle.v = [vs[at:at + p.numel()] for p, at in zip(opt._params, opt.offsets)]
    oracle.t = [20] * 10
    opt.zero_grad()
    m.backward()
    opt.step()
    oracle.step([f64(p.grad) for p in opt._params])

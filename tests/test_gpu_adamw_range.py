"""GPU: GroupedAdamW, grad_norm and clip_grad_norm_ at the ends of float32's range and around captured calls, against float64 numpy
(adamw_formulas.py).  h = 2^-24 is the half step of float32."""
import numpy as np
import pytest
import torch

import adamw_formulas as F
from pde_amd._native import NORM_SMALL_ELEMENTS
from pde_amd.optim import GroupedAdamW, clip_grad_norm_, grad_norm

pytestmark = pytest.mark.gpu
H = 2.0 ** -24


def cuda():
    return torch.device("cuda", 0)


def f64(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def on_gpu(x, dtype=torch.float32):
    return torch.tensor(np.asarray(x), dtype=torch.float32).to(dtype).to(cuda())


# ---- the weights' update with 8-bit moments ------------------------------------------------------------------------
@pytest.mark.parametrize("lo,hi,eps", [(1e38, 3e38, 1e-8), (1e37, 1e38, 0.0), (1e-40, 1e-38, 0.0), (1e-44, 1e-42, 0.0), (1e-40, 1e-38, 1e-39)])
@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, False), (torch.bfloat16, True)])
def test_eight_bit_update_over_the_range(dtype, master, lo, hi, eps):
    """The first step moves a weight by lr |m^| / (sqrt(v^) + eps), lr where eps is nothing beside the gradient, however large or small that is:
    the denominator passes 2^126 above and float32's subnormals below.  At most 16 roundings of the update (half a step of a 16-bit weight more)."""
    rng = np.random.default_rng(1)
    n, lr = 1000, 1e-2
    g = on_gpu(rng.uniform(lo, hi, n) * rng.choice([-1.0, 1.0], n), dtype)
    p = torch.nn.Parameter(torch.zeros(n, dtype=dtype, device=cuda()))
    p.grad = g
    opt = GroupedAdamW([p], lr=lr, eps=eps, weight_decay=0.0, state_bits=8, master_weights=master)
    opt.step()
    p1, _, _ = F.step(np.zeros(n), f64(g), np.zeros(n), np.zeros(n), 1, lr, 0.9, 0.999, eps, 0.0)
    # a gradient that its type rounds to 0 is 0 / 0 where eps is 0
    zero = f64(g) == 0.0
    assert zero.all() == (dtype != torch.float32 and hi < 1e-41) and np.array_equal(np.isnan(p1), zero) and np.array_equal(np.isnan(f64(p)), zero)
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    assert (np.abs(f64(p) - p1) <= (16 * H + half) * np.abs(p1))[~zero].all()


@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, True), (torch.float16, True)])
def test_eight_bit_step_rounds_float32_weights_once(dtype, master):
    """The sum (1 - lr wd) p - U is formed in float64 and rounded to float32 once: half a step of the result.  U has the two approximations of
    its root and its reciprocal, each within 2^29 of float64's last places (2^-23 of the value), and nothing else that counts."""
    rng = np.random.default_rng(2)
    sizes, lr, wd = [5000, 127, 2049], 1e-3, 1e-2
    params = [torch.nn.Parameter(on_gpu(0.1 * rng.standard_normal(n), dtype)) for n in sizes]
    opt = GroupedAdamW(params, lr=lr, weight_decay=wd, state_bits=8, master_weights=master, max_norm=3.0)

    def weights(i):
        return f64(opt.master[opt.offsets[i]:opt.offsets[i] + sizes[i]] if master else params[i])
    for t in range(1, 5):
        for p in params:
            p.grad = on_gpu(rng.standard_normal(p.numel()), dtype)
        ms, vs = (f64(x) for x in opt.moments())
        had = [weights(i) for i in range(len(sizes))]
        grads = [f64(p.grad) for p in params]
        _, factor = F.clip_factor(grads, 3.0)
        opt.step()
        for i, n in enumerate(sizes):
            at = slice(opt.offsets[i], opt.offsets[i] + n)
            p1, _, _ = F.step(had[i], grads[i] * factor, ms[at], vs[at], t, lr, 0.9, 0.999, 1e-8, wd)
            update = np.abs(p1 - had[i] * (1 - lr * wd))
            half = np.spacing(np.abs(p1).astype(np.float32)).astype(np.float64) / 2
            assert (np.abs(weights(i) - p1) <= half * (1 + 1e-6) + 2.0 ** -22 * update).all(), (t, i)


# ---- norms beyond float32 ------------------------------------------------------------------------------------------
def huge(n, dtype, seed):
    rng = np.random.default_rng(seed)
    return on_gpu(rng.uniform(1e38, 3e38, n) * rng.choice([-1.0, 1.0], n), dtype)


@pytest.mark.parametrize("max_norm", [1.0, 1e-20, 1e30])
@pytest.mark.parametrize("n", [1000, 100000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_clipping_of_a_norm_beyond_float32(dtype, n, max_norm):
    """The norm reads infinity there, the factor comes from its float64 value (1e-40 and less: not a float32 with 24 bits), which is rounded once as is
    the product: h each, and half a step of bfloat16"""
    p = torch.nn.Parameter(torch.zeros(n, dtype=dtype, device=cuda()))
    p.grad = huge(n, dtype, 3)
    g = f64(p.grad)
    norm, factor = F.clip_factor([g], max_norm)
    assert norm > torch.finfo(torch.float32).max and factor < 1e-7
    assert float(clip_grad_norm_(p, max_norm)) == float("inf")
    want = g * factor
    assert (np.abs(f64(p.grad) - want) <= 2 * H * np.abs(want) + (torch.finfo(dtype).eps / 2 * np.abs(want) if dtype != torch.float32 else 0.0)).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_clipped_from_a_norm_beyond_float32(dtype, bits):
    """first moments after one step: the tolerance of test_gpu_adamw_group.py, 8-bit codes equal"""
    n = 3000
    p = torch.nn.Parameter(torch.zeros(n, dtype=dtype, device=cuda()))
    p.grad = huge(n, dtype, 4)
    opt = GroupedAdamW([p], state_bits=bits, max_norm=1.0)
    opt.step()
    g = f64(p.grad)
    _, factor = F.clip_factor([g], 1.0)
    _, m1, v1 = F.step(np.zeros(n), g * factor, np.zeros(n), np.zeros(n), 1)
    m, v = (f64(x)[:n] for x in opt.moments())
    assert float(opt.grad_norm) == float("inf") and opt.device_state[0, 0] == 1.0
    if bits == 8:
        assert np.array_equal(m, F.round_flat(m1, 0, 1, F.M)[0]) and np.array_equal(v, F.round_flat(v1, 0, 1, F.V)[0])
    else:
        assert (np.abs(m - m1) <= H * (np.abs(m1) + 0.4 * np.abs(g * factor))).all() and (np.abs(v - v1) <= 8 * H * v1).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_skip_goes_by_the_norm_that_is_reported(bits):
    p = torch.nn.Parameter(on_gpu(np.ones(2000)))
    p.grad = huge(2000, torch.float32, 5)
    opt = GroupedAdamW([p], state_bits=bits, skip_nonfinite=True)
    before = opt.state_dict()["fused"]
    opt.step()
    after = opt.state_dict()["fused"]
    assert float(opt.grad_norm) == float("inf") and (p == 1).all() and all(torch.equal(before[k], after[k]) for k in after)
    p.grad.mul_(1e-10)
    opt.step()
    assert torch.isfinite(opt.grad_norm) and opt.device_state[0, 0] == 1.0 and not (p == 1).any()


# ---- what a step without gradients reports ---------------------------------------------------------------------------
@pytest.mark.parametrize("options", [dict(max_norm=1.0), dict(skip_nonfinite=True)])
def test_norm_of_a_step_without_gradients(options):
    p = torch.nn.Parameter(on_gpu(np.ones(50)))
    opt = GroupedAdamW([p], **options)
    p.grad = on_gpu(np.full(50, 2.0))
    opt.step()
    assert abs(float(opt.grad_norm) / (2.0 * 50 ** 0.5) - 1) < 1e-6
    after = p.detach().clone()
    opt.zero_grad()
    opt.step()
    assert float(opt.grad_norm) == 0.0 and torch.equal(p, after) and opt.device_state[0, 0] == 1.0


# ---- captured clippings beyond the one-launch form ---------------------------------------------------------------------
def test_captured_clippings_of_many_elements_on_two_streams():
    """Lists that need partial sums, 300 tensors (two launches of sums and two of scaling), one of them strided: each graph has its
    partial sums to itself, so two that replay at once do not disturb each other."""
    sizes = [(1 + 37 * i % 900,) for i in range(298)] + [(3_000_000,)]
    assert sum(s[0] for s in sizes) > NORM_SMALL_ELEMENTS
    sets, graphs, norms = [], [], []

    def fresh(seed, scale):
        gen = torch.Generator(cuda()).manual_seed(seed)
        return [scale * torch.empty(s, device=cuda()).normal_(generator=gen) for s in sizes + [(500, 3)]]
    for k in range(2):
        params = [torch.nn.Parameter(torch.zeros(s, device=cuda())) for s in sizes + [(500,)]]
        wide = torch.zeros(500, 3, device=cuda())
        for p in params[:-1]:
            p.grad = torch.zeros_like(p)
        params[-1].grad = wide[:, 1]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            clip_grad_norm_(params, 1.0)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norms.append(clip_grad_norm_(params, 1.0))
        sets.append((params, wide))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for r in range(4):
        given = [fresh(2 * r + k, 3.0 + k) for k in range(2)]
        for (params, wide), grads in zip(sets, given):
            for p, g in zip(params, grads[:-1]):
                p.grad.copy_(g)
            wide.copy_(grads[-1])
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (params, wide), grads, norm in zip(sets, given, norms):
            seen = grads[:-1] + [grads[-1][:, 1].contiguous()]
            assert torch.equal(norm, grad_norm(seen))
            want, factor = F.clip_factor([f64(g) for g in seen], 1.0)
            assert abs(float(norm) / want - 1) <= 2 * H
            for p, g in zip(params, seen):
                assert (np.abs(f64(p.grad) - f64(g) * factor) <= 2 * H * np.abs(f64(g) * factor)).all()
            assert torch.equal(wide[:, ::2], grads[-1][:, ::2])


# ---- the largest 8-bit scales ----------------------------------------------------------------------------------------
def held(x, first, t, form):
    """one block as it is held in 8 bits, also where its values are beyond what the largest scale can hold: those take the largest code"""
    tab = F.table(form)
    a = np.abs(x)
    scale = 0
    while scale < form["most"] and a.max() >= tab[-1] * 2.0 ** (scale - 127):
        scale += 1
    y = a * 2.0 ** (127 - scale)
    c = np.clip(np.searchsorted(tab, y, side="right") - 1, 0, len(tab) - 2)
    i = np.arange(first, first + len(x), dtype=np.uint64)
    word = (i * np.uint64(form["place"]) + np.uint64(t * form["step"] % 2 ** 32)) % np.uint64(2 ** 32)
    u = ((word >> np.uint64(15)) | np.uint64(1)).astype(np.float64) / 2 ** 17
    c = np.minimum(np.floor(c + (y - tab[c]) / (tab[c + 1] - tab[c]) + u), len(tab) - 1).astype(np.int64)
    if form is F.V:
        c = np.where(a > 0, np.maximum(c, 1), c)
    return np.where(x < 0, -1.0, 1.0) * tab[c] * 2.0 ** (scale - 127), scale


@pytest.mark.parametrize("scale", [1e18, 3e19, 1e21, 1e30, 7e37])
def test_eight_bit_moments_at_their_largest(scale):
    """exp_avg_sq holds 1.75 2^127 at most and exp_avg too: beyond, the largest code of the largest scale, in the blocks that need it alone.  Scales and
    codes equal the formula's, and the weights follow the moments before they are rounded (at most 16 roundings)."""
    n, lr = 1024, 1e-2
    rng = np.random.default_rng(7)
    p = torch.nn.Parameter(torch.zeros(n, device=cuda()))
    opt = GroupedAdamW([p], lr=lr, weight_decay=0.0, state_bits=8)
    m, v = np.zeros(n), np.zeros(n)
    top = False
    for t in range(1, 5):
        g = rng.standard_normal(n) * scale
        g[256:512] *= 1e-9
        g[5] = 0.0
        p.grad = on_gpu(g)
        had = f64(p)
        opt.step()
        p1, m, v = F.step(had, f64(p.grad), m, v, t, lr, 0.9, 0.999, 1e-8, 0.0)
        assert (np.abs(f64(p) - p1)[6:] <= 16 * H * (np.abs(p1 - had) + np.abs(p1))[6:]).all()
        for x, form, codes, scales in ((m, F.M, opt.exp_avg, opt.exp_avg_scale), (v, F.V, opt.exp_avg_sq, opt.exp_avg_sq_scale)):
            out = [held(x[b:b + 128], b, t, form) for b in range(0, n, 128)]
            x[:] = np.concatenate([o[0] for o in out])
            assert scales.cpu().tolist() == [o[1] for o in out], t
            got = opt.moments()[0 if form is F.M else 1]
            assert np.array_equal(f64(got), x), t
            top |= form is F.V and max(o[1] for o in out) == form["most"] and int(codes.max()) == 254
        assert torch.isfinite(p).all() and torch.isfinite(opt.moments()[1]).all()
    assert top == (scale >= 1e21)                                             # (1 - b2) (3 scale)^2 against 3e38: 1e37 for 3e19, 1e40 for 1e21

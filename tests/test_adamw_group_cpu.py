"""CPU: what GroupedAdamW, grad_norm, clip_grad_norm_ and their C entries refuse before anything reaches a GPU, and the float64
formulas the GPU tests use (adamw_formulas.py) against torch.optim.AdamW and against the 8-bit format's own properties."""
import ctypes
import os

import numpy as np
import pytest
import torch

import adamw_formulas as F
from pde_amd._native import LIB_PATH, ADAMW_BLOCK, ADAMW_CHUNK32, ADAMW_CHUNK8, ADAMW_CHUNK_DTYPE, ADAMW_MAX_CHUNKS, ADAMW_MAX_TENSORS, ADAMW_TICKET_WORDS, NORM_SMALL_ELEMENTS, NORM_SMALL_TENSORS, NativeError, PinnAdamWGroup, load_library
from pde_amd.optim import GroupedAdamW, _runs, _share_memory, clip_grad_norm_, grad_norm
from conftest import GOLDEN, ROOT

needs_lib = pytest.mark.skipif(not os.path.exists(LIB_PATH), reason="libpinnjet.so not built")
needs_list = pytest.mark.skipif(not os.path.exists(os.path.join(ROOT, "pde_amd", "_tensorlist.so")), reason="_tensorlist.so not built")


def test_formulas_follow_torch():
    """float64 against float64: three steps of torch.optim.AdamW, 1e-14 of |p| + lr for the few roundings of each"""
    torch.manual_seed(0)
    p = torch.nn.Parameter(torch.randn(50, dtype=torch.float64))
    opt = torch.optim.AdamW([p], lr=1e-2, weight_decay=0.1)
    q, m, v = p.detach().numpy().copy(), np.zeros(50), np.zeros(50)
    for t in range(1, 4):
        p.grad = torch.randn(50, dtype=torch.float64)
        opt.step()
        q, m, v = F.step(q, p.grad.numpy(), m, v, t, lr=1e-2, wd=0.1)
        assert np.abs(p.detach().numpy() - q).max() < 1e-14 * (np.abs(q).max() + 1e-2)


@pytest.mark.parametrize("form", [F.M, F.V])
def test_eight_bit_format(form):
    rng = np.random.default_rng(1)
    tab = F.table(form)
    assert len(tab) == form["codes"] and (np.diff(tab) > 0).all() and tab[-1] == 1.75 * 2.0 ** (15 - form["bias"] if form is F.M else 31 - form["bias"])
    x = rng.standard_normal(128) * np.exp(3 * rng.standard_normal(128))
    x = np.abs(x) if form is F.V else x
    up = 0
    for t in range(64):
        y, s = F.round_block(x, 256, t, form)
        step = np.maximum(np.abs(x) / 8, tab[1] * 2.0 ** (s - 127))            # between codes: 3 bits, below the normals the smallest code
        assert (np.abs(y - x) <= step * (1 + 1e-12)).all()                     # a whole step at most, either way
        assert np.array_equal(F.round_block(y, 256, t, form)[0], y)            # what is on a code stays
        up += y - x
    assert (np.abs(up / 64) <= step * 4 / 64).all()                            # an even sequence: within 4 of 64 places
    y, s = F.round_block(np.zeros(128), 0, 1, form)
    assert s == 0 and not y.any()
    assert F.round_block(np.full(128, np.inf), 0, 1, form)[1] == 255
    if form is F.V:
        tiny = np.full(128, 1e-60)
        tiny[0] = 1.0
        assert (F.round_block(tiny, 0, 1, form)[0] > 0).all()


@needs_list
def test_refusals_without_a_gpu():
    p = torch.nn.Parameter(torch.ones(3))
    with pytest.raises(NativeError, match="no CPU fallback"):
        GroupedAdamW([p])
    for kw, word in ((dict(state_bits=16), "state_bits"), (dict(max_norm=-1.0), "max_norm"), (dict(max_norm=float("nan")), "max_norm"),
                     (dict(lr=-1.0), "lr"), (dict(betas=(1.0, 0.9)), "betas"), (dict(betas=(0.9, -0.1)), "betas"), (dict(eps=-1e-8), "eps"),
                     (dict(weight_decay=-1.0), "weight_decay"), (dict(lr=float("nan")), "lr")):
        with pytest.raises(ValueError, match=word):
            GroupedAdamW([p], **kw)
    with pytest.raises(ValueError):
        GroupedAdamW([])
    p.grad = torch.ones(3)
    with pytest.raises(NativeError, match="no CPU fallback"):
        clip_grad_norm_(p, 1.0)
    with pytest.raises(NativeError, match="no CPU fallback"):
        grad_norm([p.grad])
    with pytest.raises(ValueError, match="max_norm"):
        clip_grad_norm_(p, -0.5)
    with pytest.raises(TypeError):
        grad_norm([3.0])


@needs_lib
def test_c_entries_refuse_without_a_gpu():
    lib = load_library()
    header = open(os.path.join(ROOT, "include", "pinnjet.h")).read()
    for name, value in (("PINN_ADAMW_BLOCK", ADAMW_BLOCK), ("PINN_ADAMW_CHUNK32", ADAMW_CHUNK32), ("PINN_ADAMW_CHUNK8", ADAMW_CHUNK8), ("PINN_ADAMW_MAX_TENSORS", ADAMW_MAX_TENSORS), ("PINN_ADAMW_MAX_CHUNKS", ADAMW_MAX_CHUNKS),
                        ("PINN_ADAMW_TICKET_WORDS", ADAMW_TICKET_WORDS), ("PINN_NORM_SMALL_TENSORS", NORM_SMALL_TENSORS),
                        ("PINN_NORM_SMALL_ELEMENTS", NORM_SMALL_ELEMENTS)):
        assert "#define %s %d " % (name, value) in header
    assert ADAMW_CHUNK_DTYPE.itemsize == 32 and ctypes.sizeof(PinnAdamWGroup) == 168
    one = (ctypes.c_uint64 * 2)(4096, 8192)
    INVALID, NULL, LARGE, OVERLAP = -1, -4, -6, -7

    def group(**kw):
        d = PinnAdamWGroup(n_tensors=2, n_chunks=2, dtype=0, state_bits=32, chunks=16, rows=16, exp_avg=16, exp_avg_sq=16, device_state=16, ticket=16)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.pinn_adamw_group_step(ctypes.byref(d), one, one, None)
    assert lib.pinn_adamw_group_step(None, one, one, None) == NULL
    assert lib.pinn_adamw_group_step(ctypes.byref(PinnAdamWGroup()), None, one, None) == NULL
    for kw in (dict(n_tensors=-1), dict(n_tensors=241), dict(n_chunks=-1), dict(dtype=3), dict(dtype=-1), dict(state_bits=16), dict(n_partials=-1), dict(master=16)):
        assert group(**kw) == INVALID, kw
    for kw in (dict(chunks=None), dict(rows=None), dict(exp_avg=None), dict(exp_avg_sq=None), dict(device_state=None), dict(ticket=None),
               dict(state_bits=8), dict(n_partials=4)):
        assert group(**kw) == NULL, kw
    assert group(n_chunks=1 << 40) == LARGE and group(n_chunks=1 << 24) == LARGE          # 2^24 workgroups of 256: 2^32 threads
    assert lib.pinn_adamw_moments(16, 16, 16, 16, 16, 16, 1 << 50, None) == LARGE
    assert group(n_tensors=0) == 0 and group(n_chunks=0) == 0
    d = PinnAdamWGroup(n_tensors=1, n_chunks=1, state_bits=32, chunks=16, rows=16, exp_avg=16, exp_avg_sq=16, device_state=16, ticket=16)
    zero = (ctypes.c_uint64 * 1)(0)
    assert lib.pinn_adamw_group_step(ctypes.byref(d), zero, one, None) == NULL
    assert lib.pinn_adamw_group_step(ctypes.byref(d), zero, zero, None) == 0                    # no gradient: nothing to do

    assert lib.pinn_adamw_moments(16, 16, 16, 16, 16, 16, 100, None) == INVALID
    assert lib.pinn_adamw_moments(16, 16, 16, 16, 16, 16, -128, None) == INVALID
    assert lib.pinn_adamw_moments(16, None, 16, 16, 16, 16, 128, None) == NULL
    assert lib.pinn_adamw_moments(None, None, None, None, None, None, 0, None) == 0

    assert lib.pinn_grad_norm_partials(-1) == INVALID and lib.pinn_grad_norm_partials(0) == 0
    assert lib.pinn_grad_norm_partials(250) == 1024 and lib.pinn_grad_norm_partials(251) == 2048
    count = ctypes.c_int32()
    n2, f32 = (ctypes.c_int64 * 2)(100, 100), (ctypes.c_int32 * 2)(0, 0)

    def sums(x=one, n=n2, dt=f32, k=2, part=16, room=4096):
        return lib.pinn_grad_sumsq(x, n, dt, k, part, room, ctypes.byref(count), None)
    assert sums(k=-1) == INVALID and sums(n=(ctypes.c_int64 * 2)(5, -1)) == INVALID and sums(dt=(ctypes.c_int32 * 2)(0, 7)) == INVALID
    assert sums(x=None) == NULL and sums(part=None) == NULL and sums(x=(ctypes.c_uint64 * 2)(16, 0)) == NULL
    assert sums(n=(ctypes.c_int64 * 2)(1, 1 << 62)) == LARGE and sums(room=1) == LARGE
    assert lib.pinn_grad_sumsq(one, n2, f32, 2, 16, 4096, None, None) == NULL

    def norm(x=one, n=n2, dt=f32, k=2, part=16, room=4096, out=16):
        return lib.pinn_grad_norm(x, n, dt, k, part, room, out, None)
    big = (ctypes.c_int64 * 2)(1 << 20, 100)
    assert norm(part=None, n=big) == NULL and norm(out=None) == NULL and norm(x=None) == NULL and norm(k=-1) == INVALID and norm(n=big, room=1) == LARGE

    def clip(x=one, n=n2, k=2, part=16, m=1.0, out=16, room=4096):
        return lib.pinn_grad_clip(x, n, f32, k, part, room, m, out, None)
    assert clip(m=-1.0) == INVALID and clip(m=float("nan")) == INVALID and clip(k=-1) == INVALID and clip(n=big, x=(ctypes.c_uint64 * 2)(1 << 30, 16), room=1) == LARGE
    assert clip(part=None, n=big, x=(ctypes.c_uint64 * 2)(1 << 30, 16)) == NULL and clip(out=None) == NULL
    assert clip(x=(ctypes.c_uint64 * 2)(4096, 4096 + 396)) == OVERLAP and clip(x=(ctypes.c_uint64 * 2)(8192, 8192)) == OVERLAP
    assert clip(x=(ctypes.c_uint64 * 2)(4096 + 396, 4096)) == OVERLAP
    assert lib.pinn_error_string(OVERLAP) == b"two tensors share memory"


def test_shared_memory_of_any_strides():
    """exact: columns that lie between each other's do not share, whatever their extents"""
    a, b = torch.zeros(64, 6), torch.zeros(64, 6, dtype=torch.bfloat16)
    flat = torch.zeros(100)
    assert not _share_memory([])
    assert not _share_memory([a, b, flat, torch.zeros(0), torch.tensor(1.0)])
    assert not _share_memory([a[:, 0], a[:, 1], a[:, 2:4], a[:, 5], b[::2], b[1::2]])
    assert not _share_memory([a.t()[4], a[:, 3], flat[:50], flat[50:], a[:0]])
    assert _share_memory([flat, b[:, 0], b[:, 0]]) and _share_memory([a[:, 1:3], a[:, 2]]) and _share_memory([a[7], b, a[:, 5]])
    assert _share_memory([flat[::2], flat[3::4], flat[2:3]])
    assert not _share_memory([flat[::2], flat[3::4], flat[1:2]])
    whole = torch.zeros(32, dtype=torch.float32)
    assert _share_memory([whole, whole.view(torch.bfloat16)[::2][3:4]])


def test_what_a_launch_takes():
    """240 tensors, and fewer than 2^24 chunks"""
    assert _runs([], [], 1024) == []
    assert [len(r) for r in _runs(list(range(500)), [5] * 500, 1024)] == [240, 240, 20]
    half = (1 << 23) * 1024
    assert _runs([3, 7, 8, 9], [half, half, 0, 1], 1024) == [[3], [7, 8, 9]]
    assert _runs([3, 7, 8], [half, half - 1024, 1], 1024) == [[3, 7], [8]]
    assert _runs([3, 7, 8], [half, half, half], 2048) == [[3, 7, 8]]
    assert _runs([0], [2 * half - 1024], 1024) == [[0]]
    with pytest.raises(ValueError, match="elements"):
        _runs([0], [2 * half - 1023], 1024)


def test_options_that_need_the_grouped_step():
    from test_host_logic import feed, make_model
    from pde_amd import scripts
    g = np.load(os.path.join(GOLDEN, "burgers_9x20_xavier.npz"))
    for kw in (dict(max_grad_norm=1.0), dict(adam_state_bits=8), dict(adam_impl="torch", max_grad_norm=1.0)):
        m = make_model(g, scripts.burgers.PI.PhysicsInformedNN)
        feed(m, g, "burgers")
        for k, v in kw.items():
            setattr(m, k, v)
        with pytest.raises(ValueError, match="grouped"):
            m.train(1, LBFGS_max_iter=0)
    m = make_model(g, scripts.burgers.PI.PhysicsInformedNN)
    feed(m, g, "burgers")
    m.adam_impl = "grouped"
    with pytest.raises(NativeError, match="no CPU fallback"):
        m.train(1, LBFGS_max_iter=0)


@needs_list
def test_lists_of_tensors():
    """csrc/tensorlist.cpp on CPU tensors: what it reads, which gradients it hands back, what it refuses"""
    import ctypes as C
    from pde_amd._native import load_tensorlist
    native = load_tensorlist()
    ps = [torch.nn.Parameter(x) for x in (torch.randn(3, 5), torch.randn(0), torch.randn(7, 4).t(), torch.randn(6).half(), torch.randn(1, 9), torch.randn(2).bfloat16())]
    n = len(ps)
    numel, dtype = (C.c_int64 * n)(*(p.numel() for p in ps)), (C.c_int32 * n)(0, 0, 0, 2, 0, 1)
    p, g, count = (C.c_uint64 * n)(), (C.c_uint64 * n)(), (C.c_int64 * n)()

    def gather():
        return native.gather(ps, *(C.addressof(x) for x in (numel, dtype, p, g, count)))
    assert gather() == (0, [], True) and list(g) == [0] * n and list(count) == [0] * n
    for q in ps[:5]:
        q.grad = torch.ones_like(q)
    before = [q._version for q in ps]
    assert gather() == (4, [], False) and list(count) == [15, 0, 28, 6, 9, 0]
    assert list(p) == [q.data_ptr() for q in ps] and g[0] == ps[0].grad.data_ptr() and g[1] == g[5] == 0
    ps[2].grad = torch.ones(4, 7)                                              # another order than its parameter's
    ps[4].grad = torch.ones(9, 1).t()                                          # another stride of a dimension of one element: the same order
    assert gather() == (4, [2], False) and g[2] == 0 and g[4] == ps[4].grad.data_ptr()
    assert [q._version - b for q, b in zip(ps, before)] == [2, 0, 2, 2, 2, 0]
    dtype[3] = 1
    with pytest.raises(ValueError, match="parameter 3 is not what it was"):
        gather()
    dtype[3] = 2
    ps[0].data = torch.randn(3, 6)
    with pytest.raises(ValueError, match="parameter 0"):
        gather()
    assert p[0] == 0                                                           # so that the next call says "moved"
    ps[0].data = torch.randn(3, 5)
    assert gather() == (4, [2], True) and gather() == (4, [2], False)
    ps[0].grad.data = torch.ones(5, 3)
    with pytest.raises(ValueError, match="gradient of parameter 0"):
        gather()
    ps[0].grad = None
    ps[0].grad = torch.sparse_coo_tensor(torch.tensor([[0], [1]]), torch.tensor([1.0]), (3, 5))
    with pytest.raises(ValueError, match="gradient of parameter 0"):
        gather()
    x = (C.c_uint64 * 6)()

    def describe(ts, of_grads=False):
        return native.describe(ts, of_grads, C.addressof(x), C.addressof(numel), C.addressof(dtype))
    a = torch.randn(4, 6)
    with pytest.raises(NativeError, match="no CPU fallback"):
        describe([a])
    a = torch.empty(4, 6, device="meta")                                       # no GPU here: what it reads beside the addresses
    assert describe([a, a.t(), a[:, ::2], a[:0].bfloat16()]) == (4, [(2, 2)], -1, 60)
    assert list(numel)[:4] == [24, 24, 12, 0] and list(dtype)[:4] == [0, 0, 0, 1]
    qs = [torch.nn.Parameter(t) for t in (a, a[0], a[1])]
    assert describe(qs, True) == (0, [], None, 0)
    qs[1].grad, qs[2].grad = torch.empty(6, device="meta"), torch.empty(12, device="meta")[::2]
    before = [q.grad._version for q in qs[1:]]
    assert describe(qs, 1) == (2, [(1, 2)], -1, 12) and [q.grad._version for q in qs[1:]] == before
    assert describe(qs, 2) == (2, [(1, 2)], -1, 12) and [q.grad._version for q in qs[1:]] == [b + 1 for b in before]
    for bad in (a.double(), a.long(), torch.empty(4, 6, layout=torch.sparse_coo, device="meta")):
        with pytest.raises(ValueError, match="tensor 1"):
            describe([a, bad])
    with pytest.raises(ValueError, match="one device"):
        describe([a, torch.empty(2)])
    for call in (lambda: describe([a, 3]), lambda: native.gather([None] * 6, 0, 0, 0, 0, 0), lambda: describe((a,)), lambda: describe([a, None], 2)):
        with pytest.raises(TypeError):
            call()

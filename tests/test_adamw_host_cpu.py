"""CPU: the host side of GroupedAdamW, grad_norm and clip_grad_norm_ - arguments that would be taken for others, parameter lists without
a parameter, gradients that share memory, libraries that do not fit this package."""
import copy
import os
import pickle

import numpy as np
import pytest
import torch

from pde_amd import _native as native
from pde_amd.optim import GroupedAdamW, _share_memory, clip_grad_norm_

needs_lib = pytest.mark.skipif(not os.path.exists(native.LIB_PATH), reason="libpinnjet.so not built")


@pytest.mark.parametrize("third", [2.0, 1.0, 2, 1, float("inf"), "inf", None])
def test_a_norm_type_is_not_taken_for_error_if_nonfinite(third):
    """torch.nn.utils.clip_grad_norm_ takes the norm's type third; here it is always 2"""
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = torch.ones(3)
    with pytest.raises(TypeError, match="2-norm"):
        clip_grad_norm_([p], 1.0, third)
    assert torch.equal(p.grad, torch.ones(3))


def test_groups_without_any_parameter_are_refused():
    with pytest.raises(ValueError, match="no parameter"):
        GroupedAdamW([dict(params=[]), dict(params=[])])


def test_copies_that_would_lose_the_moments_are_refused():
    opt = object.__new__(GroupedAdamW)
    opt.__dict__.update(defaults={}, state={}, param_groups=[], exp_avg=torch.ones(3))
    for call in (copy.copy, copy.deepcopy, pickle.dumps):
        with pytest.raises(TypeError, match="load_state_dict"):
            call(opt)


def columns(rows, n, dtype=torch.float32):
    return list(torch.zeros(rows, n, dtype=dtype).unbind(1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n", [(1, 5), (7, 40), (100, 512), (1000, 65)])
def test_many_columns_are_not_compared_pair_by_pair(monkeypatch, rows, n, dtype):
    """... which is the square of their number (512 columns: 131 000 comparisons)"""
    calls = []
    real = np.shares_memory
    monkeypatch.setattr(np, "shares_memory", lambda *a, **k: calls.append(1) or real(*a, **k))
    cols = columns(rows, n, dtype)
    assert not _share_memory(cols)
    assert _share_memory(cols + [cols[n // 2][rows // 2:]]) and _share_memory([cols[-1][-1:]] + cols)
    assert len(calls) <= 3 * rows * n / 32


def test_shared_memory_by_pairs_and_by_marks_agree():
    """random strided views of one buffer against the sets of their elements"""
    rng = np.random.default_rng(0)
    seen = set()
    for k in range(400):
        kinds = [torch.float32, torch.bfloat16, torch.float16]
        base = torch.zeros(4000, dtype=torch.bfloat16)
        views, sets = [], []
        for _ in range(int(rng.integers(2, 5))):
            t = base.view(kinds[int(rng.integers(0, 3))])
            shape, strides = [int(x) for x in rng.integers(1, 9, 3)], [int(x) for x in rng.integers(1, 60, 3)]
            room = t.numel() - 1 - sum(st * (s - 1) for s, st in zip(shape, strides))
            at = int(rng.integers(0, room + 1))
            views.append(t.as_strided(shape, strides, at))
            size = t.element_size() // 2
            places = (at + sum(i * st for i, st in zip(np.indices(shape), strides))).ravel()
            sets.append({int(size * x + h) for x in places for h in range(size)})
        want = any(sets[i] & sets[j] for i in range(len(sets)) for j in range(i))
        seen.add(want)
        assert _share_memory(views) == want, k
    assert seen == {True, False}


def test_shared_memory_needs_no_numpy_2(monkeypatch):
    monkeypatch.delattr(np.lib, "array_utils", raising=False)
    cols = columns(30, 3)
    assert not _share_memory(cols) and _share_memory(cols + [cols[1]])
    big = columns(100000, 2)                            # by pairs
    assert not _share_memory(big) and _share_memory(big + [big[0][5:6]])


def test_shared_memory_that_is_hard_to_decide():
    """strides for which the search by pairs would take hours are marked element by element"""
    base = torch.zeros(1 << 22)
    strides = [1009, 1013, 1019, 1021, 1031, 1033, 1039]
    a, b = base.as_strided([6] * 7, strides, 0), base.as_strided([6] * 7, [s + 2 for s in strides], 1)
    assert isinstance(_share_memory([a, b]), bool)


@needs_lib
def test_a_library_of_another_build_is_noticed(monkeypatch):
    """its chunk size, the order or the size of the structs' fields, a missing entry point: it is not called"""
    import ctypes

    def loads():
        monkeypatch.setattr(native, "_lib", None)
        return native.load_library()
    loads()

    class Swapped(ctypes.Structure):
        fields = list(native.PinnAdamWGroup._fields_)
        i = [name for name, _ in fields].index("exp_avg")
        fields[i], fields[i + 1] = fields[i + 1], fields[i]
        _fields_ = fields
    for name, value in (("ADAMW_CHUNK8", 4096), ("ADAMW_TICKET_WORDS", 1), ("PinnAdamWGroup", Swapped), ("SYMBOLS", native.SYMBOLS + ["pinn_not_there"]),
                        ("ADAMW_CHUNK_DTYPE", np.dtype([("base", np.int64), ("place", np.int64), ("tensor", np.int32), ("count", np.int32),
                                                        ("row", np.int32), ("reserved", np.int32)]))):
        with monkeypatch.context() as m:
            m.setattr(native, name, value)
            with pytest.raises(native.NativeError, match="build it again"):
                loads()
    loads()

"""Adam / AdamW for a net whose parameters are views of ONE flat buffer: one HIP launch per step.

The reference's Adam phase is `torch.optim.Adam(self.dnn.parameters())` / `AdamW(..., weight_decay=1e-2)`
(7kdv/PI-7kdv3soliton.py:138,154-157; 7kdv/sw73-adamW.py:170): ten parameter tensors, ~15 foreach launches per
step.  `FusedAdam` has the same constructor arguments, the same update rule (torch's default, non-amsgrad
Adam; `decoupled=True` is AdamW) and the usual `zero_grad()` / `step()` protocol; the step count lives on the
device, so a captured HIP graph replays it as is.

`GroupedAdamW` is the step for everything else: tensors that lie anywhere, several parameter groups, bfloat16 and float16
weights, moments in 32 or 8 bits, clipping of the global gradient norm; `grad_norm` and `clip_grad_norm_` are that norm alone.

There is no CPU fallback: all of it needs libpinnjet.so and a GPU.
"""
import bisect
import ctypes

import numpy as np
import torch
import torch.optim.optimizer as _hooks

from ._native import (ADAMW_BLOCK, ADAMW_CHUNK32, ADAMW_CHUNK8, ADAMW_CHUNK_DTYPE, ADAMW_MAX_CHUNKS, ADAMW_MAX_TENSORS, ADAMW_TICKET_WORDS,
                      DTYPE_CODES, ERR_OVERLAP, NORM_SMALL_ELEMENTS, NORM_SMALL_TENSORS, NativeError, PinnAdamWGroup, _check, _cur_stream, _on,
                      load_library, load_tensorlist)


class FusedAdam(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, decoupled=False,
                 flat_params=None):
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, decoupled=decoupled)
        super().__init__(params, defaults)
        if len(self.param_groups) != 1:
            raise ValueError("FusedAdam takes one parameter group")
        self._params = self.param_groups[0]["params"]
        if flat_params is None or not flat_params.is_cuda:
            raise NativeError("FusedAdam needs the flat float32 CUDA buffer the parameters are views of; "
                              "there is no CPU fallback (use torch.optim.Adam)")
        off = 0
        for p in self._params:
            if p.data_ptr() != flat_params.data_ptr() + 4 * off or p.dtype != torch.float32:
                raise ValueError("flat_params is not the buffer the parameters are views of")
            off += p.numel()
        if off != flat_params.numel():
            raise ValueError("flat_params has %d elements, the parameters %d" % (flat_params.numel(), off))
        self.lib = load_library()
        self._x = flat_params
        dev = flat_params.device
        n = flat_params.numel()
        self._g = torch.zeros(n, dtype=torch.float32, device=dev)
        # The moments (flat, unlike the parameters they belong to) and the float64 device-side counters live
        # OUTSIDE `self.state`: torch.optim.Optimizer.load_state_dict casts every floating state tensor to its
        # parameter's dtype, which would hand the kernel a float32 buffer where it reads doubles.
        self.exp_avg = torch.zeros(n, dtype=torch.float32, device=dev)
        self.exp_avg_sq = torch.zeros(n, dtype=torch.float32, device=dev)
        self.device_state = torch.zeros(4, dtype=torch.float64, device=dev)   # step, beta1^t, beta2^t, ticket
        self._attach_grads()

    def state_dict(self):
        """torch's layout plus `fused`: the flat moments and the float64 counters, dtypes preserved."""
        sd = super().state_dict()
        sd["fused"] = {"exp_avg": self.exp_avg.clone(), "exp_avg_sq": self.exp_avg_sq.clone(),
                       "device_state": self.device_state.clone()}
        return sd

    def load_state_dict(self, state_dict):
        sd = dict(state_dict)
        fused = sd.pop("fused", None)
        super().load_state_dict(sd)
        self._params = self.param_groups[0]["params"]
        if fused is not None:
            for name in ("exp_avg", "exp_avg_sq", "device_state"):
                dst, src = getattr(self, name), fused[name]
                if src.shape != dst.shape or src.dtype != dst.dtype:
                    raise ValueError("FusedAdam.load_state_dict: %s is %s %s, expected %s %s"
                                     % (name, tuple(src.shape), src.dtype, tuple(dst.shape), dst.dtype))
                dst.copy_(src)

    def _intact(self):
        """every `.grad` is still the view this optimizer attached (identity checks: the per-step host path)"""
        views = getattr(self, "_views", None)
        return views is not None and all(p.grad is v for p, v in zip(self._params, views))

    def _attach_grads(self):
        if self._intact():
            return
        off = 0
        for p in self._params:
            n = p.numel()
            if p.grad is None or p.grad.data_ptr() != self._g.data_ptr() + 4 * off:
                p.grad = self._g[off:off + n].view(p.shape)
            off += n
        self._views = [p.grad for p in self._params]

    def zero_grad(self, set_to_none=True):
        """Zeroes the flat gradient; `.grad` stay views into it (one memset instead of ten)."""
        self._g.zero_()
        self._attach_grads()

    def flat_grad(self):
        return self._g

    def _gather(self):
        if self._intact():
            return
        off = 0
        for p in self._params:
            n = p.numel()
            seg = self._g[off:off + n]
            if p.grad is None:
                seg.zero_()
            elif p.grad.data_ptr() != seg.data_ptr():
                seg.copy_(p.grad.reshape(-1))
            off += n

    @property
    def step_count(self):
        return int(self.device_state[0].item())

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._gather()
        grp = self.param_groups[0]
        dev = self._x.device
        with torch.cuda.device(dev):
            _check(self.lib.pinn_adam_step(self._x.data_ptr(), self._g.data_ptr(), self.exp_avg.data_ptr(),
                                           self.exp_avg_sq.data_ptr(), self.device_state.data_ptr(), self._x.numel(),
                                           float(grp["lr"]), float(grp["betas"][0]), float(grp["betas"][1]),
                                           float(grp["eps"]), float(grp["weight_decay"]), 1 if grp["decoupled"] else 0,
                                           ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)),
                   "pinn_adam_step")
        return loss


def _flat(t):
    """`t`'s elements in the order in which they lie in memory, as a 1-D view; None where they have gaps or overlap."""
    if not t.is_contiguous():
        expect = 1
        for size, stride in sorted(zip(t.shape, t.stride()), key=lambda x: (x[1], x[0])):
            if size != 1 and stride != expect:
                return None
            expect *= size
    return t.as_strided((t.numel(),), (1,), t.storage_offset())


class _TensorList:
    """Tensors, or with `of_grads` the gradients of those that have one (2: to be written to), as the C interface takes them: host arrays of addresses, lengths
    and types.  `back`: (tensor, copy) of those whose memory has gaps or overlaps, the copy is what the arrays name."""

    def __init__(self, tensors, of_grads=0):
        n = len(tensors)
        self.x, self.numel, self.dtype = (ctypes.c_uint64 * n)(), (ctypes.c_int64 * n)(), (ctypes.c_int32 * n)()
        at = ctypes.addressof(self.x), ctypes.addressof(self.numel), ctypes.addressof(self.dtype)
        self.n, other, index, total = load_tensorlist().describe(tensors, of_grads, *at)
        self.device = None if index is None else torch.device("cuda", index)
        self.back = []
        for k, i in other:
            t = tensors[i].grad.detach() if of_grads else tensors[i].detach()
            self.back.append((t, t.contiguous()))
            self.x[k] = self.back[-1][1].data_ptr()
        self.partials = None                            # the call's own workspace
        if index is not None and (self.n > NORM_SMALL_TENSORS or total > NORM_SMALL_ELEMENTS):
            self.partials, room = _partials(self.n, self.device)
            self.args = self.x, self.numel, self.dtype, self.n, self.partials.data_ptr(), room
        else:
            self.args = self.x, self.numel, self.dtype, self.n, None, 0


def _partials(n, device):
    """(room for partial sums, its length)"""
    room = load_library().pinn_grad_norm_partials(n)
    return torch.empty(room, dtype=torch.float64, device=device), room


class _Place:
    """where a tensor's elements lie, as numpy is told it: nothing is read"""

    def __init__(self, t):
        size = t.element_size()
        self.begin = t.data_ptr()
        self.end = self.begin + size * (1 + sum(st * (n - 1) for n, st in zip(t.shape, t.stride())))     # torch's strides are never negative
        self.numel = t.numel()
        self.strides = tuple(size * st for st in t.stride())
        self.__array_interface__ = dict(version=3, shape=tuple(t.shape), typestr="<i%d" % size, data=(self.begin, True), strides=self.strides)


def _share_memory(tensors):
    """Do two of the tensors have an element in common?  Exact for any strides: gradients may lie between each other's elements."""
    places = sorted((_Place(t) for t in tensors if t.numel()), key=lambda p: p.begin)
    first, end = 0, 0
    for i, p in enumerate(places):                      # runs of tensors whose extents hang together
        if p.begin >= end:
            if _run_shares(places[first:i]):
                return True
            first = i
        end = max(end, p.end)
    return _run_shares(places[first:])


def _run_shares(places):
    """Two ways.  numpy compares two arrays in 0.7 us whatever their size (where their strides are simple: the search is cut off at
    10^5 steps); marking every element takes about 20 ns for each.  512 columns of 100 elements: 90 ms by pairs, 4.8 by marks; 65 of 1000: 1.6 and
    1.3; 2 of 10^7: 0.014 and 250."""
    begins = [p.begin for p in places]
    meets = [bisect.bisect_left(begins, p.end) for p in places]                     # the first behind those that begin before p ends
    if 32 * sum(m - i - 1 for i, m in enumerate(meets)) <= sum(p.numel for p in places):
        try:
            arrays = [np.asarray(p) for p in places]
            return any(np.shares_memory(a, b, max_work=100000) for i, a in enumerate(arrays) for b in arrays[i + 1:meets[i]])
        except RuntimeError:                            # TooHardError
            pass
    if len(places) < 2:
        return False
    taken = np.zeros((max(p.end for p in places) - begins[0]) // 2, dtype=bool)     # two bytes each: a 16-bit element or half of another
    for p in places:
        a = np.asarray(p)
        mine = np.ndarray(a.shape + (a.itemsize // 2,), bool, taken, (p.begin - begins[0]) // 2, tuple(st // 2 for st in p.strides) + (1,))
        if mine.any():
            return True
        mine[...] = True
    return False


def _runs(rows, numel, chunk):
    """`rows`, tensors of `numel` elements, cut into what one launch of the step takes"""
    runs, chunks = [], 0
    for i, n in zip(rows, numel):
        more = -(-n // chunk)
        if more > ADAMW_MAX_CHUNKS:
            raise ValueError("parameter %d has %d elements, a launch takes %d" % (i, n, ADAMW_MAX_CHUNKS * chunk))
        if not runs or len(runs[-1]) == ADAMW_MAX_TENSORS or chunks + more > ADAMW_MAX_CHUNKS:
            runs.append([])
            chunks = 0
        runs[-1].append(i)
        chunks += more
    return runs


_SHARED = "two of the gradients share memory: scaling them in place would scale it twice"


def _as_list(tensors):
    return [tensors] if torch.is_tensor(tensors) else list(tensors)


def grad_norm(tensors):
    """2-norm over all elements of all `tensors` (one, or an iterable; float32, bfloat16, float16, mixed as they come): a 0-dim
    float32 tensor on their device.  Squares and sums are float64, in a fixed order: the same inputs give the same bits, and
    no float32 value overflows or vanishes on the way (a norm beyond float32's largest value reads infinity).  An empty list gives 0."""
    tensors = _as_list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    lst = _TensorList(tensors)
    norm = torch.empty((), dtype=torch.float32, device=lst.device)
    with _on(lst.device):
        _check(load_library().pinn_grad_norm(*lst.args, norm.data_ptr(), _cur_stream(norm)), "pinn_grad_norm")
    return norm


def clip_grad_norm_(parameters, max_norm, error_if_nonfinite=False):
    """Scales the gradients of `parameters` in place so that their global 2-norm is at most `max_norm`, and returns the norm
    they had (0-dim float32, on the device): torch.nn.utils.clip_grad_norm_ in two launches per 250 tensors (one for few elements),
    without a copy of the gradients.  The factor is min(1, max_norm / (norm + 1e-6)); with a norm that is not finite it is 0 or NaN, as
    there (the factor goes by the float64 norm, also where the one returned is beyond float32 and reads infinity);
    `error_if_nonfinite` raises instead and waits for the GPU.  Gradients that share memory are refused (ValueError), and so is
    a third argument that is not a truth value (TypeError): there is no `norm_type`."""
    if not isinstance(error_if_nonfinite, (bool, np.bool_)):
        raise TypeError("error_if_nonfinite is %r: True or False is needed (the norm is always the 2-norm)" % (error_if_nonfinite,))
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError("max_norm is %r: 0 or more is needed" % max_norm)
    parameters = _as_list(parameters)
    lst = _TensorList(parameters, of_grads=2)
    if lst.n == 0:
        return torch.tensor(0.0)
    if any(0 in (st for sz, st in zip(g.shape, g.stride()) if sz > 1) for g, _ in lst.back):
        raise ValueError("a gradient that was expanded cannot be scaled in place")
    # the C entry compares the memory that it scales; of these that is a copy
    if lst.back and _share_memory([p.grad for p in parameters if p.grad is not None]):
        raise ValueError(_SHARED)
    norm = torch.empty((), dtype=torch.float32, device=lst.device)
    lib = load_library()
    with _on(lst.device):
        stream = _cur_stream(norm)
        if error_if_nonfinite:
            _check(lib.pinn_grad_norm(*lst.args, norm.data_ptr(), stream), "pinn_grad_norm")
            if not torch.isfinite(norm):
                raise RuntimeError("the gradients' norm is %s: they were not clipped" % norm.item())
        rc = lib.pinn_grad_clip(*lst.args, max_norm, norm.data_ptr(), stream)
        if rc == ERR_OVERLAP:
            raise ValueError(_SHARED)
        _check(rc, "pinn_grad_clip")
        for g, c in lst.back:
            g.copy_(c)
    return norm


class GroupedAdamW(torch.optim.Optimizer):
    """AdamW over many tensors at once: one launch per 240 tensors (or 2^24 chunks of 1024 elements, 2048 with 8-bit moments) of one
    group and type.

    torch.optim.AdamW's constructor arguments and update rule (decoupled weight decay, no amsgrad; `weight_decay=0` is Adam), plus

    state_bits      32: moments in float32.  8: one byte each, in blocks of 128 elements with a power-of-two scale (2 1/64 bytes
                    per weight instead of 8): exp_avg keeps 4 significant bits and a range of 2^17 in a block, exp_avg_sq 4 bits and 2^33;
                    rounded by an even sequence, so that small changes are not lost.  Both hold 1.75 * 2^127 at most: an exp_avg_sq
                    beyond (gradients above 1.7e19 that last) stays at that.  A gradient that is not finite makes its whole block's moments NaN.
    max_norm        clip the gradients' global 2-norm (over all groups, tensors without a gradient left out) inside the step; the gradients themselves
                    stay as they are.  `grad_norm` holds the norm of the last step, on the device.
    skip_nonfinite  a step whose gradient norm is not finite, as `grad_norm` gives it, changes nothing, counters included (decided on the device).
    master_weights  bfloat16 and float16 parameters are the rounded copy of float32 weights held here (`master`); after writing to
                    such a parameter from outside call `sync_master()`.

    Parameters are dense float32, bfloat16 or float16 CUDA tensors on one device that do not share memory, in any number of groups;
    gradients have their parameter's type.  A parameter whose `.grad` is None is left alone and its step count with it.  Step counts and powers of beta
    live on the device (`device_state`), so a captured step replays; learning rates and the like are taken at the call.
    After a change of betas the bias correction takes the product of the betas that were used.

    Moments lie in flat buffers in the order of the parameters, each at the next multiple of 128 elements, in the order its
    parameter has in memory: `moments()`."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, max_norm=None, skip_nonfinite=False,
                 master_weights=False):
        if state_bits not in (8, 32):
            raise ValueError("state_bits is %r: 8 or 32 is needed" % (state_bits,))
        if max_norm is not None and not float(max_norm) >= 0.0:
            raise ValueError("max_norm is %r: 0 or more is needed" % (max_norm,))
        self.state_bits, self.max_norm, self.skip_nonfinite = state_bits, None if max_norm is None else float(max_norm), bool(skip_nonfinite)
        self._planned = False
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        for grp in self.param_groups:
            self._hyper(grp)
        self._chunk = ADAMW_CHUNK32 if state_bits == 32 else ADAMW_CHUNK8
        self._params = [p for grp in self.param_groups for p in grp["params"]]
        if not self._params:
            raise ValueError("the groups have no parameter")
        self.device = self._params[0].device
        if self.device.type != "cuda":
            raise NativeError("GroupedAdamW needs parameters on an AMD GPU, got %s; there is no CPU fallback (use torch.optim.AdamW)" % self.device)
        self._check_params()
        self.lib, self._native = load_library(), load_tensorlist()
        self._plan(bool(master_weights))
        self._planned = True

    def add_param_group(self, param_group):
        if self._planned:
            raise ValueError("GroupedAdamW takes all parameter groups when it is made")
        super().add_param_group(param_group)

    def __getstate__(self):
        # torch's would leave out the moments and the tables, all that is not in `state`
        raise TypeError("GroupedAdamW cannot be copied or pickled: make another and load_state_dict(state_dict())")

    @staticmethod
    def _hyper(grp):
        lr, (b1, b2), eps, wd = float(grp["lr"]), grp["betas"], float(grp["eps"]), float(grp["weight_decay"])
        if not (lr >= 0.0 and eps >= 0.0 and wd >= 0.0 and 0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError("lr %r, betas %r, eps %r, weight_decay %r: none may be negative, betas are below 1"
                             % (grp["lr"], grp["betas"], grp["eps"], grp["weight_decay"]))
        return lr, float(b1), float(b2), eps, wd

    def _check_params(self):
        spans = []
        for i, p in enumerate(self._params):
            if p.layout is not torch.strided or p.dtype not in DTYPE_CODES:
                raise ValueError("parameter %d is %s, %s: dense float32, bfloat16 or float16 is needed" % (i, p.layout, p.dtype))
            if p.device != self.device:
                raise ValueError("parameters lie on one device, got %s and %s" % (self.device, p.device))
            if _flat(p) is None:
                raise ValueError("parameter %d (shape %s, strides %s) has gaps or overlaps in memory" % (i, tuple(p.shape), p.stride()))
            if p.numel():
                spans.append((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()))
        spans.sort()
        if any(b[0] < a[1] for a, b in zip(spans, spans[1:])):
            raise ValueError("two parameters share memory")

    def _plan(self, master_weights):
        """Flat state, and the device tables of each launch."""
        dev, at = self.device, 0
        self.offsets = []
        for p in self._params:
            self.offsets.append(at)
            at += -(-p.numel() // ADAMW_BLOCK) * ADAMW_BLOCK
        self.state_numel = at
        kind = torch.float32 if self.state_bits == 32 else torch.uint8
        self.exp_avg, self.exp_avg_sq = (torch.zeros(at, dtype=kind, device=dev) for _ in range(2))
        self.exp_avg_scale = self.exp_avg_sq_scale = self.master = None
        if self.state_bits == 8:
            self.exp_avg_scale, self.exp_avg_sq_scale = (torch.zeros(at // ADAMW_BLOCK, dtype=torch.uint8, device=dev) for _ in range(2))
        if master_weights and any(p.dtype != torch.float32 for p in self._params):
            self.master = torch.zeros(at, dtype=torch.float32, device=dev)
            self.sync_master()
        self.device_state = torch.ones((len(self._params), 3), dtype=torch.float64, device=dev)    # step, beta1^step, beta2^step
        self.device_state[:, 0] = 0.0
        self._ticket = torch.zeros(ADAMW_TICKET_WORDS, dtype=torch.int32, device=dev)
        self._norm = torch.zeros((), dtype=torch.float32, device=dev)
        # launches: consecutive runs of the parameters sorted by group and type
        plan, first = [], 0
        for grp in self.param_groups:
            rows = range(first, first + len(grp["params"]))
            first += len(grp["params"])
            for dt in DTYPE_CODES:
                mine = [i for i in rows if self._params[i].dtype == dt]
                plan += [(grp, dt, run) for run in _runs(mine, [self._params[i].numel() for i in mine], self._chunk)]
        order = [i for _, _, rows in plan for i in rows]
        n = len(order)
        self._ordered = [self._params[i] for i in order]
        self._numel = (ctypes.c_int64 * n)(*(p.numel() for p in self._ordered))
        self._dtype = (ctypes.c_int32 * n)(*(DTYPE_CODES[p.dtype] for p in self._ordered))
        self._p = (ctypes.c_uint64 * n)(*(p.data_ptr() for p in self._ordered))      # as they were checked
        self._g, self._count = (ctypes.c_uint64 * n)(), (ctypes.c_int64 * n)()
        self._gather_args = tuple(ctypes.addressof(x) for x in (self._numel, self._dtype, self._p, self._g, self._count))
        self._launches, first = [], 0
        for grp, dt, rows in plan:
            self._launches.append(self._launch(grp, dt, rows, first))
            first += len(rows)

    def _launch(self, grp, dtype, rows, first):
        chunk = self._chunk
        numel = np.array([self._params[i].numel() for i in rows], dtype=np.int64)
        count = -(-numel // chunk)
        k = np.repeat(np.arange(len(rows)), count)
        parts = np.zeros(len(k), dtype=ADAMW_CHUNK_DTYPE)
        parts["base"] = (np.arange(len(k)) - (np.cumsum(count) - count)[k]) * chunk
        parts["place"] = np.array([self.offsets[i] for i in rows], dtype=np.int64)[k] + parts["base"]
        parts["count"] = np.minimum(numel[k] - parts["base"], chunk)
        parts["tensor"], parts["row"] = k, np.array(rows)[k]
        chunks = torch.from_numpy(parts.view(np.uint8)).to(self.device)
        where = torch.tensor(rows, dtype=torch.int32, device=self.device)
        d = PinnAdamWGroup()
        d.chunks, d.rows, d.n_chunks, d.n_tensors = chunks.data_ptr(), where.data_ptr(), len(parts), len(rows)
        d.dtype, d.state_bits = DTYPE_CODES[dtype], self.state_bits
        d.exp_avg, d.exp_avg_sq, d.device_state, d.ticket = (t.data_ptr() for t in (self.exp_avg, self.exp_avg_sq, self.device_state, self._ticket))
        if self.state_bits == 8:
            d.exp_avg_scale, d.exp_avg_sq_scale = self.exp_avg_scale.data_ptr(), self.exp_avg_sq_scale.data_ptr()
        if self.master is not None and dtype != torch.float32:
            d.master = self.master.data_ptr()
        d.norm = self._norm.data_ptr()
        return dict(grp=grp, desc=d, ref=ctypes.byref(d), rows=rows, p=ctypes.addressof(self._p) + 8 * first,
                    g=ctypes.addressof(self._g) + 8 * first, tables=(chunks, where))

    @torch.no_grad()
    def sync_master(self):
        """The float32 weights take the parameters' present values."""
        if self.master is None:
            return
        for p, at in zip(self._params, self.offsets):
            self.master[at:at + p.numel()].copy_(_flat(p))

    @property
    def grad_norm(self):
        """norm of the gradients of the last step (0-dim float32, overwritten by the next; 0 where no parameter had one); steps without `max_norm` or `skip_nonfinite` do not form it"""
        return self._norm

    def moments(self):
        """(exp_avg, exp_avg_sq) as flat float32 tensors in the order of the flat state: the buffers themselves, or with 8 bits what they stand for."""
        if self.state_bits == 32:
            return self.exp_avg, self.exp_avg_sq
        m = torch.empty(self.state_numel, dtype=torch.float32, device=self.device)
        v = torch.empty_like(m)
        with _on(self.device):
            _check(self.lib.pinn_adamw_moments(self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr(), self.exp_avg_scale.data_ptr(),
                                               self.exp_avg_sq_scale.data_ptr(), m.data_ptr(), v.data_ptr(), self.state_numel, _cur_stream(m)),
                   "pinn_adamw_moments")
        return m, v

    def _held(self):
        names = ["exp_avg", "exp_avg_sq", "device_state"]
        names += ["exp_avg_scale", "exp_avg_sq_scale"] if self.state_bits == 8 else []
        return names + (["master"] if self.master is not None else [])

    def state_dict(self):
        """torch's layout plus `fused`: the flat state, types preserved."""
        sd = super().state_dict()
        sd["fused"] = {name: getattr(self, name).clone() for name in self._held()}
        return sd

    def load_state_dict(self, state_dict):
        sd = dict(state_dict)
        fused = sd.pop("fused", {})                      # another optimizer's moments would be dropped without a word
        if sorted(fused) != sorted(self._held()):
            raise ValueError("GroupedAdamW.load_state_dict: the state has %s, expected %s" % (sorted(fused), sorted(self._held())))
        for name in self._held():
            dst, src = getattr(self, name), fused[name]
            if src.shape != dst.shape or src.dtype != dst.dtype:
                raise ValueError("GroupedAdamW.load_state_dict: %s is %s %s, expected %s %s"
                                 % (name, tuple(src.shape), src.dtype, tuple(dst.shape), dst.dtype))
        super().load_state_dict(sd)
        first = 0
        for grp in self.param_groups:                   # torch has replaced the groups' dicts
            for launch in self._launches:
                if first <= launch["rows"][0] < first + len(grp["params"]):
                    launch["grp"] = grp
            first += len(grp["params"])
        for name in self._held():
            getattr(self, name).copy_(fused[name])

    def step(self, closure=None):
        """One step of every parameter that has a gradient; `closure` is called first, as in torch, and its loss returned."""
        # torch wraps every optimizer's `step` for its profiler's label and for step hooks, which takes as long as all the rest of a small
        # net's step (6.7 us): here the wrapper is used where one of them is
        if (self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _hooks._global_optimizer_pre_hooks
                or _hooks._global_optimizer_post_hooks or torch.autograd._profiler_enabled()):
            return self._hooked_step(closure)
        return self._step(closure)

    step.hooked = True

    def _step(self, closure):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        hyper = {id(grp): self._hyper(grp) for grp in self.param_groups}
        given, other, moved = self._native.gather(self._ordered, *self._gather_args)
        if moved:
            self._p[0], first = 0, self._p[0]           # found wanting, they are looked at again in the next step
            self._check_params()
            self._p[0] = first
        clipped = self.max_norm is not None or self.skip_nonfinite
        if not given:
            if clipped:
                self._norm.zero_()                      # the norm of no gradients, not the last step's
            return loss
        keep = []
        for i in other:                                 # a gradient in another order in memory than its parameter
            p = self._ordered[i]
            keep.append(torch.empty_strided(p.shape, p.stride(), dtype=p.dtype, device=p.device).copy_(p.grad.detach()))
            self._g[i] = keep[-1].data_ptr()
        with _on(self.device):
            stream = _cur_stream(self._norm)
            partials, n_partials = None, 0
            if clipped:
                partials, room = _partials(len(self._ordered), self.device)
                found = ctypes.c_int32()
                _check(self.lib.pinn_grad_sumsq(self._g, self._count, self._dtype, len(self._ordered), partials.data_ptr(), room,
                                                ctypes.byref(found), stream), "pinn_grad_sumsq")
                n_partials = found.value
            for launch in self._launches:
                d = launch["desc"]
                d.lr, d.beta1, d.beta2, d.eps, d.weight_decay = hyper[id(launch["grp"])]
                d.partials, d.n_partials = partials.data_ptr() if n_partials else None, n_partials
                d.max_norm, d.skip_nonfinite = -1.0 if self.max_norm is None else self.max_norm, self.skip_nonfinite
                _check(self.lib.pinn_adamw_group_step(launch["ref"], launch["p"], launch["g"], stream), "pinn_adamw_group_step")
        return loss

    _hooked_step = torch.optim.Optimizer.profile_hook_step(_step)

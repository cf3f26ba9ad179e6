"""Operators of a training step beside the collectives, on torch tensors (include/msccl_amd_ops.h).

Between ReduceScatter and AllGather: SquareSum, whose result AllReduce sums over the ranks for gradient
clipping, and AdamW, one step over all of a rank's tensors with its states in 32 or in 8 bits.
sharded_step makes the whole chain on communicators.  Beside AllToAll: the counts of the tokens each
expert gets and the experts' balance loss (balance_stats, balance_all_reduce over the ranks,
balance_loss) with its gradient (balance_backward).

Every call is enqueued on the current torch stream of its tensors' device and returns; nothing waits
for the device but the creation of a plan.  Calls may be captured into a graph (plans are made before
the capture, and must outlive the graph, as their tensors must).  Wrong arguments raise ValueError or
TypeError here, or NcclError from the library.
"""
import ctypes
import struct
import warnings
from typing import Optional, Sequence, Union

import torch

from . import BFLOAT16, FLOAT16, FLOAT32, FLOAT64, INT32, INT64, Comm, NcclError, _check, group, lib

_TYPES = {torch.float32: FLOAT32, torch.float16: FLOAT16, torch.bfloat16: BFLOAT16}
_INDEX = {torch.int32: INT32, torch.int64: INT64}
_SCORES = {"softmax": 0, "sigmoid": 1}
_ROUNDINGS = {"nearest": 0, "stochastic": 1}
STATE_BLOCK = 256  # elements that share a scale in 8-bit states


# mscclAmdAdamWTensor_t: param, grad, master, expAvg, expAvgSq, expAvgScale, expAvgSqScale, count, weightDecay, lrScale
_TENSOR = struct.Struct("@PPPPPPPNdd")
# mscclAmdRouter_t: logits, type, tokens, experts, logitStride, index, indexType, topK, indexStride, valid, score
_ROUTER = struct.Struct("@PiNNNPiNNPi")


_L = None


def _lib():
    global _L
    if _L is None:
        L = lib()
        vp, i, sz, d = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t, ctypes.c_double
        L.mscclAmdSquareSumBytes.argtypes = [sz]
        L.mscclAmdSquareSumBytes.restype = sz
        L.mscclAmdSquareSumCreate.argtypes = [ctypes.POINTER(vp), vp, vp, sz, i, vp, sz, vp]
        L.mscclAmdSquareSumWorkspace.argtypes = [vp]
        L.mscclAmdSquareSumWorkspace.restype = sz
        L.mscclAmdSquareSum.argtypes = [vp, vp, vp, sz, vp]
        L.mscclAmdSquareSumDestroy.argtypes = [vp]
        L.mscclAmdAdamWBytes.argtypes = [sz]
        L.mscclAmdAdamWBytes.restype = sz
        L.mscclAmdAdamWCreate.argtypes = [ctypes.POINTER(vp), ctypes.c_char_p, sz, i, i, i, vp, vp, sz, vp]
        L.mscclAmdAdamWSetRounding.argtypes = [vp, i, ctypes.c_uint64]
        L.mscclAmdAdamWSetGrads.argtypes = [vp, vp, sz, vp]
        L.mscclAmdAdamWStep.argtypes = [vp, d, vp, d, d, d, d, vp, d, vp]
        L.mscclAmdAdamWCheck.argtypes = [d, d, d, d, d, d]
        L.mscclAmdAdamWDestroy.argtypes = [vp]
        L.mscclAmdBalanceWorkspace.argtypes = [sz, sz]
        L.mscclAmdBalanceWorkspace.restype = sz
        L.mscclAmdBalanceStats.argtypes = [ctypes.c_char_p, vp, vp, vp, sz, vp]
        L.mscclAmdBalanceLoss.argtypes = [vp, vp, sz, sz, d, vp, vp]
        L.mscclAmdBalanceBackward.argtypes = [ctypes.c_char_p, vp, d, vp, vp, sz, i, vp]
        _L = L
    return _L


def _stream(device) -> int:
    """The handle of the device's current stream (without a Stream object: it sits on every call's path)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _elsewhere(device) -> bool:
    """Whether another device is the current one (the launches go to the current device)."""
    return torch._C._cuda_getDevice() != device.index


def _flat(t, what: str, dtypes, device=None, numel: Optional[int] = None, i: Optional[int] = None) -> None:
    """A contiguous device tensor of one of `dtypes`, or an exception."""
    if (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in dtypes and t.is_contiguous() and
            (device is None or t.device == device) and (numel is None or t.numel() == numel)):
        return
    if i is not None:
        what = "%s[%d]" % (what, i)
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch tensor" % what)
    if t.device.type != "cuda":
        raise ValueError("%s must be on a GPU" % what)
    if t.dtype not in dtypes:
        raise TypeError("%s: %s is not one of %s" % (what, t.dtype, ", ".join(str(x) for x in dtypes)))
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % what)
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, not %s" % (what, t.device, device))
    raise ValueError("%s has %d elements, not %d" % (what, t.numel(), numel))


def _span(tensors):
    """The first address of these tensors and the one behind the last (None: they are all empty)."""
    ends = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors if t.numel()]
    return (min(a for a, _ in ends), max(b for _, b in ends)) if ends else None


def _inside(span, at: int, nbytes: int) -> bool:
    return span is None or (at <= span[0] and span[1] <= at + nbytes)


def _changed(tensors) -> None:
    """Tells autograd that a kernel wrote these: a graph that holds their old values refuses to use the new ones."""
    torch._C._increment_version(tensors)


def _versions(tensors):
    """One of these for each version counter (views share their base's)."""
    seen = {}
    for t in tensors:
        base = t if t._base is None else t._base
        seen.setdefault(id(base), (t, base))   # (held: a number may be another's once its object is gone)
    return [t for t, _ in seen.values()]


class _Plan:
    """A plan's handle, its device memory and the tensors whose addresses it holds."""
    _destroy = ""

    def __init__(self):
        self.handle = ctypes.c_void_p()
        self._weights = None

    def _memory(self, device, nbytes: int):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("make the plan before the capture")
        self.device = device
        self.table = torch.empty(max(8, nbytes), dtype=torch.uint8, device=device)
        self._streams = {}   # those that had a call

    def _ready(self):
        # the table was written on this stream; the plan may be used on any
        self._live()
        torch.cuda.current_stream(self.device).synchronize()

    def _held(self):
        return [self.table] + self.tensors

    def _live(self) -> int:
        """The stream of a call on the plan."""
        if not self.handle:
            raise ValueError("the plan is closed")
        s = _stream(self.device)
        if s not in self._streams:
            # whoever drops the plan or its tensors: their memory is not used again before this stream is done
            self._streams[s] = stream = torch.cuda.current_stream(self.device)
            for t in _versions(self._held()):
                t.record_stream(stream)
        return s

    def close(self) -> None:
        """Ends the plan.  The device must be done with its calls."""
        if self.handle:
            h, self.handle = self.handle, ctypes.c_void_p()
            _check(getattr(_lib(), self._destroy)(h), self._destroy)
        self.table = None
        self.tensors = self._weights = self._captured = None

    def __del__(self):
        try:
            if self.handle:  # host memory alone: no device call, whatever the moment
                getattr(_lib(), self._destroy)(self.handle)
        except Exception:  # noqa: BLE001
            pass


class SquareSum(_Plan):
    """The sum of the squares of all elements of `tensors` (one type: float32, float16 or bfloat16; one
    device; contiguous).  Calling it returns a float64 tensor of one element."""
    _destroy = "mscclAmdSquareSumDestroy"

    def __init__(self, tensors: Sequence[torch.Tensor]):
        super().__init__()
        self.tensors = list(tensors)
        if not self.tensors:
            raise ValueError("no tensors")
        first = self.tensors[0]
        dev = getattr(first, "device", None)
        dtypes = (first.dtype,) if getattr(first, "dtype", None) in _TYPES else tuple(_TYPES)
        for i, t in enumerate(self.tensors):
            _flat(t, "tensors", dtypes, dev, None, i)
        n = len(self.tensors)
        L = _lib()
        with torch.cuda.device(first.device):
            self._memory(first.device, L.mscclAmdSquareSumBytes(n))
            ptrs = (ctypes.c_void_p * n)(*[t.data_ptr() for t in self.tensors])
            counts = (ctypes.c_size_t * n)(*[t.numel() for t in self.tensors])
            _check(L.mscclAmdSquareSumCreate(ctypes.byref(self.handle), ptrs, counts, n, _TYPES[first.dtype],
                                             self.table.data_ptr(), self.table.numel(), _stream(first.device)),
                   "mscclAmdSquareSumCreate")
            self._ready()
        self._scratch = L.mscclAmdSquareSumWorkspace(self.handle)
        self.span = _span(self.tensors)

    def __call__(self, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        stream = self._live()
        if out is not None:
            _flat(out, "out", (torch.float64,), self.device, 1)
        dev = self.device
        if _elsewhere(dev):
            with torch.cuda.device(dev):
                return self(out)
        # scratch of this call's own: calls on several streams, or in several graphs, do not meet in it
        scratch = torch.empty(self._scratch, dtype=torch.uint8, device=dev) if self._scratch else None
        given = out is not None
        if not given:
            out = torch.empty(1, dtype=torch.float64, device=dev)
        rc = _lib().mscclAmdSquareSum(self.handle, out.data_ptr(), scratch.data_ptr() if self._scratch else None,
                                      self._scratch, stream)
        if rc:
            raise NcclError(rc, "mscclAmdSquareSum")
        if given:
            _changed((out,))
        return out


def adamw_state(param: torch.Tensor, bits: int = 32):
    """The state of `param` before its first step: (exp_avg, exp_avg_sq), or with bits=8
    (exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale), all zeros."""
    n, dev = param.numel(), param.device
    if bits == 32:
        return tuple(torch.zeros(n, dtype=torch.float32, device=dev) for _ in range(2))
    if bits != 8:
        raise ValueError("states of %r bits (32 or 8)" % (bits,))
    return (tuple(torch.zeros(n, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn) for _ in range(2)) +
            tuple(torch.zeros(-(-n // STATE_BLOCK), dtype=torch.float32, device=dev) for _ in range(2)))


def dequantize_state(code: torch.Tensor, scale: torch.Tensor, second: bool = False) -> torch.Tensor:
    """The 32-bit values of an 8-bit state (second: of exp_avg_sq, whose codes hold square roots)."""
    x = code.reshape(-1).float() * scale.repeat_interleave(STATE_BLOCK)[:code.numel()]
    return x.square() if second else x


class AdamW(_Plan):
    """AdamW over many tensors of one device in one launch.

    params and grads: contiguous, one type each (float32, float16, bfloat16); masters: None, or the
    weights in float32 (read in place of params, both are written).  exp_avgs, exp_avg_sqs: float32, or
    torch.float8_e4m3fn with exp_avg_scales and exp_avg_sq_scales, one float32 for each 256 elements of
    a tensor (the last may be shorter); adamw_state makes them.  step: one int64, the steps taken so far,
    this plan's own.  weight_decay, lr_scale: a number, or one for each tensor.  Tensors may have any size
    and start anywhere; they must not overlap (a weight that layers share is listed once).  Steps of one
    plan must be ordered after each other.

    rounding, seed: how 8-bit states are rounded.  "stochastic" is right in the mean over any number of
    steps; one element's sqrt(exp_avg_sq) is then within about a sixth of the 32-bit state's.  "nearest" is
    closer within a step but never follows what changes by less than half a code's step (3.1 to 6.3 %) in
    each: second moments neither decay by themselves nor stay when a neighbour's growth raises their scale,
    and drift to many times their value over thousands of steps at beta2 of 0.94 and more (mscclAmdAdamWSetRounding).
    None is nearest, with a warning at the first such step."""
    _destroy = "mscclAmdAdamWDestroy"

    def __init__(self, params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
                 exp_avg_sqs: Sequence[torch.Tensor], step: torch.Tensor, masters: Optional[Sequence[torch.Tensor]] = None,
                 exp_avg_scales: Optional[Sequence[torch.Tensor]] = None,
                 exp_avg_sq_scales: Optional[Sequence[torch.Tensor]] = None,
                 weight_decay: Union[float, Sequence[float]] = 0.0, lr_scale: Union[float, Sequence[float]] = 1.0,
                 rounding: Optional[str] = None, seed: int = 0):
        super().__init__()
        n = len(params)
        if not n:
            raise ValueError("no tensors")
        dev = params[0].device
        bits = 8 if exp_avgs and exp_avgs[0].dtype == torch.float8_e4m3fn else 32
        if bits == 8 and (exp_avg_scales is None or exp_avg_sq_scales is None):
            raise ValueError("8-bit states need their scales")
        if bits == 32 and (exp_avg_scales is not None or exp_avg_sq_scales is not None):
            raise ValueError("32-bit states have no scales")
        if rounding is not None and rounding not in _ROUNDINGS:
            raise ValueError("rounding %r is not one of %s" % (rounding, ", ".join(_ROUNDINGS)))
        if rounding == "stochastic" and bits != 8:
            raise ValueError("32-bit states are rounded to nearest")
        if not 0 <= seed < 1 << 64:
            raise ValueError("seed %r is not a 64-bit number" % (seed,))
        decay = list(weight_decay) if isinstance(weight_decay, (list, tuple)) else [weight_decay] * n
        rates = list(lr_scale) if isinstance(lr_scale, (list, tuple)) else [lr_scale] * n
        state = (torch.float8_e4m3fn,) if bits == 8 else (torch.float32,)
        lists = [("params", params, (params[0].dtype,) if params[0].dtype in _TYPES else tuple(_TYPES), 1),
                 ("grads", grads, tuple(_TYPES), 1), ("masters", masters, (torch.float32,), 1),
                 ("exp_avgs", exp_avgs, state, 1), ("exp_avg_sqs", exp_avg_sqs, state, 1),
                 ("exp_avg_scales", exp_avg_scales, (torch.float32,), STATE_BLOCK),
                 ("exp_avg_sq_scales", exp_avg_sq_scales, (torch.float32,), STATE_BLOCK)]
        for what, ts, dtypes, per in lists:
            if ts is None:
                continue
            if len(ts) != n:
                raise ValueError("%d %s for %d tensors" % (len(ts), what, n))
            for i, (t, p) in enumerate(zip(ts, params)):
                _flat(t, what, dtypes, dev, -(-p.numel() // per), i)
        if len(decay) != n or len(rates) != n:
            raise ValueError("weight_decay and lr_scale: a number, or one for each tensor")
        if any(g.dtype != grads[0].dtype for g in grads):
            raise TypeError("grads must have one type")
        _flat(step, "step", (torch.int64,), dev, 1)
        self.tensors = [list(ts) if ts is not None else None for _, ts, _, _ in lists] + [step]
        self._grad_type = grads[0].dtype
        self.param_span, self.grad_span = _span(params), _span(grads)
        at = [[t.data_ptr() for t in ts] if ts is not None else [0] * n for _, ts, _, _ in lists]
        rows = b"".join(_TENSOR.pack(*row, t.numel(), float(d), float(r))
                        for *row, t, d, r in zip(*at, params, decay, rates))
        L = _lib()
        with torch.cuda.device(dev):
            self._memory(dev, L.mscclAmdAdamWBytes(n))
            _check(L.mscclAmdAdamWCreate(ctypes.byref(self.handle), rows, n, _TYPES[params[0].dtype],
                                         _TYPES[grads[0].dtype], bits, step.data_ptr(), self.table.data_ptr(),
                                         self.table.numel(), _stream(dev)), "mscclAmdAdamWCreate")
            if rounding == "stochastic":
                _check(L.mscclAmdAdamWSetRounding(self.handle, _ROUNDINGS[rounding], seed), "mscclAmdAdamWSetRounding")
            self._ready()
        self._unsaid = bits == 8 and rounding is None
        self._weights = _versions(list(params) + list(masters or ()))
        self._captured = []

    def _held(self):
        return [self.table] + [t for ts in self.tensors[:-1] if ts for t in ts] + self.tensors[-1:]

    def set_grads(self, grads: Sequence[torch.Tensor]) -> None:
        """Other gradient tensors (same sizes and type) for the steps enqueued from now on; the earlier
        steps must be on the current stream or ordered before it.  Captured, it changes them at each replay
        and not before: the plan then keeps the earlier ones too."""
        stream = self._live()
        params = self.tensors[0]
        if len(grads) != len(params):
            raise ValueError("%d gradients for %d tensors" % (len(grads), len(params)))
        for i, g in enumerate(grads):
            _flat(g, "grads[%d]" % i, (self._grad_type,), self.device, params[i].numel())
        ptrs = (ctypes.c_void_p * len(grads))(*[g.data_ptr() for g in grads])
        with torch.cuda.device(self.device):
            _check(_lib().mscclAmdAdamWSetGrads(self.handle, ptrs, len(grads), stream), "mscclAmdAdamWSetGrads")
        for s in self._streams.values():
            for g in grads:
                g.record_stream(s)
        with torch.cuda.device(self.device):
            captured = torch.cuda.is_current_stream_capturing()
        if captured:   # until a replay the table holds the earlier ones, and every replay sets these again
            self._captured.append((self.tensors[1], list(grads)))
        self.tensors[1] = list(grads)
        self.grad_span = _span(grads)

    def _say(self, betas, level) -> None:
        """The warning of a plan that was told no rounding, once."""
        if betas[1] > 0.9375:   # a root of v decays by 1 - sqrt(beta2), half a code's step is 2^-5 or more
            self._unsaid = False
            warnings.warn("AdamW: second moments of 8 bits that are rounded to nearest drift over many steps with beta2 %g; "
                          "rounding=\"stochastic\" follows them (rounding=\"nearest\" says that this is meant)" % betas[1],
                          stacklevel=level)

    def _check_step(self, lr, betas, eps, grad_scale, max_norm) -> None:
        """What step and the library refuse, without a step."""
        if not self.handle:
            raise ValueError("the plan is closed")
        if isinstance(lr, torch.Tensor):
            _flat(lr, "lr", (torch.float32,), self.device, 1)
            lr = 0.0
        if max_norm is not None and not max_norm > 0:
            raise ValueError("max_norm must be above zero")
        _check(_lib().mscclAmdAdamWCheck(lr, betas[0], betas[1], eps, grad_scale, max_norm or 0.0), "mscclAmdAdamWCheck")
        if self._unsaid:   # (here, where a warning that is an error stops no collective)
            self._say(betas, 4)

    def step(self, lr: Union[float, torch.Tensor], betas=(0.9, 0.999), eps: float = 1e-8, grad_scale: float = 1.0,
             grad_square_sum: Optional[torch.Tensor] = None, max_norm: Optional[float] = None) -> None:
        """One step (the formulas: mscclAmdAdamWStep).  lr: a number, or a float32 tensor of one element,
        which a captured step reads at each replay.  grad_scale: a factor on the gradients (one over the
        ranks that were summed, or over a loss scale).  grad_square_sum: the square sum of the gradients as
        they are, over all ranks; if it is not finite the step changes nothing.  max_norm: clips to it."""
        stream = self._live()
        at = None
        if isinstance(lr, torch.Tensor):
            _flat(lr, "lr", (torch.float32,), self.device, 1)
            at, lr = lr.data_ptr(), 0.0
        total = None
        if grad_square_sum is not None:
            _flat(grad_square_sum, "grad_square_sum", (torch.float64,), self.device, 1)
            total = grad_square_sum.data_ptr()
        if max_norm is not None and not max_norm > 0:
            raise ValueError("max_norm must be above zero")
        if self._unsaid:
            self._say(betas, 3)
        launch, args = _lib().mscclAmdAdamWStep, (self.handle, lr, at, betas[0], betas[1], eps, grad_scale, total,
                                                  max_norm or 0.0, stream)
        if _elsewhere(self.device):
            with torch.cuda.device(self.device):
                rc = launch(*args)
        else:
            rc = launch(*args)
        if rc:
            raise NcclError(rc, "mscclAmdAdamWStep")
        _changed(self._weights)


def sharded_step(comms: Sequence[Comm], grads: Sequence[torch.Tensor], shards: Sequence[torch.Tensor],
                 params: Sequence[torch.Tensor], plans: Sequence[AdamW], sums: Sequence[SquareSum],
                 lr: Union[float, Sequence[torch.Tensor]], betas=(0.9, 0.999), eps: float = 1e-8,
                 max_norm: Optional[float] = None) -> list:
    """One data-parallel step with the optimizer's state sharded over the ranks, for the ranks of `comms`
    that this process holds (lists: one entry for each).  grads[r]: that rank's whole flat gradient, nranks
    equal blocks; shards[r]: a buffer of one block, which ReduceScatter fills with the sum over ranks and
    plans[r] and sums[r] read; params[r]: the whole flat weights, whose block number `rank` plans[r]
    updates and AllGather sends to every rank.  The gradients are averaged over the ranks.  A gradient
    that is not finite on any rank leaves every rank's weights and state as they were.  Returns the
    square sums of the summed gradient (one float64 of one element for each; its norm is
    sqrt(sum) / nranks)."""
    if not len(comms) == len(grads) == len(shards) == len(params) == len(plans) == len(sums) or not comms:
        raise ValueError("one gradient, shard, weight buffer, plan and square sum for each communicator")
    # all of it before the first collective, for which other ranks would wait: a step that is refused
    # afterwards would leave them waiting, and some plans a step ahead of others
    rates = list(lr) if isinstance(lr, (list, tuple)) else [lr] * len(comms)
    if len(rates) != len(comms):
        raise ValueError("lr: a number, or one for each communicator")
    n = comms[0].nranks
    for p, x in zip(plans, rates):
        p._check_step(x, betas, eps, 1.0 / n, max_norm)
    for r, c in enumerate(comms):
        block = shards[r].numel()
        dev = torch.device("cuda", c.device)
        _flat(shards[r], "shards[%d]" % r, tuple(_TYPES), dev)
        _flat(grads[r], "grads[%d]" % r, (shards[0].dtype,), dev, n * block)
        _flat(params[r], "params[%d]" % r, (params[0].dtype,) if params[0].dtype in _TYPES else tuple(_TYPES), dev, n * block)
        if shards[r].dtype != shards[0].dtype or block != shards[0].numel():
            raise ValueError("the shards must have one size and type")
        if not sums[r].handle:
            raise ValueError("sums[%d] is closed" % r)
        if plans[r].device != dev or sums[r].device != dev:
            raise ValueError("plans[%d] or sums[%d] is on another device than its communicator" % (r, r))
        if plans[r]._grad_type != shards[r].dtype or sums[r].tensors[0].dtype != shards[r].dtype:
            raise TypeError("plans[%d] or sums[%d] reads gradients of another type than shards[%d]'s" % (r, r, r))
        if plans[r].tensors[0][0].dtype != params[r].dtype:
            raise TypeError("plans[%d] writes weights of another type than params[%d]'s" % (r, r))
        size = block * shards[r].element_size()
        if not (_inside(plans[r].grad_span, shards[r].data_ptr(), size) and _inside(sums[r].span, shards[r].data_ptr(), size)):
            raise ValueError("plans[%d] or sums[%d] reads gradients outside shards[%d]" % (r, r, r))
        size = block * params[r].element_size()
        if not _inside(plans[r].param_span, params[r].data_ptr() + c.rank * size, size):
            raise ValueError("plans[%d] writes weights outside its rank's block of params[%d]" % (r, r))
    block, es = shards[0].numel(), params[0].element_size()
    gt, pt = _TYPES[shards[0].dtype], _TYPES[params[0].dtype]
    with group():
        for r, c in enumerate(comms):
            c.reduce_scatter(grads[r].data_ptr(), shards[r].data_ptr(), block, gt, stream=_stream(shards[r].device))
    totals = [s() for s in sums]
    with group():
        for r, c in enumerate(comms):
            c.all_reduce(totals[r].data_ptr(), totals[r].data_ptr(), 1, FLOAT64, stream=_stream(totals[r].device))
    for r, p in enumerate(plans):
        p.step(rates[r], betas, eps, 1.0 / n, totals[r], max_norm)
    with group():
        for r, c in enumerate(comms):
            base = params[r].data_ptr()
            c.all_gather(base + c.rank * block * es, base, block, pt, stream=_stream(params[r].device))
    _changed(list(shards) + list(params))
    return totals


# ---- balance loss of a router's experts ----------------------------------------------------------

class _Stats(torch.autograd.Function):
    """balance_stats of logits that need a gradient: their sums are tied to them, and backward says what is missing."""

    @staticmethod
    def forward(ctx, logits, index, valid, score):
        counts, probs = balance_stats(logits, index, valid, score)
        ctx.mark_non_differentiable(counts)
        return counts, probs

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("the balance loss's gradient is balance_backward's: add that to the logits' gradient, and leave "
                           "the loss out of backward (detach it)")


class _Loss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, counts, probs, top_k, coef):
        return balance_loss(counts, probs, top_k, coef)

    backward = _Stats.backward


def _rows(t: torch.Tensor, what: str, rows: int, cols: int) -> int:
    """The stride from row to row of a matrix whose rows are whole and apart."""
    down, along = t.stride()
    if (cols > 1 and along != 1) or (rows > 1 and down < cols):
        raise ValueError("%s: a row's elements must be neighbours, and rows must not overlap" % what)
    return down if rows > 1 else cols


def _router(logits, index, top_k, valid, score) -> bytes:
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise ValueError("logits must be a tensor on a GPU")
    code = _TYPES.get(logits.dtype)
    if code is None or logits.dim() != 2:
        raise TypeError("logits must be [tokens, experts] of float32, float16 or bfloat16")
    t, e = logits.shape
    if e > 1024:
        raise ValueError("%d experts: at most 1024" % e)
    stride = _rows(logits, "logits", t, e)
    at = itype = istride = ok = 0
    if index is not None:
        if not isinstance(index, torch.Tensor) or index.dtype not in _INDEX or index.dim() != 2 or index.shape[0] != t:
            raise TypeError("index must be [tokens, k] of int32 or int64")
        if index.device != logits.device:
            raise ValueError("index is on %s, not %s" % (index.device, logits.device))
        top_k = index.shape[1]
        at, itype, istride = index.data_ptr(), _INDEX[index.dtype], _rows(index, "index", t, top_k)
    elif not 0 < top_k <= e:
        raise ValueError("top_k %r of %d experts" % (top_k, e))
    if valid is not None:
        _flat(valid, "valid", (torch.bool, torch.uint8), logits.device, t)
        ok = valid.data_ptr()
    if score not in _SCORES:
        raise ValueError("score %r is not one of %s" % (score, ", ".join(_SCORES)))
    return _ROUTER.pack(logits.data_ptr(), code, t, e, stride, at, itype, top_k, istride, ok, _SCORES[score])


def balance_stats(logits: torch.Tensor, index: torch.Tensor, valid: Optional[torch.Tensor] = None,
                  score: str = "softmax"):
    """(counts, probs) of a router's choice: counts int64 [experts + 1], the slots of valid tokens that chose
    each expert and then the number of valid tokens; probs float32 [experts], the sums over valid tokens of
    softmax(logits), or with score="sigmoid" of sigmoid(logits) over its row's sum.  index [tokens, k]: the
    chosen experts (one outside [0, experts) is a dropped slot); valid [tokens]: None, or false for padding.
    The gradient is balance_backward's, not autograd's: backward through probs of logits that need one raises."""
    if index is None:
        raise TypeError("index must be [tokens, k] of int32 or int64")
    if isinstance(logits, torch.Tensor) and logits.requires_grad and torch.is_grad_enabled():
        return _Stats.apply(logits, index, valid, score)
    r = _router(logits, index, 0, valid, score)
    dev = logits.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return balance_stats(logits, index, valid, score)
    t, e = logits.shape
    L = _lib()
    size = L.mscclAmdBalanceWorkspace(t, e)
    scratch = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    counts = torch.empty(e + 1, dtype=torch.int64, device=dev)
    probs = torch.empty(e, dtype=torch.float32, device=dev)
    rc = L.mscclAmdBalanceStats(r, counts.data_ptr(), probs.data_ptr(), scratch.data_ptr() if size else None, size,
                                _stream(dev))
    if rc:
        raise NcclError(rc, "mscclAmdBalanceStats")
    return counts, probs


def balance_all_reduce(comms: Sequence[Comm], counts: Sequence[torch.Tensor], probs: Sequence[torch.Tensor]) -> None:
    """Sums the statistics of balance_stats over all ranks, in place (lists: one entry for each of `comms`,
    the ranks that this process holds): the loss and gradients are then those of the whole batch."""
    if not len(comms) == len(counts) == len(probs) or not comms:
        raise ValueError("one counts and probs for each communicator")
    for r, c in enumerate(comms):
        dev = torch.device("cuda", c.device)
        _flat(probs[r], "probs[%d]" % r, (torch.float32,), dev, probs[0].numel())
        _flat(counts[r], "counts[%d]" % r, (torch.int64,), dev, probs[0].numel() + 1)
    for ts, code in ((counts, INT64), (probs, FLOAT32)):
        with group():
            for r, c in enumerate(comms):
                c.all_reduce(ts[r].data_ptr(), ts[r].data_ptr(), ts[r].numel(), code, stream=_stream(ts[r].device))
        _changed(list(ts))


def balance_loss(counts: torch.Tensor, probs: torch.Tensor, top_k: int, coef: float = 1.0) -> torch.Tensor:
    """coef * experts / (k N^2) * sum of counts[e] * probs[e] (N valid tokens; 0 for none), float32 of one element.
    Its gradient at the logits is balance_backward's, not autograd's (see balance_stats)."""
    _flat(probs, "probs", (torch.float32,))
    if probs.requires_grad and torch.is_grad_enabled():
        return _Loss.apply(counts, probs, top_k, coef)
    dev, e = probs.device, probs.numel()
    _flat(counts, "counts", (torch.int64,), dev, e + 1)
    if not 0 < top_k <= e:
        raise ValueError("top_k %r of %d experts" % (top_k, e))
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return balance_loss(counts, probs, top_k, coef)
    loss = torch.empty(1, dtype=torch.float32, device=dev)
    rc = _lib().mscclAmdBalanceLoss(counts.data_ptr(), probs.data_ptr(), e, top_k, coef, loss.data_ptr(), _stream(dev))
    if rc:
        raise NcclError(rc, "mscclAmdBalanceLoss")
    return loss


def balance_backward(logits: torch.Tensor, counts: torch.Tensor, top_k: int, coef: float = 1.0,
                     grad_output: Optional[torch.Tensor] = None, valid: Optional[torch.Tensor] = None,
                     score: str = "softmax", out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """The gradient of balance_loss at these logits (counts: the loss's own, over all ranks; they carry no
    gradient), in the type of logits; padded rows get zeros.  grad_output: the loss's own gradient, float32
    of one element.  out: where to write it (logits itself, or no element of theirs); accumulate: it is added
    to what `out` holds, which is not logits then."""
    r = _router(logits, None, top_k, valid, score)
    dev = logits.device
    t, e = logits.shape
    _flat(counts, "counts", (torch.int64,), dev, e + 1)
    up, given = None, out is not None
    if grad_output is not None:
        _flat(grad_output, "grad_output", (torch.float32,), dev, 1)
        up = grad_output.data_ptr()
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        out, stride = torch.empty((t, e), dtype=logits.dtype, device=dev), e
    else:
        if out.shape != logits.shape or out.dtype != logits.dtype or out.device != dev:
            raise ValueError("out must have the shape, type and device of logits")
        stride = _rows(out, "out", t, e)
    launch, args = _lib().mscclAmdBalanceBackward, (r, counts.data_ptr(), coef, up, out.data_ptr(), stride,
                                                    int(accumulate), _stream(dev))
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            rc = launch(*args)
    else:
        rc = launch(*args)
    if rc:
        raise NcclError(rc, "mscclAmdBalanceBackward")
    if given:
        _changed((out,))
    return out


__all__ = ["SquareSum", "AdamW", "adamw_state", "dequantize_state", "sharded_step", "balance_stats",
           "balance_all_reduce", "balance_loss", "balance_backward", "STATE_BLOCK"]

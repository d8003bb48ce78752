"""
Operators over a pool of candidates, the step after the acquisition values (gpax/acquisition/acquisition.py:22-35; the
reference chooses by argmax, or by a softmax over the rewards, gpax/hypo.py:115-167, on the host): the softmax policy over
a row of scores, its gradient, the weight that candidates gather over many rows, and the eviction that keeps a pool within
a budget by that weight (include/gpx.h, csrc/choice.hip, csrc/pool.hip).

Arguments are either all NumPy arrays, which are staged through the default engine's GPU and come back as NumPy arrays, or
all torch tensors on one GPU, which are worked on in place on torch's current stream, without a copy and without waiting
(import torch before the library is loaded, so that both use one HIP runtime; the first call on a GPU makes its context and
must not be inside a graph capture).  No autograd graph is recorded: `choice_logprobs_grad` is the backward pass, and a
tensor that requires grad is refused while gradients are enabled, one with a forward-mode tangent always.

Scores are (M,), (rows, M) or (pools, rows, M), of any strides, in float64, float32, bfloat16 or float16.  Sums,
statistics and all real results but gradients are float64 for float64 scores and float32 for the others.  A candidate
exists for a row if it lies below the row's length, its mask is true and its score is not -inf (as penalised acquisition
values are); what is stored in other places is never used.
"""
import functools
import math
import sys
from typing import NamedTuple, Optional, Sequence

import numpy as np

from .. import _lib

MAX_TOP = 64
MAX_PAYLOAD = 16
_MAX_POOL = (1 << 31) - 1 - (1 << 20)
_DTYPES = {"float64": 0, "float32": 1, "bfloat16": 2, "float16": 3}
_INTS = ("int64", "int32")
_MASKS = ("bool", "uint8")
_pack = _lib.POOL_SCORES.pack
_PAYLOAD = ("float64", "float32", "bfloat16", "float16", "float8_e4m3fn", "float8_e5m2", "int64", "int32", "int16", "int8",
            "uint8", "bool", "complex64", "complex128")


class ChoiceLogprobs(NamedTuple):
    """Results of `choice_logprobs`.  The real ones are views of one array, `state`, which also holds what
    `choice_logprobs_grad` reads of the forward pass."""
    logprobs: object
    entropy: object
    logsumexp: object
    top_indices: object
    top_logprobs: object
    state: object


class PoolEviction(NamedTuple):
    """Results of `pool_evict`."""
    indices: object
    lengths: object
    weights: object
    payload: tuple


def _is_torch(a) -> bool:
    if _torch is not None:
        return isinstance(a, _torch.Tensor)
    return type(a).__module__.partition(".")[0] == "torch"


@functools.lru_cache(maxsize=1)
def _one_runtime() -> bool:
    """Device addresses and streams of torch mean something to the library only if both run on one HIP runtime."""
    _lib.load_library()
    try:
        with open("/proc/self/maps") as f:
            found = {line.split(None, 5)[5].strip() for line in f if "libamdhip64.so" in line}
    except OSError:
        return True
    return len(found) <= 1


_torch = None  # torch, its types and the address of a stream, once a tensor has been seen (the package does not import it)
_kind_of: dict = {}
_type_of: dict = {}
_stream_of = None
_forward_ad = None


def _bind_torch() -> None:
    global _torch, _stream_of, _forward_ad
    torch = sys.modules["torch"]
    if not _one_runtime():
        raise _lib.GpxError("libgpx and torch have loaded two HIP runtimes: import torch before gpax_amd's library is loaded "
                            "(before the first engine)")
    for name in (*_DTYPES, *_INTS, *_MASKS, *_PAYLOAD):
        _type_of[name] = getattr(torch, name)
        _kind_of[_type_of[name]] = name
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # current_stream() without making a Stream object of it
    _stream_of = raw or (lambda index: torch.cuda.current_stream(index).cuda_stream)
    _forward_ad = torch.autograd.forward_ad
    _torch = torch


class _Device:
    """Torch tensors on one GPU."""
    host = False

    def __init__(self, ref):
        if not getattr(ref, "is_cuda", False):
            raise ValueError("torch tensors must be on a GPU; pass NumPy arrays for data on the host")
        if _torch is None:
            _bind_torch()
        self.ref, self.index = ref, ref.get_device()
        self.engine = _lib._device_engines.get(self.index)
        if self.engine is None:  # (making one sets the current device)
            with _torch.cuda.device(self.index):
                self.engine = _lib.get_device_engine(self.index)

    def take(self, a, name: str, kinds: Sequence[str], contiguous: bool = False):
        if not isinstance(a, _torch.Tensor) or a.get_device() != self.index:  # -1: on the host
            raise ValueError(f"{name} must be a torch tensor on cuda:{self.index}, as the first argument is")
        if _kind_of.get(a.dtype) not in kinds:
            raise ValueError(f"{name} has dtype {a.dtype}; expected {' or '.join(kinds)}")
        if a.requires_grad and _torch.is_grad_enabled():
            raise ValueError(f"{name} requires grad, and no graph is recorded: detach it and call choice_logprobs_grad")
        if getattr(_forward_ad, "_current_level", 0) >= 0 and _forward_ad.unpack_dual(a).tangent is not None:
            raise ValueError(f"{name} has a tangent, which forward mode would lose here: pass its primal")
        if a.is_neg() or a.is_conj():
            a = a.resolve_conj().resolve_neg()
        return a.contiguous() if contiguous else a

    def kind(self, a) -> str:
        return _kind_of[a.dtype]

    def strides(self, a):
        return a.stride()

    def new(self, shape, kind: str):
        return self.ref.new_empty(shape, dtype=_type_of[kind])

    def view(self, base, shape, offset: int):
        """Contiguous part of a 1-D array: one allocation for several results costs half of one for each."""
        n = len(shape)
        stride = (1,) if n == 1 else (shape[1], 1) if n == 2 else (shape[1] * shape[2], shape[2], 1) if n == 3 else ()
        return base.as_strided(shape, stride, offset)

    def room(self, nbytes: int):
        return self.ref.new_empty(nbytes, dtype=_type_of["uint8"]) if nbytes else None

    def write_to(self, a, *others) -> None:
        """`a` is a result in the caller's memory: nothing else that the call reads may lie there."""
        start, end = _extent(a)
        for o in others:
            if o is not None:
                s, e = _extent(o)
                if s < end and start < e:
                    raise ValueError("out overlaps another argument")
        if not a.is_inference():
            _torch.autograd.graph.increment_version(a)

    def run(self, inputs, outputs, fn, room=None) -> None:
        with self.engine._pool_lock:
            fn(self.engine, _address, _stream_of(self.index))


def _address(a) -> int:
    return 0 if a is None else a.data_ptr()


def _extent(a):
    """Addresses from the first to behind the last element of a tensor."""
    start = a.data_ptr()
    if a.numel() == 0:
        return start, start
    return start, start + (sum((n - 1) * s for n, s in zip(a.shape, a.stride())) + 1) * a.element_size()


class _Room(NamedTuple):
    """Workspace of a host call: space in the scratch, nothing to copy."""
    nbytes: int


class _Host:
    """NumPy arrays, staged through the default engine's scratch."""
    host = True

    def __init__(self, ref):
        self.engine = _lib.get_engine()

    def take(self, a, name: str, kinds: Sequence[str], contiguous: bool = False):
        if _is_torch(a):
            raise ValueError(f"{name} is a torch tensor and the first argument is not")
        a = np.asarray(a)
        if a.dtype.name not in kinds:
            want = kinds[0]
            if want == "bool" or a.dtype.kind not in "iuf" or (want == "int64" and a.dtype.kind == "f"):
                raise ValueError(f"{name} has dtype {a.dtype.name}; expected {' or '.join(kinds)}")
            a = a.astype(want)
        elif not a.dtype.isnative:
            a = a.astype(a.dtype.newbyteorder("="))
        return np.ascontiguousarray(a) if a.ndim else a.copy()

    def kind(self, a) -> str:
        return a.dtype.name

    def strides(self, a):
        return tuple(s // a.itemsize for s in a.strides)

    def new(self, shape, kind: str):
        return np.empty(shape, dtype=kind)

    def view(self, base, shape, offset: int):
        return base[offset:offset + math.prod(shape)].reshape(shape)

    def room(self, nbytes: int):
        return _Room(nbytes) if nbytes else None

    def run(self, inputs, outputs, fn, room=None) -> None:
        place, at = {}, 0
        for a in (*inputs, *outputs, room):
            if a is not None and id(a) not in place:
                place[id(a)] = at
                at += (a.nbytes + 255) // 256 * 256
        with self.engine._pool_lock:
            base = self.engine.scratch(at)
            for a in inputs:
                if a is not None:
                    self.engine.upload(base + place[id(a)], a)
            fn(self.engine, lambda a: 0 if a is None else base + place[id(a)], self.engine.stream())
            for a in outputs:
                if a is not None:
                    self.engine.download(a, base + place[id(a)])


def _space(a):
    return _Device(a) if _is_torch(a) else _Host(a)


def _broadcast_strides(shape, strides, to, name: str):
    """Strides that read an array of `shape` as one of shape `to`."""
    if shape == to:
        return strides
    if len(shape) == 1 and to and shape[0] == to[-1]:
        return (0,) * (len(to) - 1) + strides
    lead = len(to) - len(shape)
    out = [0] * len(to)
    for i, (n, s) in enumerate(zip(shape, strides)):
        if lead + i < 0 or (n != 1 and n != to[lead + i]):
            raise ValueError(f"{name} has shape {tuple(shape)}, which does not broadcast to {tuple(to)}")
        out[lead + i] = 0 if n == 1 else s
    return out


def _pad3(v):
    n = len(v)
    return v if n == 3 else (0, v[0], v[1]) if n == 2 else (0, 0, v[0])


def _pad2(v):
    n = len(v)
    return v if n == 2 else (0, v[0]) if n == 1 else (0, 0)


class _Policy:
    """Checked scores, mask, lengths and temperature of a call."""

    def __init__(self, scores, temperature, mask, lengths):
        self.space = space = _space(scores)
        self.scores = x = space.take(scores, "scores", ("float64", "float32", "float16") if space.host else tuple(_DTYPES))
        if not 1 <= x.ndim <= 3:
            raise ValueError(f"scores have shape {tuple(x.shape)}; expected (M,), (rows, M) or (pools, rows, M)")
        self.kind = kind = space.kind(x)
        self.acc = acc = "float64" if kind == "float64" else "float32"
        self.shape = shape = tuple(x.shape)
        self.lead = lead = shape[:-1]
        self.M = M = shape[-1]
        self.pools, self.rows = p, r = lead if len(lead) == 2 else (1, lead[0]) if lead else (1, 1)
        if p * r > 1 << 25:
            raise ValueError("more than 2^25 rows of scores")
        if M > _MAX_POOL:
            raise ValueError("more than 2^31 - 2^20 candidates")
        self.mask = self.lengths = self.temps = None
        ms, ls, ts = (0, 0, 0), (0, 0), (0, 0)
        n64 = 0
        if mask is not None:
            self.mask = m = space.take(mask, "mask", _MASKS)
            ms = _pad3(_broadcast_strides(tuple(m.shape), space.strides(m), shape, "mask"))
        if lengths is not None:
            self.lengths = n = space.take(lengths, "lengths", _INTS)
            ls = _pad2(_broadcast_strides(tuple(n.shape), space.strides(n), lead, "lengths"))
            n64 = int(space.kind(n) == "int64")
        if isinstance(temperature, (int, float, np.number)):
            T = float(temperature)
            if not (2.3e-308 <= T < math.inf if acc == "float64" else 1.2e-38 <= T <= 3.4e38):
                raise ValueError("the temperature must be positive and finite")
        else:
            T = 1.0
            self.temps = t = space.take(temperature, "temperature", (acc,))
            ts = _pad2(_broadcast_strides(tuple(t.shape), space.strides(t), lead, "temperature"))
            if space.host and not (np.all(t >= np.finfo(acc).tiny) and np.all(np.isfinite(t))):  # 1 / T must be finite too
                raise ValueError("the temperature must be positive and finite")
        self._fields = (p, r, M, *_pad3(space.strides(x))), ms, ls, (*ts, T, _DTYPES[kind], n64)

    def struct(self, ptr) -> bytes:
        a, ms, ls, rest = self._fields
        return _pack(ptr(self.scores), *a, ptr(self.mask) if self.mask is not None else 0, *ms,
                     ptr(self.lengths) if self.lengths is not None else 0, *ls, ptr(self.temps) if self.temps is not None else 0, *rest)

    def inputs(self):
        return self.scores, self.mask, self.lengths, self.temps

    def choices(self, choices):
        """(choices, number per row, shape of the log probabilities)"""
        if choices is None:
            return None, 0, None
        if isinstance(choices, (int, np.integer)) and self.space.host:
            choices = np.int64(choices)
        c = self.space.take(choices, "choices", _INTS, contiguous=True)
        shape = tuple(c.shape)
        if shape != self.lead and (not shape or shape[:-1] != self.lead):
            raise ValueError(f"choices have shape {shape}; expected {self.lead} or {self.lead + ('C',)}")
        if self.space.kind(c) == "int32":
            c = c.astype(np.int64) if self.space.host else c.long()
        if self.space.host and c.size and (c.min() < -1 or c.max() >= self.M):
            raise ValueError(f"choices must lie in 0 .. {self.M - 1}, or be -1")
        n = 1 if len(shape) == len(self.lead) else shape[-1]
        return c, n, shape


@functools.lru_cache(maxsize=4096)
def _choice_workspace(pools, rows, M, dtype, top) -> int:
    return _lib.load_library().gpx_choice_workspace(pools, rows, M, dtype, top)


@functools.lru_cache(maxsize=4096)
def _weights_workspace(pools, rows, M, dtype) -> int:
    return _lib.load_library().gpx_pool_weights_workspace(pools, rows, M, dtype)


@functools.lru_cache(maxsize=4096)
def _evict_workspace(pools, M, dtype) -> int:
    return _lib.load_library().gpx_pool_evict_workspace(pools, M, dtype)


def choice_logprobs(scores, choices=None, *, temperature=1.0, mask=None, lengths=None, top: int = 0) -> ChoiceLogprobs:
    """Softmax policy p_j = exp(x_j / T) / sum_i exp(x_i / T) over every row of scores, in one pass over them.

    Args:
        scores: (M,), (rows, M) or (pools, rows, M)
        choices: the candidates whose log probabilities are wanted, shape scores.shape[:-1] (one a row) or
            scores.shape[:-1] + (C,); -1 is a filler (log probability 0), a candidate that does not exist has -inf
            (a number outside the pool: ValueError for NumPy arrays, NaN for tensors)
        temperature: T, a number or an array broadcast to the rows (of the accumulator's type); positive, finite and not
            subnormal (anything else: ValueError for numbers and NumPy arrays; for tensors a row of NaN where it is not positive
            or log2(e) / T is not finite)
        mask: which candidates may be chosen, bool or uint8, broadcast to the scores
        lengths: how many candidates each row has, int64 or int32, broadcast to the rows (clamped to 0 .. M)
        top: number of best alternatives to return, at most 64

    Returns:
        ChoiceLogprobs: logprobs (as choices; None without them), entropy and logsumexp (one a row), top_indices and
        top_logprobs (rows, top; None for top = 0): score descending, equal scores by index, -1 and -inf where fewer exist;
        a row in which nothing exists has entropy 0 and logsumexp -inf; a row with a NaN or +inf among what exists is NaN
        (NaN scores are never alternatives)
    """
    pol = _Policy(scores, temperature, mask, lengths)
    top = int(top)
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top is {top}; expected 0 .. {MAX_TOP}")
    c, n, lp_shape = pol.choices(choices)
    sp = pol.space
    lead, rows = pol.lead, pol.pools * pol.rows
    e, l, t, p = 2 * rows, 3 * rows, 4 * rows, (4 + top) * rows  # where the parts of `state` start; the statistics first
    state = sp.new((p + n * rows,), pol.acc)
    top_i = sp.new(lead + (top,), "int64") if top else None
    nbytes = _choice_workspace(pol.pools, pol.rows, pol.M, _DTYPES[pol.kind], top)
    ws = sp.room(nbytes)
    size = 8 if pol.acc == "float64" else 4

    def call(engine, ptr, stream):
        base = ptr(state)
        engine.choice_logprobs(pol.struct(ptr), ptr(c), n, top, base + p * size, base + e * size, base + l * size, base,
                               ptr(top_i), base + t * size, ptr(ws), nbytes, stream)

    sp.run((*pol.inputs(), c), (state, top_i), call, ws)
    return ChoiceLogprobs(None if c is None else sp.view(state, lp_shape, p), sp.view(state, lead, e), sp.view(state, lead, l), top_i,
                          sp.view(state, lead + (top,), t) if top else None, state)


def choice_logprobs_grad(scores, forward: ChoiceLogprobs, choices=None, *, grad_logprobs=None, grad_entropy=None,
                         grad_logsumexp=None, grad_top_logprobs=None, temperature=1.0, mask=None, lengths=None):
    """Gradient with respect to the scores of sum(grad_logprobs * logprobs) + sum(grad_entropy * entropy) +
    sum(grad_logsumexp * logsumexp) + sum(grad_top_logprobs * top_logprobs), the selection of alternatives held fixed.

    Args:
        scores, choices, temperature, mask, lengths: as in the forward call
        forward: what the forward call returned
        grad_logprobs, grad_entropy, grad_logsumexp, grad_top_logprobs: gradients of the results, of their shapes and of the
            accumulator's type; None: zero

    Returns:
        the gradient, contiguous, of the scores' shape and type (computed in the accumulator's type, rounded once).  Fillers
        and choices that do not exist have none; a choice named twice counts twice, in the order of the choices.
    """
    pol = _Policy(scores, temperature, mask, lengths)
    sp, acc = pol.space, pol.acc
    c, n, lp_shape = pol.choices(choices)

    def result(a, name, shape, kinds):
        a = sp.take(a, name, kinds, contiguous=True)
        if tuple(a.shape) != tuple(shape):
            raise ValueError(f"{name} has shape {tuple(a.shape)}; expected {tuple(shape)}")
        return a

    if not isinstance(forward, ChoiceLogprobs):
        raise ValueError("forward must be what choice_logprobs returned")
    state = sp.take(forward.state, "forward.state", (acc,), contiguous=True)
    if state.ndim != 1 or state.shape[0] < 4 * pol.pools * pol.rows or tuple(forward.entropy.shape) != pol.lead:
        raise ValueError("forward is not the forward call on these scores")
    logprobs = entropy = top_i = None
    g_lp = g_h = g_lse = g_top = None
    top = 0
    if grad_logprobs is not None:
        if c is None:
            raise ValueError("grad_logprobs needs the choices of the forward call")
        g_lp = result(grad_logprobs, "grad_logprobs", lp_shape, (acc,))
        logprobs = result(forward.logprobs, "forward.logprobs", lp_shape, (acc,))
    if grad_entropy is not None:
        g_h = result(grad_entropy, "grad_entropy", pol.lead, (acc,))
        entropy = result(forward.entropy, "forward.entropy", pol.lead, (acc,))
    if grad_logsumexp is not None:
        g_lse = result(grad_logsumexp, "grad_logsumexp", pol.lead, (acc,))
    if grad_top_logprobs is not None:
        if forward.top_indices is None:
            raise ValueError("grad_top_logprobs needs the alternatives of the forward call")
        top = int(forward.top_indices.shape[-1])
        top_i = result(forward.top_indices, "forward.top_indices", pol.lead + (top,), ("int64",))
        g_top = result(grad_top_logprobs, "grad_top_logprobs", pol.lead + (top,), (acc,))
    grad = sp.new(pol.shape, pol.kind)

    def call(engine, ptr, stream):
        engine.choice_logprobs_grad(pol.struct(ptr), ptr(c), n, ptr(logprobs), ptr(g_lp), top, ptr(top_i), ptr(g_top),
                                    ptr(entropy), ptr(state), ptr(g_h), ptr(g_lse), ptr(grad), stream)

    sp.run((*pol.inputs(), c, logprobs, g_lp, top_i, g_top, entropy, state, g_h, g_lse), (grad,), call)
    return grad


def pool_weights(scores, weights=None, *, decay: float = 1.0, row_weights=None, temperature=1.0, mask=None, lengths=None,
                 out=None):
    """The weight each candidate has gathered: decay * weights + the sum of its probability p over the rows.  Over posterior
    draws, divided by their number, it is the (tempered) probability of being the best candidate.

    Args:
        scores: (M,), (rows, M) or (pools, rows, M)
        weights: weights gathered before, (M,) or (pools, M), of the accumulator's type; None: zeros
        decay: factor on them, finite and not negative; 0 forgets them, whatever they are
        row_weights: factor of each row, of the accumulator's type, shape scores.shape[:-1]; a row of weight 0 is not read
        temperature, mask, lengths: as for choice_logprobs
        out: array for the result; may be `weights`, and may not overlap any other argument

    Returns:
        the new weights, (M,) or (pools, M).  A row in which nothing exists adds nothing; a NaN row makes what exists in it
        NaN.  The sums have a fixed order: the same call gives the same bits.
    """
    pol = _Policy(scores, temperature, mask, lengths)
    sp = pol.space
    decay = float(decay)
    if not 0.0 <= decay < math.inf:
        raise ValueError("the decay must be finite and not negative")
    if pol.pools > 65535:
        raise ValueError("more than 65535 pools")
    shape = (pol.pools, pol.M) if len(pol.shape) == 3 else (pol.M,)
    w = u = None
    if weights is not None and decay != 0.0:
        w = sp.take(weights, "weights", (pol.acc,), contiguous=True)
        if tuple(w.shape) != shape:
            raise ValueError(f"weights have shape {tuple(w.shape)}; expected {shape}")
    if row_weights is not None:
        u = sp.take(row_weights, "row_weights", (pol.acc,), contiguous=True)
        if tuple(u.shape) != pol.lead:
            raise ValueError(f"row_weights have shape {tuple(u.shape)}; expected {pol.lead}")
    if out is None:
        res = sp.new(shape, pol.acc)
    else:
        res = out if sp.host else sp.take(out, "out", (pol.acc,))
        ok = tuple(res.shape) == shape and (res.flags.c_contiguous and res.flags.writeable and res.dtype.name == pol.acc and
                                            res.dtype.isnative if sp.host else res is out and res.is_contiguous())
        if not ok:
            raise ValueError(f"out must be contiguous, of shape {shape} and of type {pol.acc}")
        if not sp.host:
            sp.write_to(res, *pol.inputs(), u, None if w is None or w.data_ptr() == res.data_ptr() else w)
    nbytes = _weights_workspace(pol.pools, pol.rows, pol.M, _DTYPES[pol.kind])
    ws = sp.room(nbytes)

    def call(engine, ptr, stream):
        engine.pool_weights(pol.struct(ptr), ptr(u), ptr(w), decay, ptr(res), ptr(ws), nbytes, stream)

    sp.run((*pol.inputs(), w, u), (res,), call, ws)
    return res


def pool_evict(weights, budget: int, payload: Sequence = (), *, first: int = 0, recent: int = 0,
               lengths: Optional[object] = None) -> PoolEviction:
    """Cut a pool, or every one of several, to at most `budget` candidates: the `first` first and the `recent` last ones
    stay, of the others those of largest weight (equal weights: the lower index; NaN: the smallest).

    Args:
        weights: gathered weights, (M,) or (pools, M), float64 or float32
        budget: how many candidates stay at most, positive
        payload: at most 16 arrays of shape weights.shape + (...) whose rows move along (the points themselves)
        first, recent: how many of the first and of the last stay whatever their weight; together at most the budget
        lengths: how many candidates each pool has, int64 or int32, broadcast to (pools,); clamped to 0 .. M

    Returns:
        PoolEviction: indices (budget, ascending), lengths, weights and payload of what stayed, in the order it had; behind
        the last one index -1 and zeros.  Nothing is changed in place.
    """
    sp = _space(weights)
    w = sp.take(weights, "weights", ("float64", "float32"), contiguous=True)
    if not 1 <= w.ndim <= 2:
        raise ValueError(f"weights have shape {tuple(w.shape)}; expected (M,) or (pools, M)")
    lead, M = tuple(w.shape[:-1]), int(w.shape[-1])
    pools = lead[0] if lead else 1
    budget, first, recent = int(budget), int(first), int(recent)
    if not 1 <= budget <= (1 << 31) - 1:
        raise ValueError(f"the budget is {budget}; expected a positive number")
    if first < 0 or recent < 0 or first + recent > budget:
        raise ValueError(f"first = {first} and recent = {recent} must not be negative, and together at most the budget {budget}")
    if pools > 65535 or M > _MAX_POOL:
        raise ValueError("more than 65535 pools, or 2^31 - 2^20 candidates")
    n, n_stride, n64 = None, 0, False
    if lengths is not None:
        n = sp.take(lengths, "lengths", _INTS)
        stride = _broadcast_strides(tuple(n.shape), sp.strides(n), lead, "lengths")
        n_stride, n64 = (stride[0] if stride else 0), sp.kind(n) == "int64"
    payload = tuple(payload)
    if len(payload) > MAX_PAYLOAD:
        raise ValueError(f"{len(payload)} payload arrays; at most {MAX_PAYLOAD}")
    moved, moved_out, row_bytes = [], [], []
    dims = len(lead) + 1
    for a in payload:
        a = sp.take(a, "payload", _PAYLOAD if not sp.host else (np.asarray(a).dtype.name,), contiguous=True)
        shape = tuple(a.shape)
        if sp.host and a.dtype.kind not in "biufc":
            raise ValueError(f"payload has dtype {a.dtype.name}; expected numbers")
        if shape[:dims] != lead + (M,):
            raise ValueError(f"payload has shape {shape}; expected {lead + (M,)} + (...)")
        row = shape[dims:]
        moved.append(a)
        moved_out.append(sp.new(lead + (budget,) + row, sp.kind(a)))
        row_bytes.append(math.prod(row) * (a.itemsize if sp.host else a.element_size()))
        if row_bytes[-1] > (1 << 31) - 1:
            raise ValueError("payload has rows of 2 GiB or more")
    indices, left, w_out = sp.new(lead + (budget,), "int64"), sp.new(lead, "int64"), sp.new(lead + (budget,), sp.kind(w))

    dtype = _DTYPES[sp.kind(w)]
    nbytes = _evict_workspace(pools, M, dtype)
    ws = sp.room(nbytes)

    def call(engine, ptr, stream):
        engine.pool_evict(dtype, pools, M, ptr(w), ptr(n), n64, n_stride, budget, first, recent, ptr(indices),
                          ptr(left), ptr(w_out), [ptr(a) for a in moved], [ptr(a) for a in moved_out], row_bytes, ptr(ws), nbytes, stream)

    sp.run((w, n, *moved), (indices, left, w_out, *moved_out), call, ws)
    return PoolEviction(indices, left, w_out, tuple(moved_out))


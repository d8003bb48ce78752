"""A stand-in for the engine's pool operators on host memory, for the CPU tests of the argument handling and of the models'
wrappers: addresses are host addresses, results come from tests/pool_oracle.py (test infrastructure)."""
import ctypes as C
import threading

import numpy as np

from gpax_amd import _lib
from tests import pool_oracle as ref
from tests.oracle_engine import OracleEngine

KIND = {0: "float64", 1: "float32", 3: "float16"}


def view(address, dtype, shape, strides=None):
    dtype = np.dtype(dtype)
    if strides is None:
        strides = [int(np.prod(shape[i + 1:])) for i in range(len(shape))]
    if not all(shape):
        return np.empty(shape, dtype)
    n = sum((s - 1) * t for s, t in zip(shape, strides)) + 1
    flat = np.ctypeslib.as_array((C.c_uint8 * (n * dtype.itemsize)).from_address(address)).view(dtype)
    return np.lib.stride_tricks.as_strided(flat, shape, [t * dtype.itemsize for t in strides])


class PoolEngine(OracleEngine):
    def __init__(self):
        super().__init__()
        self._pool_lock = threading.Lock()
        self._room = None

    def scratch(self, nbytes):
        self._room = np.zeros(nbytes + 64, dtype=np.uint8)
        return (self._room.ctypes.data + 63) // 64 * 64

    def upload(self, address, a):
        C.memmove(address, a.ctypes.data, a.nbytes)

    def download(self, a, address):
        C.memmove(a.ctypes.data, address, a.nbytes)

    def stream(self):
        return 0

    def _read(self, s):
        (d_scores, pools, rows, M, x0, x1, x2, d_mask, m0, m1, m2, d_lengths, l0, l1, d_temps, t0, t1, T, dtype,
         n64) = _lib.POOL_SCORES.unpack(s)
        shape, kind = (pools, rows, M), KIND[dtype]
        acc = "float64" if kind == "float64" else "float32"
        x = view(d_scores, kind, shape, [x0, x1, x2])
        mask = view(d_mask, "uint8", shape, [m0, m1, m2]) if d_mask else None
        lengths = view(d_lengths, "int64" if n64 else "int32", shape[:2], [l0, l1]) if d_lengths else None
        T = view(d_temps, acc, shape[:2], [t0, t1]) if d_temps else T
        return x, mask, lengths, T, shape, acc

    def choice_logprobs(self, scores, choices, nchoices, top, logprobs, entropy, logsumexp, stats, top_indices, top_logprobs,
                        workspace, workspace_bytes, stream):
        x, mask, lengths, T, shape, acc = self._read(scores)
        n = shape[0] * shape[1]
        c = view(choices, "int64", (n, nchoices)) if nchoices else None
        f = ref.choice(x, None if c is None else c.reshape(shape[:2] + (nchoices,)), T, mask, lengths, top)
        view(entropy, acc, (n,))[...] = f["entropy"]
        view(logsumexp, acc, (n,))[...] = f["logsumexp"]
        if nchoices:
            view(logprobs, acc, (n, nchoices))[...] = f["logprobs"]
        if top:
            view(top_indices, "int64", (n, top))[...] = f["top_indices"]
            view(top_logprobs, acc, (n, top))[...] = f["top_logprobs"]

    def choice_logprobs_grad(self, scores, choices, nchoices, logprobs, grad_logprobs, top, top_indices, grad_top, entropy, stats,
                             grad_entropy, grad_logsumexp, grad_scores, stream):
        x, mask, lengths, T, shape, acc = self._read(scores)
        n = shape[0] * shape[1]
        get = lambda a, k: view(a, acc, (n, k) if k else (n,)) if a else None
        c = view(choices, "int64", (n, nchoices)).reshape(shape[:2] + (nchoices,)) if nchoices else None
        f = ref.choice(x, c, T, mask, lengths, top)
        g, _ = ref.grad(x, f, c, get(grad_logprobs, nchoices), get(grad_entropy, 0), get(grad_logsumexp, 0), get(grad_top, top), T)
        view(grad_scores, x.dtype, (n, shape[2]))[...] = g

    def pool_weights(self, scores, row_weights, weights, decay, out, workspace, workspace_bytes, stream):
        x, mask, lengths, T, shape, acc = self._read(scores)
        w = view(weights, acc, (shape[0], shape[2])) if weights else None
        u = view(row_weights, acc, shape[:2]) if row_weights else None
        view(out, acc, (shape[0], shape[2]))[...] = ref.weights(x, w, decay, u, T, mask, lengths)

    def pool_evict(self, dtype, pools, candidates, weights, lengths, lengths_64, lengths_stride, budget, first, recent, indices,
                   new_lengths, weights_out, payload, payload_out, row_bytes, workspace, workspace_bytes, stream):
        w = view(weights, KIND[dtype], (pools, candidates))
        n = view(lengths, "int64" if lengths_64 else "int32", (pools,), [lengths_stride]) if lengths else None
        pay = [view(p, "uint8", (pools, candidates, b)) for p, b in zip(payload, row_bytes)]
        i, left, wo, po = ref.evict(w, budget, pay, first, recent, n)
        view(indices, "int64", (pools, budget))[...] = i
        view(new_lengths, "int64", (pools,))[...] = left
        view(weights_out, KIND[dtype], (pools, budget))[...] = wo
        for a, v, b in zip(payload_out, po, row_bytes):
            view(a, "uint8", (pools, budget, b))[...] = v

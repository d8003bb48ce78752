"""Plain NumPy implementations in 64 bits of the operators over a pool of candidates, row by row from the definitions, and
the tolerances their tests use (test infrastructure)."""
import numpy as np

U = {"float64": 2.0 ** -53, "float32": 2.0 ** -24, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -24}  # of the accumulator
# largest relative error of one rounding to the storage type, and the spacing of its subnormals
HALF = {"float64": 2.0 ** -53, "float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float64": 0.0, "float32": 2.0 ** -126, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -126}


def allowed(x, mask=None, lengths=None):
    ok = np.ones(x.shape, dtype=bool)
    if mask is not None:
        ok &= np.broadcast_to(np.asarray(mask) != 0, x.shape)
    if lengths is not None:
        ok &= np.arange(x.shape[-1]) < np.clip(np.broadcast_to(lengths, x.shape[:-1]), 0, x.shape[-1])[..., None]
    return ok & ~np.isneginf(np.where(ok, x, 0.0))


def policy(x, T=1.0, mask=None, lengths=None):
    """z (-inf where nothing exists), log p, p, log-sum-exp and entropy, rows flattened"""
    x = np.asarray(x, dtype=np.float64)
    ok = allowed(x, mask, lengths)
    T = np.broadcast_to(np.asarray(T, dtype=np.float64), x.shape[:-1])
    z = np.where(ok, np.where(ok, x, 0.0) / T[..., None], -np.inf).reshape(int(np.prod(x.shape[:-1])), x.shape[-1])
    logp, p = np.full(z.shape, -np.inf), np.zeros(z.shape)
    lse, H = np.full(len(z), -np.inf), np.zeros(len(z))
    for i, row in enumerate(z):
        at = np.flatnonzero(~np.isneginf(row))
        if not at.size:
            continue
        v = row[at]
        if np.any(np.isnan(v)) or np.any(np.isposinf(v)):
            logp[i, at] = p[i, at] = lse[i] = H[i] = np.nan
            continue
        lse[i] = v.max() + np.log(np.sum(np.exp(v - v.max())))
        logp[i, at] = (v - v.max()) - np.log(np.sum(np.exp(v - v.max())))
        p[i, at] = np.exp(logp[i, at])
        H[i] = -np.sum(p[i, at] * logp[i, at])
    return z, logp, p, lse, H


def choice(x, choices=None, T=1.0, mask=None, lengths=None, top=0):
    z, logp, p, lse, H = policy(x, T, mask, lengths)
    n = len(z)
    out = {"entropy": H, "logsumexp": lse, "z": z, "logp": logp, "p": p}
    if choices is not None:
        c = np.asarray(choices).reshape(n, -1) if n else np.zeros((0, np.shape(choices)[-1]), dtype=np.int64)
        lp = np.zeros(c.shape)
        for i in range(n):
            for q, j in enumerate(c[i]):
                lp[i, q] = 0.0 if j == -1 else (logp[i, j] if 0 <= j < z.shape[1] else np.nan)
        out["logprobs"] = lp
    ti, tl = np.full((n, top), -1, dtype=np.int64), np.full((n, top), -np.inf)
    for i in range(n):
        at = [j for j in np.argsort(-z[i], kind="stable") if not np.isneginf(z[i, j]) and not np.isnan(z[i, j])][:top]
        ti[i, :len(at)] = at
        tl[i, :len(at)] = logp[i, at]
    out["top_indices"], out["top_logprobs"] = ti, tl
    return out


def grad(x, fwd, choices=None, g_lp=None, g_h=None, g_lse=None, g_top=None, T=1.0):
    """from choice()'s results"""
    z, logp, p = fwd["z"], fwd["logp"], fwd["p"]
    n, M = z.shape
    T = np.broadcast_to(np.asarray(T, dtype=np.float64), np.shape(x)[:-1]).reshape(-1)
    out, size = np.zeros((n, M)), np.zeros((n, M))
    for i in range(n):
        pairs = []
        if g_lp is not None:
            c, g = np.asarray(choices).reshape(n, -1)[i], np.asarray(g_lp).reshape(n, -1)[i]
            pairs += [(j, v) for j, v in zip(c, g) if 0 <= j < M and not np.isneginf(logp[i, j])]
        if g_top is not None:
            pairs += [(j, v) for j, v in zip(fwd["top_indices"][i], np.asarray(g_top).reshape(n, -1)[i]) if j >= 0]
        G = sum(v for _, v in pairs)
        gh = 0.0 if g_h is None else np.asarray(g_h).reshape(-1)[i]
        gl = 0.0 if g_lse is None else np.asarray(g_lse).reshape(-1)[i]
        at = ~np.isneginf(z[i])
        inner = logp[i, at] + fwd["entropy"][i]
        out[i, at] = p[i, at] * (gl - G - gh * inner)
        size[i, at] = p[i, at] * (abs(gl) + sum(abs(v) for _, v in pairs) + abs(gh) * (np.abs(logp[i, at]) + fwd["entropy"][i]))
        for j, v in pairs:
            out[i, j] += v
            size[i, j] += abs(v)
        out[i] /= T[i]
        size[i] /= T[i]
    return out, size


def weights(x, w=None, decay=1.0, u=None, T=1.0, mask=None, lengths=None):
    x = np.asarray(x, dtype=np.float64)
    shape = x.shape if x.ndim == 3 else (1,) + ((1,) if x.ndim == 1 else ()) + x.shape
    p = policy(x, T, mask, lengths)[2].reshape(shape)
    u = np.ones(shape[:2]) if u is None else np.asarray(u, dtype=np.float64).reshape(shape[:2])
    s = np.zeros((shape[0], shape[2])) if w is None else decay * np.asarray(w, dtype=np.float64).reshape(shape[0], shape[2])
    for b in range(shape[0]):
        for r in range(shape[1]):
            if u[b, r] != 0:
                s[b] += u[b, r] * p[b, r]
    return s if x.ndim == 3 else s[0]


def evict(w, budget, payload=(), first=0, recent=0, lengths=None):
    w = np.asarray(w)
    B, M = int(np.prod(w.shape[:-1])), w.shape[-1]
    flat = w.reshape(B, M)
    L = np.full(B, M) if lengths is None else np.clip(np.broadcast_to(lengths, (B,)), 0, M)
    idx, wout = np.full((B, budget), -1, dtype=np.int64), np.zeros((B, budget), dtype=w.dtype)
    pay = [np.asarray(a).reshape((B, M) + np.asarray(a).shape[w.ndim:]) for a in payload]
    out = [np.zeros((B, budget) + a.shape[2:], dtype=a.dtype) for a in pay]
    for b in range(B):
        n = int(L[b])
        at = np.arange(n)
        if n > budget:
            held = (at < first) | (at >= n - recent)
            free = at[~held]
            v = flat[b, free].astype(np.float64)
            order = sorted(range(len(free)), key=lambda q: (np.isnan(v[q]), -v[q] if not np.isnan(v[q]) else 0.0, free[q]))
            at = np.sort(np.concatenate([at[held], free[order[:budget - first - recent]]]))
        idx[b, :len(at)], wout[b, :len(at)] = at, flat[b, at]
        for o, a in zip(out, pay):
            o[b, :len(at)] = a[b, at]
    lead = w.shape[:-1]
    return (idx.reshape(lead + (budget,)), np.minimum(L, budget).reshape(lead), wout.reshape(lead + (budget,)),
            [o.reshape(lead + o.shape[1:]) for o in out])


# ---- tolerances: u = half a unit in the last place of the accumulator ---------------------------------------------------
# w = (x - m) c with c = log2(e) / T carries the roundings of T, c, x - m and the product: 4 u |w|, and the definition's own
# z = x / T one of u |z| in 64 bits (negligible for the others): |w| <= 2 (|z| + |z_max|), so 8 u (|z| + |z_max|) is enough
# for (x - m) / T.  An exponential adds 2 u and what its argument carries; arguments that matter for the sum are below 40
# in size, so a term of the sum is off by at most 4 u 40 + 2 u relatively, a lane adds M / 64 terms and a tree 16 more: s is
# off by (M / 64 + 180) u.  The logarithm adds 2 u of its value.
def tol_logp(kind, z, zmax, M):
    return U[kind] * (200.0 + M / 64 + 8 * (np.abs(z) + np.abs(zmax)))


# H = ln 2 (log2 s - t / s): t's terms carry the same errors as s's relative to their size, and sum |p w| <= H + log s
def tol_entropy(kind, H, lse_rel, zmax, M):
    return U[kind] * ((200.0 + M / 32) * (1.0 + H + 2 * lse_rel) + 8 * np.abs(zmax))


# p = exp(log p): the error of its exponent, plus 2 u; the bracket of the gradient is off by that of log p and H
def tol_grad(kind, g, size, z, zmax, M, C):
    rel = tol_logp(kind, z, zmax, M) * 3 + U[kind] * (C + 16)
    return size * rel + np.abs(g) * HALF[kind] * 1.01 + TINY[kind]

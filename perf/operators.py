"""Cases of the operators over a pool of candidates: the softmax policy over acquisition values or posterior draws (log
probabilities of given choices, entropy, best alternatives), a training step of it (forward and gradient), the weight each
candidate gathers over many draws, and the eviction that keeps a pool within its budget by that weight.

`run` computes them in elementary torch operations, or, where `own` is true, through gpax_amd.acquisition.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2}


def _acc(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def listed():
    return [
        # one vector of acquisition values over the 201-point grid of the Bayesian-optimisation loop: nothing but latency
        dict(name="choice_grid", op="choice", rows=1, pool=201, dtype="f64", choices=1, top=1, mask="none", ragged=False, temperature=0.5),
        # the predictive draws of 1000 posterior samples over the 1024 test points of the headline benchmark, measured points excluded
        dict(name="choice_draws", op="choice", rows=1000, pool=1024, dtype="f64", choices=4, top=8, mask="shared", ragged=False, temperature=0.7),
        # a batch of suggestions over every pixel of the 512 x 512 image: few rows, a long axis, a long list of alternatives
        dict(name="choice_image", op="choice", rows=8, pool=262144, dtype="f64", choices=16, top=64, mask="full", ragged=False, temperature=1.0),
        # many rows over large pools of unequal length kept in 16 bits: bound by memory
        dict(name="choice_wide", op="choice", rows=2048, pool=65536, dtype="bf16", choices=1, top=20, mask="none", ragged=True, temperature=1.3),
        # a policy-gradient step (log probabilities of the taken choices, an entropy bonus) on the draws above
        dict(name="step_draws", op="step", rows=1000, pool=1024, dtype="f64", choices=4, top=8, mask="shared", ragged=False, temperature=0.7),
        # the same on a pool of odd size in 32 bits with a mask of its own for each row
        dict(name="step_odd", op="step", rows=512, pool=32749, dtype="f32", choices=8, top=0, mask="full", ragged=False, temperature=1.0),
        # weights of the 1024 candidates over 1000 draws
        dict(name="weights_draws", op="weights", pools=1, rows=1000, pool=1024, dtype="f64", mask="shared", ragged=False, temperature=0.3),
        # sixteen tasks with pools of their own, of unequal length
        dict(name="weights_tasks", op="weights", pools=16, rows=128, pool=16381, dtype="f32", mask="none", ragged=True, temperature=0.5),
        # the pixels of an image over 64 draws
        dict(name="weights_image", op="weights", pools=1, rows=64, pool=262144, dtype="f64", mask="shared", ragged=False, temperature=0.5),
        # the grid of the loop cut to a quarter: nothing but latency
        dict(name="evict_grid", op="evict", pools=1, pool=201, budget=50, dims=1, first=4, recent=4, dtype="f64", ragged=False),
        # many pools at once, of unequal length
        dict(name="evict_tasks", op="evict", pools=64, pool=16384, budget=4096, dims=3, first=4, recent=64, dtype="f32", ragged=True),
        # the pixels of an image cut to an eighth
        dict(name="evict_image", op="evict", pools=1, pool=262144, budget=32768, dims=2, first=0, recent=128, dtype="f64", ragged=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))) - 0.5))))


def draw(rng):
    op = rng.choice(["choice", "step", "weights", "evict"])
    pool = _log_int(rng, 1, 262144)
    dtype = rng.choice(["f64", "f64", "f32", "bf16", "f16"])
    ragged = rng.random() < 0.4
    if op == "evict":
        pools = _log_int(rng, 1, max(1, min(64, (1 << 20) // pool)))
        budget = rng.randint(1, pool)
        first = rng.randint(0, min(8, budget))
        return dict(op=op, pools=pools, pool=pool, budget=budget, dims=rng.randint(1, 8), first=first,
                    recent=rng.randint(0, min(64, budget - first)), dtype=rng.choice(["f64", "f32"]), ragged=ragged)
    case = dict(op=op, pool=pool, dtype=dtype, mask=rng.choice(["none", "shared", "full"]), ragged=ragged,
                temperature=round(rng.uniform(0.2, 3.0), 3))
    if op == "weights":
        pools = _log_int(rng, 1, 16)
        return dict(case, pools=pools, rows=_log_int(rng, 1, max(1, min(4096, (1 << 24) // (pool * pools)))))
    rows = _log_int(rng, 1, max(1, min(4096, (1 << 24) // pool)))
    return dict(case, rows=rows, choices=_log_int(rng, 1, 64), top=rng.choice([0, 1, 5, 20, 64]))


def _work_rows(case):
    return case.get("pools", 1) * case["rows"]


def work(case):
    if case["op"] == "evict":
        size, n, k = _SIZE[case["dtype"]], case["pools"] * case["pool"], case["pools"] * case["budget"]
        return {"bytes": n * size + k * (2 * case["dims"] * size + size + 8), "flops": n}
    rows, pool = _work_rows(case), case["pool"]
    size, acc = _SIZE[case["dtype"]], 8 if case["dtype"] == "f64" else 4
    moved = rows * pool * (size + (1 if case["mask"] == "full" else 0)) + (pool if case["mask"] == "shared" else 0)
    if case["op"] == "weights":
        return {"bytes": moved + 2 * case["pools"] * pool * acc, "flops": 6 * rows * pool}
    moved += rows * (case["choices"] * (8 + acc) + 2 * acc + case["top"] * (8 + acc))
    if case["op"] == "step":
        return {"bytes": moved + rows * pool * size + rows * (case["choices"] + 1) * acc, "flops": 14 * rows * pool}
    return {"bytes": moved, "flops": 6 * rows * pool}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)
    dev = torch.device("cuda")
    dtype = _TYPES[case["dtype"]]
    pool = case["pool"]
    if case["op"] == "evict":
        pools = case["pools"]
        # gathered weights span many orders of magnitude; a few candidates never got any
        w = torch.exp(3.0 * torch.randn(pools, pool, generator=g, device=dev, dtype=torch.float64))
        w = torch.where(torch.rand(pools, pool, generator=g, device=dev) < 0.05, torch.zeros_like(w), w).to(dtype)
        points = torch.rand(pools, pool, case["dims"], generator=g, device=dev, dtype=dtype)
        lengths = torch.randint(0, pool + 1, (pools,), generator=g, device=dev) if case["ragged"] else None
        return dict(case, weights=w, points=points, lengths=lengths)
    lead = (case["pools"], case["rows"]) if case["op"] == "weights" else (case["rows"],)
    # posterior draws: a mean over the pool that all rows share, and each row's own deviation from it
    scores = torch.randn(pool, generator=g, device=dev) + 0.5 * torch.randn(*lead, pool, generator=g, device=dev, dtype=_acc(dtype))
    mask = None
    if case["mask"] != "none":
        mask = torch.rand(*((pool,) if case["mask"] == "shared" else (*lead, pool)), generator=g, device=dev) > 0.1
    lengths = torch.randint(0, pool + 1, lead, generator=g, device=dev) if case["ragged"] else None
    state = dict(case, scores=scores.to(dtype), mask=mask, lengths=lengths)
    if case["op"] == "weights":
        state["weights"] = torch.rand(case["pools"], pool, generator=g, device=dev, dtype=_acc(dtype))
        return state
    chosen = torch.rand(case["rows"], case["choices"], generator=g, device=dev, dtype=torch.float64)
    limit = (lengths if lengths is not None else torch.full(lead, pool, device=dev)).clamp(min=1)[:, None]
    chosen = (chosen * limit).long().clamp(max=pool - 1)
    # some rows chose fewer than the others: -1 fills them up
    chosen[:, 1:] = torch.where(torch.rand(case["rows"], case["choices"] - 1, generator=g, device=dev) < 0.1, -1, chosen[:, 1:])
    state["chosen"] = chosen
    if case["op"] == "step":  # advantages of the taken choices, and the weight of the entropy
        state["g_logprobs"] = torch.randn(case["rows"], case["choices"], generator=g, device=dev, dtype=_acc(dtype))
        state["g_entropy"] = 0.1 * torch.rand(case["rows"], generator=g, device=dev, dtype=_acc(dtype))
    return state


def _allowed(s):
    x = s["scores"]
    ok = torch.ones_like(x, dtype=torch.bool) if s["mask"] is None else s["mask"].expand(x.shape)
    if s["lengths"] is not None:
        ok = ok & (torch.arange(x.shape[-1], device=x.device) < s["lengths"][..., None])
    return ok


def _policy(s):
    """z with -inf where nothing may be chosen, its log of the sum of exponentials, the probabilities."""
    x = s["scores"].to(_acc(s["scores"].dtype))
    z = torch.where(_allowed(s), x / s["temperature"], -math.inf)
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    p = torch.where(total > 0, e / total, torch.zeros_like(e))
    return z, top, torch.log(total), p


def _choice(s):
    z, top, log_total, p = _policy(s)
    logp = torch.where(z == -math.inf, -math.inf, (z - top) - log_total)
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    chosen = s["chosen"]
    at = torch.where(chosen < 0, torch.zeros_like(logp[:, :1]), torch.gather(logp, 1, chosen.clamp(min=0)))
    out = [at, entropy, (top + log_total)[..., 0]]
    k = s["top"]
    if k:
        n = min(k, z.shape[-1])
        value, index = torch.sort(z, dim=-1, descending=True, stable=True)
        index = torch.where(value[:, :n] == -math.inf, -1, index[:, :n])
        best = torch.gather(logp, 1, index.clamp(min=0))
        best = torch.where(index < 0, -math.inf, best)
        pad = k - n
        out += [torch.nn.functional.pad(index, (0, pad), value=-1), torch.nn.functional.pad(best, (0, pad), value=-math.inf)]
    return out, logp, p, entropy


def _step(s):
    out, logp, p, entropy = _choice(s)
    g, gh, chosen = s["g_logprobs"], s["g_entropy"], s["chosen"]
    # a choice that is a filler, or that may not be made, has no gradient
    ok = (chosen >= 0) & torch.gather(logp > -math.inf, 1, chosen.clamp(min=0))
    g = torch.where(ok, g, torch.zeros_like(g))
    inner = torch.where(p > 0, logp + entropy[:, None], torch.zeros_like(p))
    grad = -p * (g.sum(-1, keepdim=True) + gh[:, None] * inner)
    grad = grad.scatter_add(1, chosen.clamp(min=0), g) / s["temperature"]
    return out + [grad.to(s["scores"].dtype)]


def _weights(s):
    return s["weights"] * 0.9 + _policy(s)[3].sum(-2)


def _evict(s):
    w, points, budget = s["weights"], s["points"], s["budget"]
    pools, pool = w.shape
    at = torch.arange(pool, device=w.device).expand(pools, pool)
    length = torch.full((pools, 1), pool, device=w.device) if s["lengths"] is None else s["lengths"][:, None]
    rank = torch.where((at < s["first"]) | (at >= length - s["recent"]), math.inf, w)
    rank = torch.where(at < length, rank, -math.inf)
    order = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :budget]
    kept = torch.where(torch.arange(budget, device=w.device) < length, order, pool)  # what does not exist sorts behind
    kept = torch.sort(kept, dim=1).values
    there = kept < pool
    safe = kept.clamp(max=pool - 1)
    out_w = torch.where(there, torch.gather(w, 1, safe), torch.zeros_like(w[:, :1]))
    out_p = torch.gather(points, 1, safe[..., None].expand(pools, budget, points.shape[-1]))
    out_p = torch.where(there[..., None], out_p, torch.zeros_like(out_p))
    return [torch.where(there, kept, -1), there.sum(1), out_w, out_p]


def run(state):
    s = state
    if own:
        from gpax_amd import acquisition as acq

        if s["op"] == "evict":
            r = acq.pool_evict(s["weights"], s["budget"], (s["points"],), first=s["first"], recent=s["recent"], lengths=s["lengths"])
            return [r.indices, r.lengths, r.weights, r.payload[0]]
        policy = dict(temperature=s["temperature"], mask=s["mask"], lengths=s["lengths"])
        if s["op"] == "weights":
            return acq.pool_weights(s["scores"], s["weights"], decay=0.9, **policy)
        r = acq.choice_logprobs(s["scores"], s["chosen"], top=s["top"], **policy)
        out = [r.logprobs, r.entropy, r.logsumexp] + ([r.top_indices, r.top_logprobs] if s["top"] else [])
        if s["op"] == "step":
            out.append(acq.choice_logprobs_grad(s["scores"], r, s["chosen"], grad_logprobs=s["g_logprobs"], grad_entropy=s["g_entropy"], **policy))
        return out
    if s["op"] == "evict":
        return _evict(s)
    if s["op"] == "weights":
        return _weights(s)
    return _step(s) if s["op"] == "step" else _choice(s)[0]


def exact(case, seed):
    """Row by row on the host in 64 bits, from the definitions: p_j = exp(x_j / T) / sum, H = log sum - sum p z."""
    if case["op"] == "evict":  # nothing is computed: what is kept is moved
        return None
    s = prepare(case, seed)
    x = s["scores"].double().cpu().numpy()
    rows = x.reshape(-1, x.shape[-1])
    if rows.size > 1 << 27:
        return None
    mask = None if s["mask"] is None else s["mask"].cpu().numpy()
    lengths = None if s["lengths"] is None else s["lengths"].cpu().numpy().reshape(-1)
    T = case["temperature"]

    def row(i):
        """Places that may be chosen in row i, their z, the log of the sum."""
        ok = np.arange(rows.shape[1]) if mask is None else np.flatnonzero(mask if mask.ndim == 1 else mask.reshape(rows.shape)[i])
        if lengths is not None:
            ok = ok[ok < lengths[i]]
        z = rows[i, ok] / T
        if not ok.size:
            return ok, z, -np.inf
        shift = float(z.max())
        return ok, z, shift + math.log(float(np.sum(np.exp(z - shift))))

    if case["op"] == "weights":
        out = 0.9 * s["weights"].double().cpu().numpy()
        for i in range(len(rows)):
            ok, z, lse = row(i)
            out[i // case["rows"], ok] += np.exp(z - lse) if ok.size else 0.0
        return out
    chosen = s["chosen"].cpu().numpy()
    k, n = case["top"], len(rows)
    logprobs, entropy, lses = np.zeros(chosen.shape), np.zeros(n), np.zeros(n)
    best = np.full((n, k), -np.inf)
    grad = np.zeros_like(rows) if case["op"] == "step" else None
    if grad is not None:
        g_lp, g_h = s["g_logprobs"].double().cpu().numpy(), s["g_entropy"].double().cpu().numpy()
    for i in range(n):
        ok, z, lse = row(i)
        lses[i] = lse
        full = {}
        if ok.size:
            d = z - lse
            p = np.exp(d)
            entropy[i] = -float(np.sum(p * d))
            m = min(k, ok.size)
            if m:
                best[i, :m] = np.sort(np.partition(d, ok.size - m)[ok.size - m:])[::-1]
            where = np.searchsorted(ok, chosen[i])
            full = {c: d[w] for c, w in zip(chosen[i], where) if c >= 0 and w < ok.size and ok[w] == c}
        logprobs[i] = [0.0 if c < 0 else full.get(c, -np.inf) for c in chosen[i]]
        if grad is not None and ok.size:
            live = [(int(c), v) for c, v in zip(chosen[i], g_lp[i]) if int(c) in full]
            grad[i, ok] = -p * (math.fsum(v for _, v in live) + g_h[i] * (d + entropy[i]))
            for c, v in live:
                grad[i, c] += v
    out = [logprobs, entropy, lses] + ([None, best] if k else [])
    return out + ([grad / T] if grad is not None else [])

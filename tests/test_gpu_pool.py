"""GPU: the operators over a pool of candidates (gpax_amd/acquisition/pool.py; csrc/choice.hip, csrc/pool.hip) against the
plain implementations in 64 bits of tests/pool_oracle.py, on torch tensors and on NumPy arrays."""
import math
import threading
import zlib

import numpy as np
import pytest
import torch  # before libgpx is loaded: one HIP runtime for both

from gpax_amd import _lib
from gpax_amd import acquisition as acq
from tests import pool_oracle as ref

pytestmark = pytest.mark.gpu

KINDS = ["float64", "float32", "bfloat16", "float16"]
ACC = {"float64": torch.float64, "float32": torch.float32, "bfloat16": torch.float32, "float16": torch.float32}


def scores_of(rng, kind, shape, spread=2.0):
    return torch.as_tensor(spread * rng.standard_normal(shape), device="cuda").to(getattr(torch, kind))


def host(t):
    return None if t is None else t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def close(got, want, tol, what=""):
    got, want, tol = np.asarray(got, dtype=np.float64), np.asarray(want, dtype=np.float64), np.asarray(tol, dtype=np.float64)
    got = got.reshape(want.shape)
    special = ~np.isfinite(want)
    np.testing.assert_array_equal(got[special], want[special], err_msg=what)
    err = np.abs(got[~special] - want[~special])
    lim = np.broadcast_to(tol, want.shape)[~special]
    assert np.all(np.isfinite(got[~special])), what
    bad = err > lim
    assert not bad.any(), (what, float(err[bad].max()), float(lim[bad].min()), int(bad.sum()))


def check_choice(r, x, kind, choices=None, T=1.0, mask=None, lengths=None, top=0):
    f = ref.choice(host(x), host(choices), T, host(mask), host(lengths), top)
    z, M = f["z"], f["z"].shape[1]
    zmax = np.max(np.where(np.isfinite(z), z, -np.inf), axis=1, initial=-np.inf)
    zmax = np.where(np.isfinite(zmax), zmax, 0.0)
    zmax = np.maximum(np.abs(zmax), np.abs(np.where(np.isfinite(f["logsumexp"]), f["logsumexp"], 0)))
    span = np.abs(np.where(np.isfinite(f["logsumexp"]), f["logsumexp"] - zmax, 0))
    close(host(r.entropy), f["entropy"], ref.tol_entropy(kind, f["entropy"], span, zmax, M), "entropy")
    close(host(r.logsumexp), f["logsumexp"], ref.tol_logp(kind, 0 * zmax, zmax, M), "logsumexp")
    if choices is not None:
        c = host(choices).reshape(f["logprobs"].shape)
        zc = np.array([[z[i, j] if 0 <= j < M and np.isfinite(z[i, j]) else 0.0 for j in row] for i, row in enumerate(c)]).reshape(c.shape)
        close(host(r.logprobs), f["logprobs"], ref.tol_logp(kind, zc, zmax[:, None], M), "logprobs")
    if top:
        got = host(r.top_indices).reshape(len(z), top)
        np.testing.assert_array_equal(got, f["top_indices"])
        zt = np.array([[z[i, j] if j >= 0 and np.isfinite(z[i, j]) else 0.0 for j in row] for i, row in enumerate(got)]).reshape(got.shape)
        close(host(r.top_logprobs), f["top_logprobs"], ref.tol_logp(kind, zt, zmax[:, None], M), "top_logprobs")
    return f, zmax


def case_inputs(rng, kind, shape, mask_kind, ragged, C, T_rows=False):
    x = scores_of(rng, kind, shape)
    lead, M = shape[:-1], shape[-1]
    mask = None
    if mask_kind == "shared":
        mask = torch.as_tensor(rng.random(M) > 0.3, device="cuda")
    elif mask_kind == "full":
        mask = torch.as_tensor(rng.random(shape) > 0.3, device="cuda")
    lengths = torch.as_tensor(rng.integers(0, M + 1, lead), device="cuda") if ragged else None
    choices = torch.as_tensor(rng.integers(-1, M, lead + (C,)), device="cuda") if C else None
    T = 0.7
    if T_rows:
        T = torch.as_tensor(rng.uniform(0.3, 3.0, lead), device="cuda").to(ACC[kind])
    return x, mask, lengths, choices, T


# every plan of the launch: one wave a row, 4 and 16 waves, several workgroups a row; ends inside a vector, a step, a split
SHAPES = [(1, 1), (4, 0), (0, 7), (1, 201), (5, 7), (3, 64), (3, 1023), (2, 1024), (2, 1025), (130, 1001), (4099, 33),
          (300, 4099), (40, 16387), (2, 70001), (1, 262144), (2, 3, 515), (7,)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_choice_logprobs_and_gradient(kind, shape):
    rng = np.random.default_rng(zlib.crc32(repr((kind, shape)).encode()))
    for mask_kind, ragged, C, top, T_rows in [("none", False, 1, 1, False), ("shared", True, 5, 20, True), ("full", False, 70, 64, False),
                                              ("full", True, 0, 0, True), ("none", True, 3, 7, False)]:
        if shape[-1] == 0 and C:
            C = 0
        x, mask, lengths, choices, T = case_inputs(rng, kind, shape, mask_kind, ragged, C, T_rows)
        T_host = host(T) if T_rows else T
        r = acq.choice_logprobs(x, choices, temperature=T, mask=mask, lengths=lengths, top=top)
        f, zmax = check_choice(r, x, kind, choices, T_host, mask, lengths, top)
        lead = shape[:-1]
        mk = lambda s: torch.as_tensor(rng.standard_normal(s), device="cuda").to(ACC[kind])
        g_lp, g_h, g_lse, g_top = mk(lead + (C,)) if C else None, mk(lead), mk(lead), mk(lead + (top,)) if top else None
        g = acq.choice_logprobs_grad(x, r, choices, grad_logprobs=g_lp, grad_entropy=g_h, grad_logsumexp=g_lse,
                                     grad_top_logprobs=g_top, temperature=T, mask=mask, lengths=lengths)
        assert g.shape == x.shape and g.dtype == x.dtype
        want, size = ref.grad(host(x), f, host(choices), host(g_lp), host(g_h), host(g_lse), host(g_top), T_host)
        if want.size:
            zf = np.where(np.isfinite(f["z"]), f["z"], 0)
            close(host(g).reshape(want.shape), want, ref.tol_grad(kind, want, size, zf, zmax[:, None], shape[-1], C + top), "gradient")


@pytest.mark.parametrize("kind", ["float64", "float32", "bfloat16"])
def test_strides_views_and_broadcasts(kind):
    rng = np.random.default_rng(3)
    big = scores_of(rng, kind, (6, 9, 2050))
    mask_big = torch.as_tensor(rng.random((9, 4100)) > 0.2, device="cuda")
    views = [big[2, :, 1:2000], big[:, 3, 5:], big[1, ::2, ::2], big[0, 1:, 3::7], big[0].t()[:9, :7], big[:2, :, 1:1030],
             big[0, 4].expand(5, 2050), big[0, :1, 1:4], big[:, :, 77].contiguous()[:, None, :].expand(6, 3, 9)]
    for x in views:
        for mask in [None, mask_big[0, 1:x.shape[-1] + 1], mask_big[3, : 2 * x.shape[-1]: 2]]:
            lead = tuple(x.shape[:-1])
            choices = torch.as_tensor(rng.integers(0, x.shape[-1], lead + (3,)), device="cuda").to(torch.int32)
            lengths = torch.full((1,), x.shape[-1] - 2, device="cuda", dtype=torch.int32)
            r = acq.choice_logprobs(x, choices, mask=mask, lengths=lengths, top=4)
            check_choice(r, x, kind, choices, 1.0, mask, lengths, 4)
            w = acq.pool_weights(x, mask=mask, lengths=lengths)
            c = acq.pool_weights(x.contiguous(), mask=mask, lengths=lengths)
            assert torch.equal(w, c)  # the order of the sums does not depend on how the scores lie
            g = acq.choice_logprobs_grad(x, r, choices, grad_logprobs=torch.ones_like(r.logprobs), mask=mask, lengths=lengths)
            h = acq.choice_logprobs_grad(x.contiguous(), r, choices, grad_logprobs=torch.ones_like(r.logprobs), mask=mask, lengths=lengths)
            assert torch.equal(g, h) and g.is_contiguous()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M", [5, 1024, 40000])
def test_rows_without_candidates_and_values_in_excluded_places(kind, M):
    rng = np.random.default_rng(M)
    x = scores_of(rng, kind, (8, M))
    mask = torch.ones(8, M, dtype=torch.bool, device="cuda")
    mask[:, 1] = False
    x[:, 1] = math.nan                                     # masked NaN
    mask[0], mask[1, 2:] = False, False                    # nothing; one candidate
    x[2] = -math.inf                                       # nothing by scores alone
    x[3, : M // 2] = torch.finfo(x.dtype).min              # the type's lowest value: a score like any other
    x[4, 3], x[5, 2] = math.nan, math.inf                  # NaN, +inf that exist
    mask[6, 4], x[6, 4] = False, math.inf                  # masked +inf
    x[7] = torch.finfo(x.dtype).min
    lengths = torch.full((8,), M, device="cuda")
    choices = torch.tensor([[0, 1, 2, -1]] * 8, device="cuda")
    k = 5
    r = acq.choice_logprobs(x, choices, mask=mask, lengths=lengths, top=k)
    check_choice(r, x, kind, choices, 1.0, mask, lengths, k)
    assert abs(float(r.entropy[7]) - math.log(M - 1)) < 1e-4 and abs(float(r.logprobs[7, 0]) + math.log(M - 1)) < 1e-4  # all equal
    ones = lambda t: torch.ones_like(t)
    g = acq.choice_logprobs_grad(x, r, choices, grad_logprobs=ones(r.logprobs), grad_entropy=ones(r.entropy),
                                 grad_logsumexp=ones(r.logsumexp), grad_top_logprobs=torch.zeros_like(r.top_logprobs), mask=mask)
    g = host(g)
    assert not g[0].any() and not g[2].any() and not g[:, 1][[0, 1, 2, 3, 6, 7]].any()
    assert np.isnan(g[4, 0]) and np.isnan(g[5, 0]) and g[4, 1] == 0 and np.isfinite(g[[0, 1, 2, 3, 6, 7]]).all()
    u = torch.tensor([1.0, 1, 1, 1, 0, 0, 1, 1], device="cuda", dtype=ACC[kind])
    w = host(acq.pool_weights(x, mask=mask, row_weights=u))  # the NaN rows count for nothing and are not read
    close(w, ref.weights(host(x), None, 1.0, host(u), 1.0, host(mask)), ref.U[kind] * (400 + M / 8) * 8, "weights")
    w = host(acq.pool_weights(x, mask=mask))
    assert w[1] == 0 and np.isnan(w[[0] + list(range(2, M))]).all()
    bad = torch.full((8,), 1.0, device="cuda", dtype=ACC[kind])
    bad[3], bad[6], bad[7] = 0.0, -1.0, math.nan
    r = acq.choice_logprobs(x, temperature=bad, mask=mask)
    assert host(r.entropy[[3, 6, 7]]).size == np.isnan(host(r.entropy[[3, 6, 7]])).sum()


@pytest.mark.parametrize("kind", ["float64", "float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(1, 300), (3, 9000), (1, 131072), (2100, 1030)], ids=str)
@pytest.mark.parametrize("order", ["ascending", "descending", "constant", "few", "zeros"])
def test_alternatives_keep_their_order_among_equals(kind, shape, order):
    rng = np.random.default_rng(5)
    M = shape[1]
    row = {"ascending": np.arange(M) / 64.0, "descending": -np.arange(M) / 64.0, "constant": np.full(M, 1.5),
           "few": rng.integers(0, 3, M).astype(float), "zeros": np.where(rng.random(M) < 0.5, 0.0, -0.0)}[order]
    x = torch.as_tensor(np.broadcast_to(row, shape).copy(), device="cuda").to(getattr(torch, kind))
    v = host(x[0])
    for k in (1, 9, 64):
        want = np.argsort(-v, kind="stable")[:k]
        got = host(acq.choice_logprobs(x, top=k).top_indices)
        np.testing.assert_array_equal(got, np.broadcast_to(want, got.shape))


def test_gradient_against_differences():
    """(F(x + h) - F(x - h)) / 2h: off by h^2 / 6 times a third derivative below 30 here, and by the rounding of F over h
    (2^-53 |F| 200 / h): 1e-5 h gives 5e-10 + 1e-7 |F| 2e-2."""
    rng = np.random.default_rng(9)
    x = torch.as_tensor(rng.standard_normal((3, 41)), device="cuda")
    mask = torch.as_tensor(rng.random((3, 41)) > 0.2, device="cuda")
    choices = torch.tensor([[0, 5, 5, -1], [1, 2, 40, 3], [7, 7, 7, 9]], device="cuda")
    kw = dict(temperature=0.8, mask=mask)
    r = acq.choice_logprobs(x, choices, top=3, **kw)
    ok = torch.isfinite(r.logprobs)
    gs = [torch.as_tensor(rng.standard_normal(tuple(t.shape)), device="cuda") for t in (r.logprobs, r.entropy, r.logsumexp, r.top_logprobs)]

    def F(x):
        q = acq.choice_logprobs(x, choices, top=3, **kw)
        return float((gs[0] * torch.where(ok, q.logprobs, 0.0)).sum() + (gs[1] * q.entropy).sum() + (gs[2] * q.logsumexp).sum()
                     + (gs[3] * q.top_logprobs).sum())

    g = acq.choice_logprobs_grad(x, r, choices, grad_logprobs=gs[0], grad_entropy=gs[1], grad_logsumexp=gs[2], grad_top_logprobs=gs[3], **kw)
    h = 1e-5
    for i in range(3):
        for j in range(0, 41, 4):
            up, dn = x.clone(), x.clone()
            up[i, j] += h
            dn[i, j] -= h
            assert abs((F(up) - F(dn)) / (2 * h) - float(g[i, j])) <= 2e-8


W_SHAPES = [(1,), (1, 5), (0, 9), (3, 0), (17, 201), (1000, 1024), (33, 1025), (9, 4096), (21, 4097), (5, 8192), (6, 8193),
            (40, 16384), (3, 16385), (37, 40001), (3, 5, 700), (2, 130, 3000), (0, 4, 10)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", W_SHAPES, ids=str)
def test_pool_weights(kind, shape):
    rng = np.random.default_rng(zlib.crc32(repr((kind, shape, "w")).encode()))
    M, R = shape[-1], shape[-2] if len(shape) > 1 else 1
    for mask_kind, ragged, T_rows, old, rows in [("none", False, False, False, False), ("shared", True, True, True, True), ("full", True, False, True, False)]:
        x, mask, lengths, _, T = case_inputs(rng, kind, shape, mask_kind, ragged, 0, T_rows)
        wshape = shape[:1] + (M,) if len(shape) == 3 else (M,)
        w = torch.as_tensor(rng.random(wshape), device="cuda").to(ACC[kind]) if old else None
        u = None
        if rows:
            u = torch.as_tensor(np.where(rng.random(shape[:-1]) < 0.2, 0.0, rng.random(shape[:-1])), device="cuda").to(ACC[kind])
        got = acq.pool_weights(x, w, decay=0.75, row_weights=u, temperature=T, mask=mask, lengths=lengths)
        want = ref.weights(host(x), host(w), 0.75, host(u), host(T) if T_rows else T, host(mask), host(lengths))
        # each term: the error of its exponent as in log p (z below 60 here) and 4 roundings; R additions
        tol = ref.U[kind] * (200 + M / 64 + 8 * 120 + 8 + R) * (np.abs(want) + 2 ** -1000)
        close(host(got), want, tol, "weights")
        assert torch.equal(got, acq.pool_weights(x, w, decay=0.75, row_weights=u, temperature=T, mask=mask, lengths=lengths))
        if old:
            nothing = acq.pool_weights(x, torch.full_like(w, math.nan), decay=0.0, row_weights=u, temperature=T, mask=mask, lengths=lengths)
            assert torch.equal(nothing, acq.pool_weights(x, row_weights=u, temperature=T, mask=mask, lengths=lengths))
            acq.pool_weights(x, w, decay=0.75, row_weights=u, temperature=T, mask=mask, lengths=lengths, out=w)
            assert torch.equal(w, got)


def check_evict(w, budget, payload=(), **kw):
    lengths = kw.pop("lengths", None)
    got = acq.pool_evict(w, budget, payload, lengths=lengths, **kw)
    want = ref.evict(w.cpu().numpy(), budget, [p.cpu().numpy() for p in payload], lengths=host(lengths), **kw)
    np.testing.assert_array_equal(host(got.indices), want[0])
    np.testing.assert_array_equal(got.lengths.cpu().numpy(), want[1])
    np.testing.assert_array_equal(got.weights.cpu().numpy(), want[2])
    for a, b in zip(got.payload, want[3]):
        np.testing.assert_array_equal(a.cpu().numpy(), b)


E_SHAPES = [((1,), 1), ((7,), 3), ((201,), 50), ((64,), 64), ((65,), 100), ((4, 1023), 1), ((3, 1025), 1024), ((5, 16384), 4096),
            ((2, 16385), 5000), ((1, 100003), 33333), ((3, 20480), 2047), ((2, 0), 4), ((0, 5), 2), ((300, 40), 17)]


@pytest.mark.parametrize("kind", ["float64", "float32"])
@pytest.mark.parametrize("shape,budget", E_SHAPES, ids=str)
def test_pool_evict(kind, shape, budget):
    rng = np.random.default_rng(zlib.crc32(repr((kind, shape, budget)).encode()))
    M = shape[-1]
    put = lambda a, k=kind: torch.as_tensor(a, device="cuda").to(getattr(torch, k))
    plain = rng.lognormal(0, 3, shape)
    values = {"plain": plain, "zeros": np.where(rng.random(shape) < 0.9, 0.0, plain), "same": np.full(shape, 0.3), "few": rng.integers(0, 3, shape) - 1.0,
              # all but one agree in the 24 highest bits in which they differ from it
              "outlier": np.where(np.arange(M) == M // 2, 1e30, 1.0 + rng.integers(0, 50, shape) * 2.0 ** (-23 if kind == "float32" else -52)),
              "close": 1.0 + rng.integers(0, 50, shape) * 2.0 ** (-23 if kind == "float32" else -52), "signs": rng.standard_normal(shape),
              "special": np.where(rng.random(shape) < 0.2, rng.choice([np.nan, np.inf, -np.inf, -0.0, 0.0], shape), plain)}
    lens = torch.as_tensor(rng.integers(-1, M + 2, shape[:-1]), device="cuda")
    for name, v in values.items():
        points = put(rng.random(shape + (3,)))
        check_evict(put(v), budget, (points,))
        check_evict(put(v), budget, (points, put(rng.random(shape), "float32")), first=min(2, budget // 2), recent=budget // 3, lengths=lens)
    check_evict(put(plain), budget, (), first=budget)
    check_evict(put(plain), budget, (), recent=budget, lengths=lens.to(torch.int32))


def test_evict_moves_payload_of_every_width():
    rng = np.random.default_rng(1)
    w = torch.as_tensor(rng.random((3, 500)), device="cuda")
    payload = [torch.as_tensor(rng.integers(0, 255, (3, 500) + s), device="cuda").to(t) for s, t in
               [((), torch.uint8), ((3,), torch.uint8), ((5,), torch.int16), ((3,), torch.int32), ((3,), torch.int64), ((2,), torch.float64),
                ((0,), torch.float32), ((4, 64), torch.float32), ((71,), torch.uint8), ((45,), torch.int16), ((19,), torch.int32), ((601,), torch.float64)]]
    check_evict(w, 77, payload, first=3)
    check_evict(w, 77, payload, first=3, lengths=torch.tensor([0, 30, 400], device="cuda"))
    view = torch.as_tensor(rng.random((3, 500, 5)), device="cuda")[:, :, 1:4]
    check_evict(w, 77, (view,), recent=9)


def test_numpy_arrays_go_through_the_default_engine():
    rng = np.random.default_rng(2)
    for dt in (np.float64, np.float32, np.float16):
        kind = np.dtype(dt).name
        x = rng.standard_normal((7, 1500)).astype(dt)
        mask, lengths = rng.random(1500) > 0.3, rng.integers(0, 1501, 7).astype(np.int32)
        c = rng.integers(-1, 1500, (7, 4))
        r = acq.choice_logprobs(x[:, ::2], c // 2, temperature=0.9, mask=mask[::2], lengths=lengths // 2, top=5)
        assert all(isinstance(a, np.ndarray) for a in r)
        dev = lambda a: torch.as_tensor(np.ascontiguousarray(a), device="cuda")
        q = acq.choice_logprobs(dev(x[:, ::2]), dev(c // 2), temperature=0.9, mask=dev(mask[::2]), lengths=dev(lengths // 2), top=5)
        for a, b in zip(r, q):
            np.testing.assert_array_equal(a, b.cpu().numpy())
        gl = rng.standard_normal((7, 4)).astype(r.entropy.dtype)
        g = acq.choice_logprobs_grad(x[:, ::2], r, c // 2, grad_logprobs=gl, temperature=0.9, mask=mask[::2], lengths=lengths // 2)
        h = acq.choice_logprobs_grad(dev(x[:, ::2]), q, dev(c // 2), grad_logprobs=dev(gl), temperature=0.9, mask=dev(mask[::2]), lengths=dev(lengths // 2))
        np.testing.assert_array_equal(g, h.cpu().numpy())
        np.testing.assert_array_equal(acq.pool_weights(x, temperature=0.5, mask=mask), acq.pool_weights(dev(x), temperature=0.5, mask=dev(mask)).cpu().numpy())
        out = np.zeros(1500, dtype=r.entropy.dtype)
        assert acq.pool_weights(x, out=out) is out and abs(out.sum() - 7) < 1e-3
    w = rng.random(900)
    pts = rng.random((900, 2))
    e = acq.pool_evict(w, 100, (pts,), first=2, recent=3)
    want = ref.evict(w, 100, [pts], 2, 3)
    for a, b in zip((e.indices, e.lengths, e.weights, e.payload[0]), (*want[:3], want[3][0])):
        np.testing.assert_array_equal(a, b)
    one = acq.choice_logprobs([0.0, 1.0, 2.0], 2, top=1)  # a list, a single choice
    assert one.logprobs.shape == () and abs(float(one.logprobs) + math.log(1 + math.exp(-1) + math.exp(-2))) < 1e-15
    assert one.top_indices.tolist() == [2]


def test_offsets_beyond_32_bits():
    rows, M = 40000, 65536  # 2.6e9 scores, 5.2 GB
    x = torch.zeros(rows, M, device="cuda", dtype=torch.bfloat16)
    last = torch.randn(3, M, device="cuda").to(torch.bfloat16)
    x[-3:] = last
    choices = torch.full((rows, 1), 5, device="cuda")
    r = acq.choice_logprobs(x, choices, top=2)
    q = acq.choice_logprobs(last, choices[:3], top=2)
    assert torch.equal(r.top_indices[-3:], q.top_indices)
    torch.testing.assert_close(r.logprobs[-3:], q.logprobs, rtol=1e-5, atol=0)
    assert torch.all((r.logsumexp[:-3] - math.log(M)).abs() < 1e-5)
    g = acq.choice_logprobs_grad(x, r, choices, grad_logprobs=torch.ones_like(r.logprobs))
    h = acq.choice_logprobs_grad(last, q, choices[:3], grad_logprobs=torch.ones_like(q.logprobs))
    torch.testing.assert_close(g[-3:].float(), h.float(), rtol=2 ** -7, atol=0)
    assert torch.all(g[:-3:1000, 5] == 1.0)
    w = acq.pool_weights(x)
    want = (rows - 3) / M + torch.softmax(last.double(), 1).sum(0)
    torch.testing.assert_close(w.double(), want, rtol=1e-3, atol=0)


def test_a_step_is_captured_and_replayed():
    """Forward, gradient, weights and eviction in one graph, replayed with other inputs and eager work in between."""
    rng = np.random.default_rng(4)
    x = scores_of(rng, "float64", (6, 20011))
    small = scores_of(rng, "float32", (4, 40, 900))
    mask = torch.as_tensor(rng.random(20011) > 0.1, device="cuda")
    choices = torch.as_tensor(rng.integers(0, 20011, (6, 4)), device="cuda")
    gl = torch.as_tensor(rng.standard_normal((6, 4)), device="cuda")
    pts = torch.as_tensor(rng.random((20011, 2)), device="cuda")

    def step():
        r = acq.choice_logprobs(x, choices, mask=mask, top=9)
        g = acq.choice_logprobs_grad(x, r, choices, grad_logprobs=gl, grad_entropy=torch.ones_like(r.entropy), mask=mask)
        w = acq.pool_weights(x, mask=mask, temperature=0.5)
        e = acq.pool_evict(w, 3000, (pts,), recent=5)
        v = acq.pool_weights(small)
        d = acq.pool_evict(v, 100)
        return [*r, g, w, e.indices, e.lengths, e.weights, e.payload[0], v, d.indices, d.weights]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        x.copy_(scores_of(rng, "float64", (6, 20011)))
        small.copy_(scores_of(rng, "float32", (4, 40, 900)))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b), i


def test_other_streams_and_threads():
    rng = np.random.default_rng(6)
    xs = [scores_of(rng, "float64", (5, 50021)) for _ in range(4)]
    want = [acq.choice_logprobs(x, top=8) for x in xs]
    got, errors = [None] * 4, []
    torch.cuda.synchronize()

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(20):
                    got[i] = acq.choice_logprobs(xs[i], top=8)
            s.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    for a, b in zip(got, want):
        for u, v in zip(a[1:], b[1:]):
            assert torch.equal(u, v)


def test_a_loop_of_the_operators_together():
    """Draws come in, gather weights, the pool is cut, the rest of the draws' scores follow the kept indices, and the policy
    over what is left names its choices: three rounds, every result against the plain implementations."""
    rng = np.random.default_rng(11)
    M, rows = 3000, 64
    points = torch.as_tensor(rng.random((M, 2)), device="cuda")
    w = torch.zeros(M, device="cuda", dtype=torch.float64)
    hp, hw = host(points), host(w)
    for budget in (2000, 700, 70):
        x = torch.as_tensor(rng.standard_normal((rows, len(hw))), device="cuda")
        w = acq.pool_weights(x, w, decay=0.9, temperature=0.4)
        hw = ref.weights(host(x), hw, 0.9, T=0.4)
        np.testing.assert_allclose(host(w), hw, rtol=1e-12)
        e = acq.pool_evict(w, budget, (points,), first=3, recent=5)
        i, n, hw, (hp,) = ref.evict(host(w), budget, [hp], 3, 5)  # of the device's own weights: equal ones are told apart by index
        np.testing.assert_array_equal(host(e.indices), i)
        assert int(e.lengths) == n == budget
        np.testing.assert_array_equal(host(e.payload[0]), hp)
        w, points = e.weights, e.payload[0]
        kept = x[:, e.indices]
        r = acq.choice_logprobs(kept, e.indices.new_zeros(rows, 1), temperature=0.4, top=5)
        check_choice(r, kept, "float64", e.indices.new_zeros(rows, 1), 0.4, None, None, 5)
        g = acq.choice_logprobs_grad(kept, r, e.indices.new_zeros(rows, 1), grad_logprobs=torch.ones_like(r.logprobs), temperature=0.4)
        assert float(g.sum(1).abs().max()) < 1e-12  # a softmax's gradient sums to nothing


def test_models_feed_the_pool_on_the_gpu():
    import bench_inputs
    from gpax_amd import ExactGP
    from gpax_amd.utils import get_keys
    _lib.set_engine(None)
    X, y, Xn, _ = bench_inputs.synthetic_problem(60, 2, 200, seed=3)
    m = ExactGP(2, "Matern")
    m.fit(get_keys()[0], X, y, num_warmup=20, num_samples=20, progress_bar=False, print_summary=False)
    _, draws = m.predict(get_keys()[1], Xn, n=3)
    want = ref.weights(-np.asarray(draws).reshape(-1, 200), T=0.3) / 60
    p = acq.PBest(get_keys()[1], m, Xn, temperature=0.3, n=3)
    np.testing.assert_allclose(p, want, rtol=1e-11)
    Xk, w, idx = acq.shrink_pool(get_keys()[1], m, Xn, 50, recent=4, temperature=0.3, n=3)
    keep = np.sort(np.concatenate([np.argsort(-want[:196], kind="stable")[:46], np.arange(196, 200)]))
    np.testing.assert_array_equal(idx, keep)
    np.testing.assert_array_equal(Xk, Xn[keep])
    np.testing.assert_allclose(w, 60 * want[keep], rtol=1e-11)
    r = acq.choice_logprobs(acq.UCB(get_keys()[1], m, Xk, n=2), top=4, temperature=0.1)
    assert r.top_indices.shape == (4,) and np.all(np.diff(r.top_logprobs) <= 0) and np.exp(r.top_logprobs).sum() <= 1


def test_refusals_of_tensors():
    x = torch.zeros(3, 10, device="cuda")
    bad = [lambda: acq.choice_logprobs(x.cpu()), lambda: acq.choice_logprobs(x.int()), lambda: acq.choice_logprobs(x.requires_grad_(True)),
           lambda: acq.choice_logprobs(x[None, None]), lambda: acq.choice_logprobs(x, top=65), lambda: acq.choice_logprobs(x, top=-1),
           lambda: acq.choice_logprobs(x, temperature=0.0), lambda: acq.choice_logprobs(x, temperature=math.inf),
           lambda: acq.choice_logprobs(x, temperature=torch.ones(3, device="cuda", dtype=torch.float64)),
           lambda: acq.choice_logprobs(x, mask=torch.ones(9, device="cuda", dtype=torch.bool)),
           lambda: acq.choice_logprobs(x, mask=torch.ones(3, 10, device="cuda")), lambda: acq.choice_logprobs(x, mask=np.ones(10, dtype=bool)),
           lambda: acq.choice_logprobs(x, torch.zeros(2, 1, device="cuda", dtype=torch.int64)),
           lambda: acq.choice_logprobs(x, torch.zeros(3, 1, device="cuda")), lambda: acq.choice_logprobs(x, lengths=torch.ones(2, device="cuda", dtype=torch.int64)),
           lambda: acq.pool_weights(x, torch.zeros(9, device="cuda")), lambda: acq.pool_weights(x, decay=-1.0), lambda: acq.pool_weights(x, decay=math.nan),
           lambda: acq.pool_weights(x, torch.zeros(10, device="cuda", dtype=torch.float64)), lambda: acq.pool_weights(x, out=torch.zeros(20, device="cuda")[::2]),
           lambda: acq.pool_weights(x, row_weights=torch.zeros(4, device="cuda")),
           lambda: acq.pool_evict(x, 0), lambda: acq.pool_evict(x, 4, first=3, recent=2), lambda: acq.pool_evict(x, 4, first=-1),
           lambda: acq.pool_evict(x.half(), 4), lambda: acq.pool_evict(x, 4, (torch.zeros(3, 9, 2, device="cuda"),)), lambda: acq.pool_evict(x[None], 4),
           lambda: acq.pool_evict(x, 4, (x,) * 17), lambda: acq.pool_evict(x, 4, lengths=torch.ones(4, device="cuda", dtype=torch.int64))]
    for i, call in enumerate(bad):
        x.requires_grad_(False)
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    x.requires_grad_(False)
    r = acq.choice_logprobs(x, torch.zeros(3, 1, device="cuda", dtype=torch.int64), top=2)
    with pytest.raises(ValueError):
        acq.choice_logprobs_grad(x, r, grad_logprobs=r.logprobs)
    with pytest.raises(ValueError):
        acq.choice_logprobs_grad(x, r, grad_entropy=torch.zeros(4, device="cuda"))
    with pytest.raises(ValueError):
        acq.choice_logprobs_grad(x, tuple(r), grad_entropy=r.entropy)
    outside = acq.choice_logprobs(x, torch.tensor([[10], [-2], [-1]], device="cuda")).logprobs
    assert torch.isnan(outside[:2]).all() and outside[2] == 0  # on the device: never read


def test_the_library_refuses_what_the_kernels_do_not_take():
    eng = _lib.get_device_engine(0)
    names = ("d_scores pools rows candidates x0 x1 x2 d_mask m0 m1 m2 d_lengths l0 l1 d_temperatures t0 t1 temperature dtype "
             "lengths_64").split()
    scores = lambda **kw: _lib.POOL_SCORES.pack(*[kw.get(n, 0) for n in names])
    ok = dict(d_scores=1 << 20, pools=1, rows=2, candidates=8, temperature=1.0, dtype=0)
    for change in [dict(dtype=4), dict(rows=-1), dict(candidates=1 << 31), dict(rows=1 << 26), dict(temperature=0.0), dict(temperature=math.nan), dict(d_scores=0)]:
        s = scores(**{**ok, **change})
        with pytest.raises(_lib.GpxError):
            eng.choice_logprobs(s, 0, 0, 0, 1, 1, 1, 1, 1, 1, 0, 0, 0)
    s = scores(**ok)
    for args in [(0, 0, 65), (0, -1, 0), (0, 1, 0)]:
        with pytest.raises(_lib.GpxError):
            eng.choice_logprobs(s, *args, 1, 1, 1, 1, 1, 1, 0, 0, 0)
    long = scores(**{**ok, "candidates": 1 << 20})
    with pytest.raises(_lib.GpxError):  # needs a workspace
        eng.choice_logprobs(long, 0, 0, 0, 1, 1, 1, 1, 1, 1, 0, 0, 0)
    with pytest.raises(_lib.GpxError):
        eng.pool_evict(0, 1, 8, 0, 0, False, 0, 4, 0, 0, 1, 1, 1, [], [], [], 0, 0, 0)
    with pytest.raises(_lib.GpxError):  # needs a workspace
        eng.pool_evict(0, 1, 1 << 20, 1, 0, False, 0, 4, 0, 0, 1, 1, 1, [], [], [], 0, 0, 0)
    for first, recent in [(1 << 62, 1 << 62), (5, 0), (0, 5), (4, 1)]:
        with pytest.raises(_lib.GpxError):
            eng.pool_evict(0, 1, 8, 1, 0, False, 0, 4, first, recent, 1, 1, 1, [], [], [], 0, 0, 0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M", [1024, 5000, 70001])
def test_alternatives_beside_nan_scores(kind, M):
    """NaN scores are never alternatives, and hide none: lanes that meet nothing else, a few places, nearly all of them."""
    rng = np.random.default_rng(M)
    for share, top in [("lanes", 20), ("lanes", 40), ("few", 64), ("most", 30)]:
        x = scores_of(rng, kind, (3, M))
        if share == "lanes":  # 16 neighbours of every 64: whole vectors of some lanes
            x[:, torch.arange(M, device="cuda") % 64 < 16] = math.nan
        else:
            x[torch.as_tensor(rng.random((3, M)) < (0.01 if share == "few" else 0.97), device="cuda")] = math.nan
        r = acq.choice_logprobs(x, top=top)
        assert torch.isnan(r.entropy).all()
        np.testing.assert_array_equal(host(r.top_indices), ref.choice(host(x), top=top)["top_indices"])


def test_out_lies_apart_from_what_is_read():
    x = torch.randn(4, 64, device="cuda")
    w = torch.randn(64, device="cuda")
    want = acq.pool_weights(x, w, decay=0.5)
    before = w._version
    assert torch.equal(acq.pool_weights(x, w, decay=0.5, out=w), want) and w._version > before
    room = torch.zeros(4, 64, device="cuda")
    assert acq.pool_weights(x, out=room[2]).data_ptr() == room[2].data_ptr()
    both = torch.zeros(80, device="cuda")
    for call in [lambda: acq.pool_weights(x, out=x[1]), lambda: acq.pool_weights(x, both[:64], out=both[16:]),
                 lambda: acq.pool_weights(x, row_weights=both[60:64], out=both[:64]), lambda: acq.pool_weights(x, temperature=both[:4] + 1, out=x[3]),
                 lambda: acq.pool_weights(x, mask=room.view(torch.uint8)[0, :64], out=room[0])]:
        with pytest.raises(ValueError):
            call()
    assert acq.pool_weights(x, both[:16].new_zeros(64), out=both[:64]).data_ptr() == both.data_ptr()


def test_lazily_conjugated_and_negated_payload():
    z = torch.randn(9, 3, dtype=torch.complex64, device="cuda")
    w = torch.randn(9, device="cuda")
    for rows in (z.conj(), z.conj().imag):
        r = acq.pool_evict(w, 4, (rows,))
        assert torch.equal(r.payload[0], rows[r.indices])
    assert torch.equal(acq.pool_evict(z[:, 0].conj().imag, 4).weights, z[:, 0].conj().imag[acq.pool_evict(-z[:, 0].imag, 4).indices])


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", [(3, 1024), (2, 5000), (2, 70001)], ids=str)
def test_alternatives_of_scores_that_lie_close_together(kind, shape, sign):
    """Scores that differ in their last bits only, around a large value of either sign, many of them equal; and rows that rise or
    fall all along, so that every step passes every threshold or none does."""
    rng = np.random.default_rng(shape[1])
    step = {"float64": 1e-12, "float32": 1e-3, "bfloat16": 8.0, "float16": 1.0}[kind]
    near = torch.as_tensor(sign * (1000.0 + step * rng.standard_normal(shape)), device="cuda").to(getattr(torch, kind))
    ramp = torch.linspace(-50, 50, shape[1], device="cuda", dtype=torch.float64).expand(shape).to(getattr(torch, kind)) * sign
    for x in (near, ramp):
        for top in (1, 20, 25, 64):
            r = acq.choice_logprobs(x, top=top)
            np.testing.assert_array_equal(host(r.top_indices), ref.choice(host(x), top=top)["top_indices"])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", [(600, 133, 1030), (300, 140, 4500), (260, 135, 9001), (1, 9001, 16500)], ids=str)
def test_pool_weights_of_many_rows(kind, shape):
    """More rows than a workgroup fetches the particulars of at once, in both kernels; some of them empty, of weight 0 or NaN."""
    g = torch.Generator(device="cuda").manual_seed(shape[1])
    pools, R, M = shape
    x = torch.empty(shape, device="cuda", dtype=getattr(torch, kind)).normal_(generator=g).mul_(2)
    lengths = torch.randint(0, M + 1, (pools, R), device="cuda", generator=g)
    lengths[:, ::7] = 0
    lengths[:, 1::7] = M
    u = torch.rand(pools, R, device="cuda", generator=g, dtype=ACC[kind])
    u[:, 3::5] = 0
    mask = torch.rand(M, device="cuda", generator=g) > 0.2
    x[:, 70, :3] = math.nan
    u[: (pools + 1) // 2, 70] = 0  # half of the pools do not read it
    got = acq.pool_weights(x, row_weights=u, temperature=0.7, mask=mask, lengths=lengths)
    want = torch.zeros(pools, M, device="cuda", dtype=torch.float64)
    at = torch.arange(M, device="cuda")
    poisoned = torch.zeros(pools, M, dtype=torch.bool, device="cuda")
    for r0 in range(0, R, 128):
        z = x[:, r0:r0 + 128].double() / 0.7
        ok = mask & (at < lengths[:, r0:r0 + 128, None])
        if r0 <= 70 < r0 + 128:
            n, v = ok[:, 70 - r0], u[:, 70]
            poisoned = n & ((v != 0) & (n & torch.isnan(x[:, 70])).any(1))[:, None]
            z[:, 70 - r0] = 0
            ok[:, 70 - r0] = False
        z.masked_fill_(~ok, -math.inf)
        e = torch.exp(z - z.amax(2, keepdim=True).clamp_min(-1e300))  # (torch.softmax of float64 is right to 1e-7 only here)
        p = e / e.sum(2, keepdim=True).clamp_min(1e-300)
        want += torch.bmm(u[:, None, r0:r0 + 128].double(), p.contiguous())[:, 0]
    want[poisoned] = math.nan
    tol = ref.U[kind] * (200 + M / 64 + 8 * 120 + 8 + R) * (host(want.nan_to_num(0.0)) + 2 ** -1000)
    close(host(got), host(want), tol, "weights")
    assert torch.equal(got[: (pools + 1) // 2].nan_to_num(7), acq.pool_weights(x, row_weights=u, temperature=0.7, mask=mask, lengths=lengths)[: (pools + 1) // 2].nan_to_num(7))


@pytest.mark.parametrize("kind", ["float64", "float32"])
@pytest.mark.parametrize("shape", [(65536,), (524288,), (524289,), (2, 700001), (3, 1048577)], ids=str)
def test_evict_from_very_long_pools(kind, shape):
    """Pools of up to 2^19 candidates and more; many of them may agree in their upper bits, or in all of them."""
    g = torch.Generator(device="cuda").manual_seed(shape[-1])
    M, budget = shape[-1], shape[-1] // 3
    tiny = 2.0 ** (-23 if kind == "float32" else -52)
    uniform = torch.rand(shape, device="cuda", generator=g, dtype=torch.float64)
    near = 1.0 + torch.randint(0, 200, shape, device="cuda", generator=g) * tiny
    outlier = near.clone()
    outlier[..., M // 2] = 1e30
    flat_top = 1.0 + 1e-5 * uniform  # nothing but the last 36 bits
    flat_top[..., 7] = 100.0
    for values in (uniform, near, outlier, flat_top, torch.zeros_like(near), torch.exp(3 * torch.randn(shape, device="cuda", generator=g, dtype=torch.float64))):
        w = values.to(getattr(torch, kind))
        pts = torch.rand(shape + (2,), device="cuda", generator=g)
        got = acq.pool_evict(w, budget, (pts,), first=3, recent=10)
        flat = w.reshape(-1, M)
        for b in range(len(flat)):
            free = flat[b, 3:M - 10]
            order = torch.sort(free, descending=True, stable=True).indices[:budget - 13] + 3
            want = torch.cat([torch.arange(3, device="cuda"), torch.sort(order).values, torch.arange(M - 10, M, device="cuda")])
            assert torch.equal(got.indices.reshape(-1, budget)[b], want)
            assert torch.equal(got.payload[0].reshape(-1, budget, 2)[b], pts.reshape(-1, M, 2)[b][want])


def test_evict_from_forty_million():
    w = torch.rand(40_000_000, device="cuda", dtype=torch.float64)
    got = acq.pool_evict(w, 1000)
    want = torch.sort(torch.topk(w, 1000).indices).values
    assert torch.equal(got.indices, want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", [(4, 200), (3, 1024), (2, 20000), (2, 70001)], ids=str)
def test_alternatives_around_zero(kind, shape):
    """Zeros of both signs and the smallest numbers there are, among the largest and the lowest ones."""
    rng = np.random.default_rng(shape[1])
    info = torch.finfo(getattr(torch, kind))
    tiny = {"float64": 5e-324, "float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -24}[kind]
    for pool in ([0.0, -0.0, -1.0], [0.0, -0.0, tiny, -tiny, 2 * tiny, -1.0], [-tiny, -2 * tiny, -3 * tiny, info.min], [info.max, info.min, 0.0, tiny]):
        for rare in (False, True):  # all of them often, or the last one nearly everywhere
            p = None if not rare else np.r_[np.full(len(pool) - 1, 0.01), 1 - 0.01 * (len(pool) - 1)]
            x = torch.as_tensor(rng.choice(np.array(pool), shape, p=p), device="cuda").to(getattr(torch, kind))
            for top in (1, 20, 64):
                np.testing.assert_array_equal(host(acq.choice_logprobs(x, top=top).top_indices), ref.choice(host(x), top=top)["top_indices"])

"""GPU: the operators over a pool of candidates at the ends of their ranges: row weights that are not finite, rows of weight 0,
scores a whole range apart, arguments that overlap, tangents, many long pools."""
import math

import numpy as np
import pytest
import torch  # before libgpx is loaded: one HIP runtime for both

from gpax_amd import _lib
from gpax_amd import acquisition as acq
from tests import pool_oracle as ref

pytestmark = pytest.mark.gpu

KINDS = ["float64", "float32", "bfloat16", "float16"]
ACC = {"float64": torch.float64, "float32": torch.float32, "bfloat16": torch.float32, "float16": torch.float32}


def host(t):
    return t.double().cpu().numpy()


# one pass a row a wave, a row a workgroup, two passes
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M", [1000, 5000, 20000])
@pytest.mark.parametrize("strided", [False, True], ids=["dense", "strided"])
@pytest.mark.parametrize("weight", [math.inf, -math.inf, math.nan], ids=str)
def test_row_weights_that_are_not_finite(kind, M, strided, weight):
    """u p is u itself for every candidate that exists (p > 0 here: scores within 8 of each other), and nothing where none does."""
    rng = np.random.default_rng(M)
    step = 2 if strided else 1
    x = torch.as_tensor(rng.uniform(-4, 4, (3, M * step)), device="cuda").to(getattr(torch, kind))[:, ::step]
    x[1, 5], x[1, M - 2] = -math.inf, -math.inf
    mask = torch.as_tensor(rng.random(M) > 0.2, device="cuda")
    lengths = torch.tensor([M, M - M // 3, M], device="cuda")
    u = torch.tensor([1.0, weight, 0.5], device="cuda", dtype=ACC[kind])
    w = torch.rand(M, device="cuda", dtype=ACC[kind])
    got = host(acq.pool_weights(x, w, decay=0.5, row_weights=u, mask=mask, lengths=lengths))
    there = ref.allowed(host(x), mask.cpu().numpy(), lengths.cpu().numpy())[1]
    want = ref.weights(host(x), host(w), 0.5, np.array([1.0, 0.0, 0.5]), 1.0, mask.cpu().numpy(), lengths.cpu().numpy())
    np.testing.assert_array_equal(got[there], np.full(there.sum(), weight))
    # each of two terms: the error of its exponent (|z| below 8, 8 u 16), of the sum of M terms and of 4 roundings; two additions
    tol = ref.U[kind] * (200 + M / 64 + 8 * 16 + 8) * np.abs(want[~there])
    assert np.all(np.abs(got[~there] - want[~there]) <= tol)


NAMES = ("d_scores pools rows candidates x0 x1 x2 d_mask m0 m1 m2 d_lengths l0 l1 d_temperatures t0 t1 temperature dtype "
         "lengths_64").split()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,M", [(37, 40000), (600, 20000), (4100, 16500)], ids=str)
def test_rows_of_weight_0_are_not_read(kind, rows, M):
    """Pools that take two passes, with several workgroups, one, and one wave a row: nothing of such a row (its scores are 1000,
    the others below 40) gets into the statistics that the first pass leaves in the workspace."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.empty(rows, M, device="cuda").normal_(generator=g).clamp_(-40, 40).to(getattr(torch, kind))
    u = torch.rand(rows, device="cuda", generator=g, dtype=ACC[kind]) + 0.5
    u[1::3], x[1::3] = 0, 1000.0
    eng, dtype = _lib.get_device_engine(0), KINDS.index(kind)
    nbytes = _lib.load_library().gpx_pool_weights_workspace(1, rows, M, dtype)
    ws = torch.zeros(nbytes, dtype=torch.uint8, device="cuda")
    out = torch.empty(M, device="cuda", dtype=ACC[kind])
    fields = dict(d_scores=x.data_ptr(), pools=1, rows=rows, candidates=M, x1=M, x2=1, temperature=1.0, dtype=dtype)
    eng.pool_weights(_lib.POOL_SCORES.pack(*[fields.get(n, 0) for n in NAMES]), u.data_ptr(), 0, 0.0, out.data_ptr(), ws.data_ptr(),
                     nbytes, torch.cuda.current_stream().cuda_stream)
    left = ws[:nbytes // 8 * 8].view(ACC[kind])
    assert not (left == 1000.0).any()
    assert torch.equal(out, acq.pool_weights(x, row_weights=u))
    x[1::3] = math.nan
    assert torch.equal(out, acq.pool_weights(x, row_weights=u))
    z = x[u != 0].double()
    e = torch.exp(z - z.amax(1, keepdim=True))
    want = (u[u != 0].double()[:, None] * (e / e.sum(1, keepdim=True))).sum(0)
    # as for other weights: the error of an exponent with |z| below 40, the sum of M terms, 4 roundings, an addition a row
    assert torch.all((out.double() - want).abs() <= ref.U[kind] * (200 + M / 64 + 8 * 80 + 8 + rows) * want)


def test_tangents_are_refused():
    """Forward mode would lose them: no result has one."""
    from torch.autograd import forward_ad
    x, w = torch.randn(3, 10, device="cuda"), torch.rand(10, device="cuda")
    c = torch.zeros(3, 1, device="cuda", dtype=torch.int64)
    want = acq.choice_logprobs(x, c, top=2)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        dx, dw = dual(x), dual(w)
        assert not dx.requires_grad
        for call in [lambda: acq.choice_logprobs(dx, c), lambda: acq.choice_logprobs(x, temperature=dual(torch.ones(3, device="cuda"))),
                     lambda: acq.choice_logprobs_grad(x, want, c, grad_entropy=dual(torch.ones(3, device="cuda"))), lambda: acq.pool_weights(dx),
                     lambda: acq.pool_weights(x, dw), lambda: acq.pool_weights(x, out=dw), lambda: acq.pool_evict(dw, 4),
                     lambda: acq.pool_evict(w, 4, (dual(torch.rand(10, 2, device="cuda")),))]:
            with pytest.raises(ValueError):
                call()
            with torch.no_grad(), pytest.raises(ValueError):
                call()
        plain = acq.choice_logprobs(forward_ad.unpack_dual(dx).primal, c, top=2)  # no tangent: as ever
        assert acq.pool_evict(w, 4, (c.expand(3, 10).t(),)).indices.shape == (4,)
    for a, b in zip(want, plain):
        assert torch.equal(a, b)


def test_out_may_lie_in_no_argument():
    """Temperatures, lengths and row weights of the same storage as `out`, behind its first element and before its last."""
    x = torch.randn(4, 64, device="cuda")
    room = torch.ones(80, device="cuda")
    ints = room.view(torch.int32)
    for kw in [dict(temperature=room[60:64]), dict(temperature=room[:1]), dict(row_weights=room[63:67]), dict(lengths=ints[60:64]), dict(lengths=ints[:1]),
               dict(temperature=room[::21][:4]), dict(lengths=room.view(torch.int64)[30:34])]:
        with pytest.raises(ValueError, match="overlaps"):
            acq.pool_weights(x, out=room[:64], **kw)
    assert acq.pool_weights(x, temperature=room[64:68], row_weights=room[68:72], lengths=ints[72:76], out=room[:64]).data_ptr() == room.data_ptr()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M", [3, 1000, 5000, 70001])
def test_log_probabilities_of_scores_a_whole_range_apart(kind, M):
    """The largest and the lowest number there are, over T = 8: their difference is infinite in the accumulator's type, the log
    probability is not.  Only three candidates exist: p = 1, 0, 0 in any type."""
    big = torch.finfo(getattr(torch, kind)).max
    x = torch.zeros(2, M, device="cuda", dtype=getattr(torch, kind))
    x[:, 0], x[:, M // 2], x[:, M - 1] = big, 0, -big
    mask = torch.zeros(M, device="cuda", dtype=torch.bool)
    mask[[0, M // 2, M - 1]] = True
    c = torch.tensor([[0, M // 2, M - 1, -1]] * 2, device="cuda")
    r = acq.choice_logprobs(x, c, temperature=8.0, mask=mask, top=3)
    want = np.array([[0.0, -(big / 8), -(big / 4), 0.0]] * 2)
    # each score by T, their difference, the logarithm of the sum: a rounding each
    assert np.all(np.abs(host(r.logprobs) - want) <= 4 * ref.U[kind] * np.abs(want))
    assert np.all(np.abs(host(r.top_logprobs) - want[:, :3]) <= 4 * ref.U[kind] * np.abs(want[:, :3]))
    assert r.top_indices.tolist() == [[0, M // 2, M - 1]] * 2
    g = torch.tensor([[0.0, 0.0, 4.0, 9.0]] * 2, device="cuda", dtype=ACC[kind])
    d = host(acq.choice_logprobs_grad(x, r, c, grad_logprobs=g, temperature=8.0, mask=mask))
    full = np.zeros((2, M))
    full[:, 0] -= 0.5
    full[:, M - 1] += 0.5  # (1 - p) g / T, and -p g / T
    np.testing.assert_array_equal(d, full)


def weights_that_agree(shape, g):
    """Weights that agree in their 36 upper bits, all over the pools, beside one that does not."""
    w = 1.0 + 1e-9 * torch.rand(shape, device="cuda", generator=g, dtype=torch.float64)
    w[..., 7] = 100.0
    return w


@pytest.mark.parametrize("shape", [(64, 65536), (65, 65537), (5, 250001), (130, 40961), (3, 524288)], ids=str)
def test_evict_from_several_long_pools_of_weights_that_agree(shape):
    """On both sides of the rule for the number of digits, which looks at all pools."""
    M, budget = shape[1], shape[1] // 3
    g = torch.Generator(device="cuda").manual_seed(M)
    w = weights_that_agree(shape, g)
    lengths = torch.randint(budget, M + 1, shape[:1], device="cuda", generator=g)
    got = acq.pool_evict(w, budget, first=3, recent=10, lengths=lengths)
    for b, n in enumerate(lengths.tolist()):
        order = torch.sort(w[b, 3:n - 10], descending=True, stable=True).indices[:budget - 13] + 3
        keep = torch.cat([torch.arange(3, device="cuda"), torch.sort(order).values, torch.arange(n - 10, n, device="cuda")])
        assert torch.equal(got.indices[b], keep if n > budget else torch.arange(budget, device="cuda"))


def test_evict_of_many_long_pools_takes_no_time_in_squares():
    """What agrees in its upper bits costs a few passes more, and not a pass for every chunk of 4096 (28 times as long here)."""
    g = torch.Generator(device="cuda").manual_seed(1)
    shape, times = (64, 524288), []
    for w in (torch.rand(shape, device="cuda", generator=g, dtype=torch.float64), weights_that_agree(shape, g)):
        acq.pool_evict(w, 100000)
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        for _ in range(3):
            acq.pool_evict(w, 100000)
        end.record()
        end.synchronize()
        times.append(start.elapsed_time(end))
    assert times[1] < 6 * times[0], times


def test_the_library_refuses_payload_without_its_arrays():
    import ctypes as C
    eng = _lib.get_device_engine(0)
    arrays, sizes = (C.c_void_p * 1)(1), (C.c_int64 * 1)(8)
    for args in [(None, arrays, sizes), (arrays, None, sizes), (arrays, arrays, None)]:
        with pytest.raises(_lib.GpxError, match="payload"):
            eng._check(eng._lib.gpx_pool_evict(eng._ctx, 0, 1, 8, 1, 0, 0, 0, 4, 0, 0, 1, 1, 1, 1, *args, 0, 0, 0), "gpx_pool_evict")

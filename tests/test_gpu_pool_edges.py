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

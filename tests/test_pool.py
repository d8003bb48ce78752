"""CPU: argument handling, refusals and staging of the operators over a pool of candidates, with a stand-in engine on host
memory (tests/pool_engine.py); the plain implementations themselves against differences; the compiled code."""
import math
import os
import re
import subprocess

import numpy as np
import pytest

from gpax_amd import _lib
from gpax_amd import acquisition as acq
from tests import pool_oracle as ref
from tests.pool_engine import PoolEngine

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(autouse=True)
def engine():
    _lib.set_engine(PoolEngine())
    yield
    _lib.set_engine(None)


def test_the_plain_gradient_is_that_of_the_plain_results():
    rng = np.random.default_rng(0)
    x, mask, c, T = rng.standard_normal((3, 20)), rng.random((3, 20)) > 0.2, rng.integers(-1, 20, (3, 4)), 0.7
    f = ref.choice(x, c, T, mask, None, 3)
    gs = [rng.standard_normal(s) for s in ((3, 4), 3, 3, (3, 3))]
    g, _ = ref.grad(x, f, c, *gs, T=T)

    def F(x):
        q = ref.choice(x, c, T, mask, None, 3)
        return ((gs[0] * np.where(np.isfinite(q["logprobs"]), q["logprobs"], 0)).sum() + (gs[1] * q["entropy"]).sum()
                + (gs[2] * q["logsumexp"]).sum() + (gs[3] * q["top_logprobs"]).sum())

    h = 1e-5  # third derivatives below 30: h^2 / 6 x 30 = 5e-10; rounding 2^-53 x 200 x 30 / h = 7e-8
    for i in range(3):
        for j in range(20):
            up, dn = x.copy(), x.copy()
            up[i, j] += h
            dn[i, j] -= h
            assert abs((F(up) - F(dn)) / (2 * h) - g[i, j]) < 1e-7


def test_plain_results_of_a_row_by_hand():
    x = np.log(np.array([1.0, 2.0, 5.0, 8.0]))
    f = ref.choice(x, np.array([2, -1, 3]), 1.0, np.array([1, 1, 1, 0]), None, 4)
    p = np.array([1, 2, 5]) / 8
    np.testing.assert_allclose(f["logprobs"][0], [np.log(p[2]), 0, -np.inf])
    np.testing.assert_allclose(f["entropy"], -(p * np.log(p)).sum())
    np.testing.assert_allclose(f["logsumexp"], np.log(8.0))
    assert f["top_indices"][0].tolist() == [2, 1, 0, -1] and np.isneginf(f["top_logprobs"][0, 3])
    assert ref.evict(np.array([0.1, 0.5, 0.5, 0.0, 0.2]), 3, (), 1, 1)[0].tolist() == [0, 1, 4]


@pytest.mark.parametrize("shape", [(9,), (4, 9), (2, 3, 9), (0, 9), (3, 0)], ids=str)
@pytest.mark.parametrize("kind", ["float64", "float32", "float16"])
def test_staging_of_every_argument(shape, kind):
    rng = np.random.default_rng(1)
    lead, M = shape[:-1], shape[-1]
    acc = "float64" if kind == "float64" else "float32"
    x = rng.standard_normal(shape).astype(kind)
    for mask in [None, rng.random(M) > 0.3, (rng.random(shape) > 0.3).astype(np.uint8)]:
        for lengths in [None, np.asarray(rng.integers(0, M + 1, lead)), np.asarray(rng.integers(0, M + 1, lead[-1:] or ()), dtype=np.int32)]:
            for T in [0.5, rng.uniform(0.5, 2, lead).astype(acc)]:
                C = 2 if M else 0
                c = rng.integers(-1, M, lead + (2,)) if M else None
                r = acq.choice_logprobs(x, c, temperature=T, mask=mask, lengths=lengths, top=3)
                f = ref.choice(x, c, T, mask, lengths, 3)
                tol = dict(rtol=1e-6, atol=1e-6)
                np.testing.assert_allclose(r.entropy.reshape(-1), f["entropy"], **tol)
                np.testing.assert_array_equal(r.top_indices.reshape(-1, 3), f["top_indices"])
                assert r.entropy.shape == lead and r.entropy.dtype == acc
                assert r.logprobs is None if c is None else r.logprobs.shape == lead + (C,) and r.logprobs.dtype == acc
                g = acq.choice_logprobs_grad(x, r, c, grad_logprobs=np.ones(lead + (C,), acc) if C else None, grad_entropy=np.ones(lead, acc),
                                             temperature=T, mask=mask, lengths=lengths)
                want, _ = ref.grad(x, f, c, np.ones(lead + (C,)) if C else None, np.ones(lead), T=T)
                np.testing.assert_allclose(g.reshape(want.shape), want, rtol=2e-3, atol=2e-3 if kind == "float16" else 1e-6)
                w = acq.pool_weights(x, temperature=T, mask=mask, lengths=lengths)
                np.testing.assert_allclose(w, ref.weights(x, None, 1.0, None, T, mask, lengths), **tol)
                assert w.shape == (shape[:1] + (M,) if len(shape) == 3 else (M,))


def test_arrays_of_the_other_byte_order():
    x = np.random.default_rng(3).standard_normal((2, 6))
    a, b = acq.choice_logprobs(x.astype(">f8"), np.zeros((2, 1), ">i8"), top=2), acq.choice_logprobs(x, np.zeros((2, 1), int), top=2)
    np.testing.assert_array_equal(a.logprobs, b.logprobs)
    np.testing.assert_array_equal(acq.pool_evict(x.astype(">f8"), 3).weights, acq.pool_evict(x, 3).weights)


def test_one_choice_a_row_and_lists():
    r = acq.choice_logprobs([[0, 1], [2, 3]], [1, 0])
    np.testing.assert_allclose(r.logprobs, [-math.log(1 + math.exp(-1)), -1 - math.log(1 + math.exp(-1))])
    assert acq.choice_logprobs([0.0, 1.0], 1).logprobs.shape == ()


def test_eviction_moves_points_and_reports_lengths():
    w = np.array([[0.1, 0.9, 0.2, 0.8, 0.3], [1.0, 2.0, 3.0, 4.0, 5.0]])
    pts = np.arange(20.0).reshape(2, 5, 2)
    e = acq.pool_evict(w, 3, (pts,), recent=1, lengths=np.array([5, 2]))
    assert e.indices.tolist() == [[1, 3, 4], [0, 1, -1]] and e.lengths.tolist() == [3, 2]
    np.testing.assert_array_equal(e.payload[0][0], pts[0, [1, 3, 4]])
    assert not e.payload[0][1, 2].any() and e.weights[1].tolist() == [1.0, 2.0, 0.0]
    one = acq.pool_evict(w[0], 2, (pts[0].astype(np.float32), np.arange(5)))
    assert one.indices.tolist() == [1, 3] and one.lengths.shape == () and one.payload[1].tolist() == [1, 3]


def test_models_feed_the_pool():
    """PBest and shrink_pool on a fitted HMC and a VI model: the draws of predict through the plain implementations."""
    import bench_inputs
    from gpax_amd.models import ExactGP, viGP
    from gpax_amd.utils import get_keys
    Xt, y, Xn, _ = bench_inputs.synthetic_problem(20, 1, 15, seed=2)
    m = ExactGP(1, "RBF")
    m.fit(get_keys()[0], Xt, y, num_warmup=15, num_samples=15, progress_bar=False, print_summary=False)
    _, draws = m.predict(get_keys()[1], Xn, n=2)
    want = ref.weights(-draws.reshape(-1, 15), T=0.2) / 30
    p = acq.PBest(get_keys()[1], m, Xn, temperature=0.2, n=2)
    np.testing.assert_allclose(p, want, rtol=1e-12)
    assert abs(p.sum() - 1) < 1e-12
    Xk, w, idx = acq.shrink_pool(get_keys()[1], m, Xn[:, 0], 6, weights=np.full(15, 4.0), decay=0.5, recent=1, temperature=0.2, n=2)
    full = 2.0 + 30 * want
    keep = np.sort(np.append(np.argsort(-full[:14], kind="stable")[:5], 14))
    assert idx.tolist() == keep.tolist() and Xk.shape == (6, 1)
    np.testing.assert_allclose(w, full[keep], rtol=1e-12)
    np.testing.assert_array_equal(Xk, Xn[keep])
    v = viGP(1, "Matern")
    v.fit(get_keys()[0], Xt, y, num_steps=10, progress_bar=False, print_summary=False)
    q = acq.PBest(get_keys()[1], v, Xn, n=7, maximize=True)
    assert q.shape == (15,) and abs(q.sum() - 1) < 1e-12
    assert acq.shrink_pool(get_keys()[1], v, Xn, 40)[2].tolist() == list(range(15))


def test_draws_that_failed_have_no_say(monkeypatch):
    class Model:
        mcmc = object()

        def predict(self, key, X, n=1, noiseless=False, **kw):
            d = np.random.default_rng(0).standard_normal((4, n, len(X)))
            d[2] = np.nan
            return d.mean((0, 1)), d

    p = acq.PBest(0, Model(), np.zeros((5, 1)), n=3)
    d = np.delete(Model().predict(0, np.zeros((5, 1)), n=3)[1], 2, axis=0).reshape(-1, 5)
    np.testing.assert_allclose(p, ref.weights(-d, T=0.1) / 9, rtol=1e-12)


X = np.zeros((3, 10))
BAD = {
    "four dimensions": lambda: acq.choice_logprobs(X[None, None]), "a scalar": lambda: acq.choice_logprobs(np.float64(1)),
    "text": lambda: acq.choice_logprobs(np.array(["a"])), "complex": lambda: acq.choice_logprobs(X + 0j),
    "top": lambda: acq.choice_logprobs(X, top=65), "negative top": lambda: acq.choice_logprobs(X, top=-1),
    "temperature 0": lambda: acq.choice_logprobs(X, temperature=0), "temperature nan": lambda: acq.choice_logprobs(X, temperature=math.nan),
    "temperature that 32 bits do not hold": lambda: acq.choice_logprobs(X.astype(np.float32), temperature=1e-50),
    "temperature array": lambda: acq.choice_logprobs(X, temperature=np.array([1.0, -1.0, 1.0])),
    "temperature shape": lambda: acq.choice_logprobs(X, temperature=np.ones(2)),
    "mask shape": lambda: acq.choice_logprobs(X, mask=np.ones(9, bool)), "mask type": lambda: acq.choice_logprobs(X, mask=np.ones(10)),
    "mask with more dimensions": lambda: acq.choice_logprobs(X, mask=np.ones((1, 3, 10), bool)),
    "lengths shape": lambda: acq.choice_logprobs(X, lengths=np.ones(4, np.int64)), "lengths type": lambda: acq.choice_logprobs(X, lengths=np.ones(3)),
    "choice beyond": lambda: acq.choice_logprobs(X, np.full((3, 1), 10)), "choice below": lambda: acq.choice_logprobs(X, np.full((3, 1), -2)),
    "choice shape": lambda: acq.choice_logprobs(X, np.zeros((2, 1), int)), "choice type": lambda: acq.choice_logprobs(X, np.zeros((3, 1))),
    "weights shape": lambda: acq.pool_weights(X, np.zeros(9)), "decay": lambda: acq.pool_weights(X, decay=-0.1),
    "infinite decay": lambda: acq.pool_weights(X, decay=math.inf), "row weights": lambda: acq.pool_weights(X, row_weights=np.zeros(4)),
    "out shape": lambda: acq.pool_weights(X, out=np.zeros(9)), "out type": lambda: acq.pool_weights(X, out=np.zeros(10, np.float32)),
    "out strides": lambda: acq.pool_weights(X, out=np.zeros(20)[::2]),
    "budget": lambda: acq.pool_evict(X, 0), "protected": lambda: acq.pool_evict(X, 4, first=3, recent=2), "negative": lambda: acq.pool_evict(X, 4, recent=-1),
    "weights of three dimensions": lambda: acq.pool_evict(X[None], 4), "payload shape": lambda: acq.pool_evict(X, 4, (np.zeros((3, 9)),)),
    "many payloads": lambda: acq.pool_evict(X, 4, (X,) * 17), "payload type": lambda: acq.pool_evict(X, 4, (np.full((3, 10), "a"),)),
    "lengths of a row that is none of several": lambda: acq.choice_logprobs(X[0], lengths=np.ones(1, np.int64)),
    "temperatures of a row that is none of several": lambda: acq.pool_weights(X[0], temperature=np.ones(1)),
    "out read-only": lambda: acq.pool_weights(X, out=np.broadcast_to(np.zeros(10), (10,))),
    "lengths of pools": lambda: acq.pool_evict(X, 4, lengths=np.ones(2, np.int64)),
}


@pytest.mark.parametrize("name", BAD)
def test_refusals(name):
    with pytest.raises(ValueError):
        BAD[name]()


def test_gradient_refusals():
    r = acq.choice_logprobs(X, np.zeros((3, 1), int), top=2)
    for kw in [dict(grad_logprobs=r.logprobs), dict(grad_entropy=np.zeros(4)), dict(grad_top_logprobs=np.zeros((3, 3)))]:
        with pytest.raises(ValueError):
            acq.choice_logprobs_grad(X, r, **kw)
    with pytest.raises(ValueError):
        acq.choice_logprobs_grad(X, tuple(r), grad_entropy=r.entropy)
    with pytest.raises(ValueError):
        acq.choice_logprobs_grad(X[:2], r, grad_entropy=r.entropy[:2])


def test_tensors_on_the_host_are_refused():
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError):
        acq.choice_logprobs(torch.zeros(3))
    with pytest.raises(ValueError):
        acq.choice_logprobs(X, mask=torch.ones(10, dtype=torch.bool))


def test_workspace_sizes_come_from_sizes_alone():
    lib = _lib.load_library()
    assert lib.gpx_choice_workspace(1, 1000, 1024, 0, 8) == 0  # a row a wave
    assert lib.gpx_choice_workspace(1, 1, 1 << 20, 0, 64) > 0  # several workgroups a row
    assert lib.gpx_choice_workspace(1, -1, 4, 0, 0) < 0 and lib.gpx_choice_workspace(1, 1, 4, 9, 0) < 0 and lib.gpx_choice_workspace(1, 1, 4, 0, 65) < 0
    assert lib.gpx_pool_weights_workspace(1, 1, 10, 0) == 0 and lib.gpx_pool_weights_workspace(1, 1000, 1024, 0) > 0
    assert lib.gpx_pool_weights_workspace(-1, 1, 1, 0) < 0
    # sizes that the operators refuse have none (2^31 - 2^20 candidates, 2^25 rows, 65535 pools)
    assert lib.gpx_choice_workspace(1, 1, (1 << 31) - (1 << 20), 0, 1) < 0 and lib.gpx_choice_workspace(1 << 40, 1 << 40, 4, 0, 1) < 0
    assert lib.gpx_pool_weights_workspace(1 << 16, 1, 4, 0) < 0 and lib.gpx_pool_weights_workspace(1 << 13, 1 << 13, 4, 0) < 0
    assert lib.gpx_pool_evict_workspace(1 << 16, 4, 0) < 0 and lib.gpx_pool_evict_workspace(1, 1 << 31, 0) < 0
    assert lib.gpx_pool_evict_workspace(2, 16384, 0) == 0 and lib.gpx_pool_evict_workspace(2, 16385, 1) > 0


@pytest.mark.parametrize("source", ["choice.hip", "pool.hip"])
def test_no_scalar_move_has_a_literal_of_more_than_32_bits(source, tmp_path):
    """s_mov_b64 holds a literal of 32 bits; hipcc has emitted it with 64 (the double -inf), which loads 0."""
    out = tmp_path / "k.s"
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature",
                    "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "-S", os.path.join(ROOT, "gpax_amd", "csrc", source), "-o", str(out)],
                   check=True, stderr=subprocess.DEVNULL)
    text = out.read_text()
    assert "s_endpgm" in text
    bad = [m for m in re.findall(r"[sv]_mov_b64(?:_e32)? [sv]\[[0-9:]+\], (-?(?:0x[0-9a-f]+|[0-9]+))", text) if not -2 ** 31 <= int(m, 0) < 2 ** 32]
    assert not bad, bad


@pytest.mark.parametrize("kind,T", [("float32", 1e-39), ("float16", 1e-39), ("float32", 1e-45), ("float64", 1e-310), ("float64", 5e-324)])
def test_temperatures_too_small_to_divide_by(kind, T):
    """A positive number below the type's normal ones is refused in an array as it is alone: 1 / T may be infinite."""
    x = np.zeros((3, 10), dtype=kind)
    temps = np.ones(3, dtype="float64" if kind == "float64" else "float32")
    temps[1] = T
    assert 0 < temps[1] < np.finfo(temps.dtype).tiny
    for t in (T, temps, temps[1:2]):
        for call in (acq.choice_logprobs, acq.pool_weights):
            with pytest.raises(ValueError):
                call(x, temperature=t)
    temps[1] = np.finfo(temps.dtype).tiny
    assert np.all(acq.choice_logprobs(x, temperature=temps).entropy > 2)


@pytest.mark.parametrize("tasks", [1, 2, 4])
def test_models_of_several_targets_are_refused(tasks):
    """A vector-valued model draws (samples, n, tasks, M) at X of (tasks, M, d): cut into rows of X's length, they would weigh the
    tasks instead of the candidates."""
    import bench_inputs
    from gpax_amd.models import vExactGP
    from gpax_amd.utils import get_keys
    Xt, y, Xn, _ = bench_inputs.synthetic_problem(12, 1, 8, seed=2)
    m = vExactGP(1, "RBF")
    m.fit(get_keys()[0], np.stack([Xt] * tasks), np.stack([y + t for t in range(tasks)]), num_warmup=4, num_samples=4, progress_bar=False,
          print_summary=False)
    Xn = np.stack([Xn] * tasks)
    assert m.predict(get_keys()[1], Xn, n=2)[1].shape == (4, 2, tasks, 8)
    for X in (Xn, Xn[..., 0]):
        for call in (lambda: acq.PBest(get_keys()[1], m, X, n=2), lambda: acq.shrink_pool(get_keys()[1], m, X, 1)):
            with pytest.raises(ValueError):
                call()


def test_gradient_of_a_forward_call_on_other_rows():
    """Whichever gradient is given, `forward` has to be of the same rows."""
    x = np.random.default_rng(0).standard_normal((4, 6))
    r = acq.choice_logprobs(x, top=2)
    for kw in [dict(), dict(grad_logsumexp=np.ones(2)), dict(grad_entropy=np.ones(2)), dict(grad_top_logprobs=np.ones((2, 2)))]:
        with pytest.raises(ValueError):
            acq.choice_logprobs_grad(x[:2], r, **kw)
    with pytest.raises(ValueError):
        acq.choice_logprobs_grad(x.reshape(2, 2, 6), r, grad_logsumexp=np.ones((2, 2)))
    assert acq.choice_logprobs_grad(x, r, grad_logsumexp=np.ones(4)).shape == (4, 6)

"""sample on the B200 against the definition in f64 on the host: tokens and kept sets equal, probabilities
within f32 rounding."""
import numpy as np
import pytest

from _paged import to_storage

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    from tensor_cuda.backend import CudaBackend
    from tensor_cuda.runtime import Device
    return CudaBackend(Device.shared(0))


def up(be, arr, dtype):
    from tensor_cuda.backend import host
    return be.from_host_sync(host(dtype, np.shape(arr), np.asarray(arr)))


def define(x, u, t, k, p, m):
    """One row by the definition: (token, probability, size of the kept set)."""
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not len(order):
        return -1, 0.0, 0
    if not t > 0:
        return int(order[0]), 1.0, 1
    if k > 0:
        order = order[:k]
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        d = (x[order] - top) / np.float64(t)
    w = np.exp(np.where(x[order] == top, 0.0, np.where(np.isnan(d), -np.inf, d)))
    keep = len(w)
    if p < 1:
        keep = max(1, int(np.sum(np.cumsum(w) - w < np.float64(p) * w.sum())))
    keep = max(1, min(keep, int(np.sum(w >= np.float64(m)))))
    order, w = order[:keep], w[:keep]
    by = np.argsort(order)
    c = np.cumsum(w[by])
    u = min(max(float(u), 0.0), 1.0) if u == u else 0.0
    j = int(np.searchsorted(c, u * c[-1], side="right"))
    if j >= keep:
        j = int(np.nonzero(w[by])[0][-1])
    return int(order[by[j]]), w[by][j] / c[-1], keep


def check(be, x, dtype, u, t=1.0, k=0, p=1.0, m=0.0):
    raw, exact = to_storage(x, dtype)
    B = x.shape[0]
    row = lambda v, dt: np.broadcast_to(np.asarray(v, dt), (B,))  # noqa: E731
    ts, ks, ps, ms = row(t, np.float32), row(k, np.int32), row(p, np.float32), row(m, np.float32)
    dev = [v if np.ndim(v) == 0 else up(be, row(v, np.float32 if dt == "f32" else np.int32), dt)
           for v, dt in ((t, "f32"), (k, "i32"), (p, "f32"), (m, "f32"))]
    logits, ud = up(be, raw, dtype), up(be, np.asarray(u, np.float32), "f32")
    tok, prob, kept = (be.read_sync(a).data for a in be.sample(logits, ud, *dev, details=True))
    want = [define(exact[i], np.float32(u[i]), ts[i], int(ks[i]), ps[i], ms[i]) for i in range(B)]
    wt, wp, wk = (np.array(v) for v in zip(*want))
    assert np.array_equal(tok, wt), (tok, wt)
    assert np.array_equal(kept, wk), (kept, wk)
    # one rounding to f32; the sums are off by at most V 2^-47 of the total
    assert np.all(np.abs(prob - wp) <= 2.0 ** -24 * wp * 1.01 + 1e-45 + x.shape[1] * 2.0 ** -47 * wp)
    assert np.array_equal(be.read_sync(be.sample(logits, ud, *dev)).data, tok)


def uniform(n, seed=0):
    return np.random.default_rng(seed).random(n).astype(np.float32)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 1025, 4099, 50257])
def test_settings_per_row(be, dtype, vocab):
    r = np.random.default_rng(vocab)
    B = 24
    x = r.standard_normal((B, vocab)) * 3
    x[:, 5::11] = -np.inf
    check(be, x, dtype, uniform(B, 1), r.choice([0.0, 0.5, 1.0, 2.0], B), r.choice([0, 1, 2, 50, vocab, 10 ** 6], B),
          r.choice([0.3, 0.9, 0.999, 1.0], B), r.choice([0.0, 0.01, 0.3, 1.0], B))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_large_vocabulary_without_filters_and_with_top_p(be, dtype):
    x = np.random.default_rng(3).standard_normal((6, 200003)) * 2
    check(be, x, dtype, uniform(6, 2))
    check(be, x, dtype, uniform(6, 3), p=0.95)
    check(be, x, dtype, uniform(6, 4), k=100000)


def test_ties_go_to_the_lowest_index(be):
    """Rows of equal logits, and of few distinct values: borders of top-k and top-p inside a tie."""
    B = 12
    x = np.zeros((B, 5000))
    for k, p in ((0, 1.0), (7, 1.0), (0, 0.5), (4999, 0.25), (1, 0.01)):
        check(be, x, "f32", uniform(B, k), k=k, p=p)
    x = np.random.default_rng(1).integers(-3, 4, (B, 5000)).astype(np.float64)
    for k, p, m in ((0, 1.0, 0.0), (300, 1.0, 0.0), (2000, 0.7, 0.0), (0, 0.6, 0.1), (0, 1.0, 1.0)):
        check(be, x, "f16", uniform(B, k), k=k, p=p, m=m)
    check(be, np.array([[-0.0, 0.0, -0.0, 0.0]] * 4), "f32", [0.1, 0.3, 0.6, 0.9], k=2)


def test_rows_without_tokens_and_extreme_logits(be):
    inf, nan = np.inf, np.nan
    x = np.array([[-inf] * 6, [nan] * 6, [nan, -inf, 3, nan, -inf, nan], [inf, 1, inf, 2, -inf, 0],
                  [3e38, -3e38, 0, 3e38, 1, -inf], [-3e38, -inf, -3.1e38, nan, -inf, -3e38], [0, -200, -1000, 5, -800, 5]])
    for u in (0.0, 0.49, 0.51, 0.999):
        us = [u] * len(x)
        check(be, x, "f32", us)
        check(be, x, "f32", us, t=0.0)
        check(be, x, "f32", us, k=2, p=0.9)
        check(be, x, "f32", us, t=1e-6)
        check(be, x, "f32", us, t=1e6, p=0.4, m=0.5)
        check(be, x, "bf16", us, t=np.inf)


def test_ends_of_the_settings(be):
    x = np.random.default_rng(5).standard_normal((4, 300)) * 2
    u = [0.0, 1.0 - 2.0 ** -24, 1.0, 7.0]
    check(be, x, "f32", u)
    check(be, x, "f32", [-1.0, np.nan, 0.5, 0.2], p=0.8)
    check(be, x, "f32", u, p=0.0)
    check(be, x, "f32", u, p=-1.0, k=-5)
    check(be, x, "f32", u, m=2.0)
    check(be, x, "f32", u, t=np.nan)
    check(be, x, "f32", u, t=-1.0)


def test_draws_follow_the_weights(be):
    """Evenly spaced u give each token its share of the rows, within one row."""
    n = 2000
    logits = np.log(np.array([0.5, 0.25, 0.125, 0.0625, 0.0625]))
    x = np.broadcast_to(logits, (n, 5)).copy()
    u = (np.arange(n) + 0.5) / n
    tok = be.read_sync(be.sample(up(be, x.astype(np.float32), "f32"), up(be, u.astype(np.float32), "f32"))).data
    share = np.bincount(tok, minlength=5)
    assert np.all(np.abs(share - np.exp(logits) * n) <= 1.5)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_small_top_k_without_bins_by_value(be, dtype):
    """An infinite temperature, one whose inverse leaves f32, an infinite largest logit: the bins are by the logits'
    bits, and the kept set is the definition's for every top_k."""
    B, inf = 6, np.inf
    for vocab in (300, 1000, 20000):
        x = np.random.default_rng(vocab).standard_normal((B, vocab)) * 3
        x[:, 7::13] = -inf
        for k in (1, 2, 50, 192, 193):
            check(be, x, dtype, uniform(B, k), t=inf, k=k)
            check(be, x, dtype, uniform(B, k), t=inf, k=k, p=0.7)
            check(be, x, dtype, uniform(B, k), t=1e-38, k=k)
        x[:, [3, vocab // 2]] = inf
        for k in (1, 2, 3, 50, 192):
            check(be, x, dtype, uniform(B, k), k=k)
            check(be, x, dtype, uniform(B, k), t=inf, k=k)
    check(be, np.array([[inf, 1, inf, 2, 0]]), dtype, [0.7], k=4)


def test_min_p_above_one_keeps_the_first_rank(be):
    """No weight reaches a min_p above 1, so the rank that is always kept is left: of equal best logits the lowest
    index alone."""
    x = np.random.default_rng(2).standard_normal((4, 5000))
    x[:, [17, 400, 4999]] = 9.0
    for m in (1.0 + 2.0 ** -23, 2.0, np.inf):
        for kw in (dict(), dict(k=2), dict(p=0.9), dict(k=1000, p=0.9)):
            check(be, x, "f32", [0.0, 0.4, 0.7, 0.999], m=m, **kw)
    check(be, x, "f32", [0.0, 0.4, 0.7, 0.999], m=1.0)
    check(be, x, "f32", [0.0, 0.4, 0.7, 0.999], m=[1.0, 2.0, 1.0, 3.0])


def test_min_p_where_its_logit_leaves_the_range(be):
    """t ln(min_p) below f32's range, the logit where min_p lies within it: 3e38 - 4.02e38."""
    x = np.array([[-2e38, 3e38, -3e38, 0, 2.9e38, -1.1e38, -1e38]])
    for u in (0.0, 0.02, 0.3, 0.8, 0.95, 0.999):
        for kw in (dict(), dict(p=0.99), dict(k=6)):
            check(be, x, "f32", [u], t=1e38, m=0.018, **kw)


def test_vocabularies_beyond_the_sums_are_refused(be):
    """The weights' fixed point holds 2^20 tokens to 2^-23 of the largest weight; more are refused."""
    from tensor_cuda import _ffi as F
    n = 1 << 20
    x = np.full((1, n + 1), -20.0, np.float16)
    x[0, 5] = 0
    u = up(be, np.float32([0.5]), "f32")
    tok, prob, kept = (be.read_sync(a).data for a in be.sample(up(be, x[:, :n].copy(), "f16"), u, details=True))
    w = (n - 1) * np.exp(-20.0)
    # 2^20 weights rounded to 2^-42: 2^-23 of the total at most, and the rounding to f32
    assert tok[0] == 5 and kept[0] == n and abs(prob[0] - 1 / (1 + w)) <= 2.0 ** -23 + 2.0 ** -24
    with pytest.raises(F.MpcError, match="2\\^20 tokens") as e:
        be.sample(up(be, x, "f16"), u)
    assert e.value.status == F.ERR_UNSUPPORTED


@pytest.mark.parametrize("t", [5.0, 10.0, 300.0])
def test_flat_rows_cut_a_bin_again(be, t):
    """Hot temperatures over a large vocabulary: a bin of T / 256 holds far more than 256 different logits, at the
    borders of top_k and of top_p."""
    x = np.random.default_rng(11).standard_normal((8, 50257))
    for kw in (dict(k=5000, p=0.9), dict(k=5000), dict(p=0.9), dict(p=0.5, m=0.3), dict(k=40000, p=0.1), dict(k=50, p=0.9)):
        check(be, x, "f32", uniform(8, int(t)), t=t, **kw)


@pytest.mark.parametrize("rows,vocab", [(24, 3000), (400, 4099), (700, 20000), (5, 2048), (297, 2047)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_blocks_per_row(be, rows, vocab, dtype):
    """Shapes that give a row one, two, four or eight blocks, each with every kind of setting."""
    r = np.random.default_rng(rows)
    x = r.standard_normal((rows, vocab)) * r.choice([0.01, 1.0, 4.0], (rows, 1))
    check(be, x, dtype, uniform(rows, 1), r.choice([0.0, 0.7, 1.0, 20.0], rows), r.choice([0, 1, 40, 192, 500, 2000], rows),
          r.choice([0.5, 0.95, 1.0], rows), r.choice([0.0, 0.0, 0.05, 0.6], rows))
    check(be, x, dtype, uniform(rows, 2))

"""Paged caches on the host, in 64 bits: the reference values of the paged-cache tests."""
import numpy as np

from _helpers import f32_to_bf16_bits, bf16_bits_to_f32

EPS = {"f32": 2.0 ** -23, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}  # finfo(t).eps: a rounding is off by at most half


def to_storage(x, dtype):
    """(array to upload, its exact values in f64)."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == "f32":
        return x, x.astype(np.float64)
    if dtype == "f16":
        h = x.astype(np.float16)
        return h, h.astype(np.float64)
    bits = f32_to_bf16_bits(x).reshape(x.shape)
    return bits, bf16_bits_to_f32(bits).astype(np.float64).reshape(x.shape)


def from_storage(a, dtype):
    if dtype == "bf16":
        return bf16_bits_to_f32(np.asarray(a).view(np.uint16)).astype(np.float64).reshape(a.shape)
    return np.asarray(a).astype(np.float64)


def e4m3_values(codes):
    """Sign, 4 bits of exponent (bias 7), 3 of mantissa; all ones is NaN."""
    c = np.asarray(codes, np.int64)
    e, m = (c >> 3) & 15, (c & 7).astype(np.float64)
    v = np.where(e > 0, np.ldexp(1 + m / 8, (e - 7).astype(int)), np.ldexp(m, -9))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c > 127, -v, v)


_POSITIVE = e4m3_values(np.arange(127))  # ascending


def e4m3_codes(x):
    """Nearest of the 8-bit numbers, ties to the even code, saturating, NaN kept; x in f64."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.where(np.isnan(x), 0, np.abs(x)), 448.0)
    hi = np.searchsorted(_POSITIVE, a).clip(0, 126)
    lo = (hi - 1).clip(0)
    up, down = _POSITIVE[hi] - a, a - _POSITIVE[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)) | (_POSITIVE[hi] == a), hi, lo)
    code = np.where(np.isnan(x), 127, code)
    return np.where(np.signbit(x) & ~np.isnan(x), code + 128, code).astype(np.uint8)


def scale_bytes(rows):
    """The least e in [-126, 127] with the row's largest finite magnitude within 448 * 2^e, + 127."""
    a = np.where(np.isfinite(rows), np.abs(rows), 0).max(-1)
    b = np.ones(a.shape, np.int64)
    for e in range(-126, 128):
        b = np.where(a > 448.0 * 2.0 ** e, e + 1 + 127, b)
    return b.astype(np.uint8)


def quantised(rows):
    """(codes, scale bytes) of rows [..., d]."""
    b = scale_bytes(rows)
    with np.errstate(invalid="ignore"):
        return e4m3_codes(np.ldexp(rows, -(b.astype(int) - 127)[..., None])), b


class HostCache:
    """The pages of a cache as the device holds them, and where its rows are."""

    def __init__(self, n_pages, page_size, hk, d, dv, dtype, seed=0, fill=None):
        self.shape, self.dtype = (n_pages, page_size, hk, d, dv), dtype
        r = np.random.default_rng(seed)
        self.pages, self.scales = [], [None, None]
        for i, w in enumerate((d, dv)):
            x = r.standard_normal((n_pages, hk, page_size, w)).astype(np.float32)
            if fill is not None:
                x[:] = fill
            if dtype == "e4m3":
                codes, b = quantised(x.astype(np.float64) * np.exp2(r.integers(-3, 4, (n_pages, hk, page_size, 1))))
                self.pages.append(codes)
                self.scales[i] = b
            else:
                self.pages.append(to_storage(x, dtype)[0])

    def values(self, which):
        """The rows' values in f64, [n_pages, hk, page_size, width]."""
        if self.dtype != "e4m3":
            return from_storage(self.pages[which], self.dtype)
        return np.ldexp(e4m3_values(self.pages[which]), (self.scales[which].astype(int) - 127)[..., None])

    def rows(self, which, table_row, n):
        """The first n rows of a sequence, [hk, n, width] in f64."""
        ps = self.shape[1]
        v = self.values(which)[np.asarray(table_row[: -(-n // ps)], int)]
        return v.transpose(1, 0, 2, 3).reshape(self.shape[2], -1, v.shape[-1])[:, :n]

    def upload(self, be):
        """A PagedKVCache holding these pages."""
        from tensor_cuda.kv_cache import PagedKVCache
        n, ps, hk, d, dv = self.shape
        c = PagedKVCache(be, n, ps, hk, d, self.dtype, head_dim_v=dv)
        for p, a in zip(c.args[1:], self.arrays()):
            if a is not None and a.size:
                be.device.copy_h2d(p.value, a)
        be.device.stream_sync()
        return c

    def arrays(self):
        return [self.pages[0], self.pages[1], self.scales[0], self.scales[1]]

    def download(self, be, cache):
        """The device's pages, in the order of arrays()."""
        out = []
        for p, a in zip(cache.args[1:], self.arrays()):
            out.append(None if a is None else be.device.download(p.value, a.nbytes, a.dtype, a.shape))
        return out


def shuffled_table(lengths, page_size, n_pages, seed=0, wide=None):
    """i32 [B, wide] over pages in a shuffled order; -1 behind each sequence's pages."""
    need = [-(-n // page_size) for n in lengths]
    assert sum(need) <= n_pages
    order = np.random.default_rng(seed).permutation(n_pages)
    t = np.full((len(lengths), wide or max(1, max(need))), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    return t


def attention(q, k, v, scale):
    """softmax(scale q k^T) v of one sequence in f64, with the error bound of an f32 evaluation.

    q [H, D], k [Hk, n, D], v [Hk, n, Dv] -> (o [H, Dv], lse [H], bound of o, bound of lse).
    A dot product of D products summed in f32 in any order is off by at most D 2^-24 sum |q_i k_i|; the
    scale, the change to base 2 and the difference to the maximum round three times more, and exp2 is
    within 2 units (2^-22). So each weight is off by a factor within 1 + delta, the quotient of two sums of n
    such weights by 2 delta + 2 n 2^-24 of sum p |v|."""
    group = q.shape[0] // k.shape[0]
    n, D = k.shape[1], q.shape[1]
    os, zs, bo, bz = [], [], [], []
    for h in range(q.shape[0]):
        kk, vv = k[h // group], v[h // group]
        s = scale * (kk @ q[h])
        m = s.max()
        p = np.exp(s - m)
        z = p.sum()
        mag = scale * (np.abs(kk) @ np.abs(q[h]))
        delta = (D + 4) * 2.0 ** -24 * mag.max() + 2.0 ** -22
        spread = (p / z) @ np.abs(vv)
        os.append((p / z) @ vv)
        zs.append(m + np.log(z))
        bo.append((2 * delta + 2 * n * 2.0 ** -24) * spread)
        bz.append(delta + n * 2.0 ** -24 + 2.0 ** -22 * (1 + abs(m + np.log(z)) + abs(m)))
    return np.array(os), np.array(zs), np.array(bo), np.array(bz)

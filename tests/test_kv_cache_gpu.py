"""kv_append and kv_read on the B200 against a host cache: plain formats bit for bit, 8-bit codes and scale
bytes equal to the definition's (nearest even, least scale), reads equal to code * 2^e rounded once."""
import numpy as np
import pytest

from _helpers import NP_STORAGE
from _paged import HostCache, e4m3_values, from_storage, quantised, shuffled_table, to_storage

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    from tensor_cuda.backend import CudaBackend
    from tensor_cuda.runtime import Device
    return CudaBackend(Device.shared(0))


def up(be, arr, dtype):
    from tensor_cuda.backend import host
    return be.from_host_sync(host(dtype, arr.shape, arr))


def places(lengths, new, seed=0, padded=0):
    """Tokens (seq, pos) adding new[b] tokens at the end of each sequence, shuffled, some of them padding."""
    seq = np.repeat(np.arange(len(lengths)), new)
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(lengths, new)])
    order = np.random.default_rng(seed).permutation(len(seq))
    seq, pos = seq[order].astype(np.int32), pos[order].astype(np.int32)
    if padded:
        pos[-padded:] = -1 - np.arange(padded) % 3
    return seq, pos


CASES = [  # input, cache, page, hk, d, dv, lengths, new, padded
    ("bf16", "bf16", 16, 12, 64, 64, [1, 17, 64], [1, 1, 1], 0),
    ("f16", "f16", 24, 3, 80, 72, [50, 7, 100], [50, 7, 60], 5),
    ("f32", "f32", 1, 2, 128, 128, [9, 3], [4, 3], 1),
    ("f32", "f32", 5, 1, 33, 7, [23], [23], 0),
    ("f16", "f16", 16, 2, 5, 250, [40, 41], [3, 41], 2),
    ("bf16", "bf16", 128, 4, 256, 256, [300, 129], [300, 1], 0),
    ("bf16", "e4m3", 16, 8, 128, 128, [100, 33, 5], [100, 33, 5], 7),
    ("f32", "e4m3", 24, 5, 80, 72, [77, 48], [70, 48], 0),
    ("f16", "e4m3", 7, 3, 64, 64, [1, 2, 3], [1, 1, 1], 0),
    ("f32", "e4m3", 3, 2, 1, 9, [10], [10], 3),
    ("f16", "e4m3", 64, 1, 248, 256, [65], [65], 0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:6])))
def test_append_and_read_back(be, case):
    inp, fmt, ps, hk, d, dv, lengths, new, padded = case
    pages = sum(-(-n // ps) for n in lengths) + 2
    h = HostCache(pages, ps, hk, d, dv, fmt, seed=1)
    table = shuffled_table(lengths, ps, pages, seed=2)
    seq, pos = places(lengths, new, seed=3, padded=padded)
    r = np.random.default_rng(4)
    n = len(seq)
    dense = [to_storage(r.standard_normal((n, hk, w)) * np.exp2(r.integers(-20, 20, (n, hk, 1))) if inp != "f16" else
                        r.standard_normal((n, hk, w)), inp) for w in (d, dv)]
    c = h.upload(be)
    t_dev, p_dev, s_dev = up(be, table, "i32"), up(be, pos, "i32"), up(be, seq, "i32")
    be.kv_append(c, up(be, dense[0][0], inp), up(be, dense[1][0], inp), t_dev, p_dev, s_dev)
    got = h.download(be, c)
    there = pos >= 0
    page, off = table[seq[there], pos[there] // ps], pos[there] % ps
    for w in (0, 1):  # the definition, applied to the host's copy; every other byte stays as it was
        if fmt == "e4m3":
            codes, b = quantised(dense[w][1][there])
            h.pages[w][page, :, off] = codes
            h.scales[w][page, :, off] = b
        else:
            h.pages[w][page, :, off] = dense[w][0][there]
    for a, b in zip(got, h.arrays()):
        assert (a is None) == (b is None) and (a is None or np.array_equal(a, b))
    for dt in ("f32", "f16", "bf16"):
        k, v = be.kv_read(c, t_dev, p_dev, s_dev, dtype=dt)
        for w, x in ((0, k), (1, v)):
            a = be.read_sync(x)
            a = np.asarray(a.data).reshape(a.shape)
            want = np.zeros((n, hk, (d, dv)[w]))
            want[there] = h.values(w)[page, :, off]
            with np.errstate(over="ignore"):
                want = to_storage(want, dt)[0]
            assert np.array_equal(np.asarray(a).view(want.dtype), want), (dt, w)
    c.dispose()


def test_rows_without_numbers(be):
    """All zeros, NaN, infinities, the ends of the exponent range: the scale comes from the finite values,
    infinities saturate, NaN stays NaN."""
    rows = np.zeros((8, 1, 16), np.float32)
    rows[1, 0, 3] = np.nan
    rows[1, 0, 4] = 5.0
    rows[2, 0, :3] = [np.inf, -np.inf, 1.0]
    rows[3, 0, :] = np.inf
    rows[4, 0, :2] = [3.4e38, -1e30]
    rows[5, 0, :2] = [1e-45, 1e-38]
    rows[6, 0, :2] = [448.0, 448.00003]
    rows[7, 0, :3] = [1.75, -1.75, 2 ** -20]
    h = HostCache(1, 8, 1, 16, 16, "e4m3")
    c = h.upload(be)
    pos, seq = np.arange(8, dtype=np.int32), np.zeros(8, np.int32)
    args = up(be, np.zeros((1, 1), np.int32), "i32"), up(be, pos, "i32"), up(be, seq, "i32")
    x = up(be, rows, "f32")
    be.kv_append(c, x, x, *args)
    codes, b = quantised(rows.astype(np.float64))
    kp, vp, ks, vs = h.download(be, c)
    assert np.array_equal(kp, codes.transpose(1, 0, 2)[None]) and np.array_equal(kp, vp)
    assert np.array_equal(ks, b.T[None]) and np.array_equal(ks, vs)
    k, _ = be.kv_read(c, *args, dtype="f32")
    got = be.read_sync(k).data.reshape(8, 16)
    want = np.ldexp(e4m3_values(codes[:, 0]), (b.astype(int) - 127))
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(got[1, 3])
    with np.errstate(over="ignore"):
        assert np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)].astype(np.float32))
    # Appending what was read keeps the values. The bytes may change: 448.00003 needs the next scale, under
    # which it is stored as 224, and what is read, 448, then fits the scale before. Row 4 stays out: 3.4e38
    # = 1.9987 * 2^127 has the 8-bit value 2 * 2^127, which is no f32.
    ok = [0, 2, 3, 5, 6, 7]
    again = up(be, got[ok].reshape(-1, 1, 16).copy(), "f32")
    sel = up(be, pos[ok], "i32"), up(be, seq[ok], "i32")
    be.kv_append(c, again, again, args[0], *sel)
    k, _ = be.kv_read(c, args[0], *sel, dtype="f32")
    assert np.array_equal(be.read_sync(k).data.reshape(-1, 16), got[ok])


@pytest.mark.parametrize("fmt,h,hk,d", [("bf16", 4, 4, 64), ("e4m3", 6, 2, 80), ("bf16", 2, 1, 33)])
def test_packed_projection(be, fmt, h, hk, d):
    """K and V read in place from [T, (H + 2 Hk) D] are kv_append of the same slices."""
    T, ps = 11, 4
    qkv, exact = to_storage(np.random.default_rng(0).standard_normal((T, (h + 2 * hk) * d)), "bf16")
    k, v = (qkv[:, i * d:(i + hk) * d].reshape(T, hk, d).copy() for i in (h, h + hk))
    pos = up(be, np.arange(T, dtype=np.int32), "i32")
    seq = up(be, np.zeros(T, np.int32), "i32")
    table = up(be, np.array([[2, 0, 1]], np.int32), "i32")
    hosts = [HostCache(3, ps, hk, d, d, fmt, fill=0.0) for _ in range(2)]
    a, b = (x.upload(be) for x in hosts)
    be.kv_append_packed(a, up(be, qkv, "bf16"), table, pos, seq)
    be.kv_append(b, up(be, k, "bf16"), up(be, v, "bf16"), table, pos, seq)
    for x, y in zip(hosts[0].download(be, a), hosts[1].download(be, b)):
        assert (x is None and y is None) or np.array_equal(x, y)


def test_no_tokens_and_one_sequence_per_token(be):
    h = HostCache(4, 2, 2, 16, 16, "f32")
    c = h.upload(be)
    none = up(be, np.zeros(0, np.int32), "i32")
    table = up(be, np.array([[0], [3]], np.int32), "i32")
    empty = up(be, np.zeros((0, 2, 16), np.float32), "f32")
    be.kv_append(c, empty, empty, table, none)
    k, v = be.kv_read(c, table, none)
    assert k.shape == (0, 2, 16) and v.shape == (0, 2, 16)
    x = np.random.default_rng(1).standard_normal((2, 2, 16)).astype(np.float32)
    be.kv_append(c, up(be, x, "f32"), up(be, x, "f32"), table, up(be, np.array([1, 0], np.int32), "i32"))
    got = h.download(be, c)
    h.pages[0][0, :, 1], h.pages[0][3, :, 0] = x[0], x[1]
    h.pages[1][0, :, 1], h.pages[1][3, :, 0] = x[0], x[1]
    assert all(np.array_equal(a, b) for a, b in zip(got[:2], h.pages))


def test_places_outside_the_cache_are_left_out_and_reported(be):
    """A page, sequence or position outside the cache: nothing is written there, the next
    synchronisation raises once, and the device stays usable."""
    from tensor_cuda import _ffi as F
    h = HostCache(2, 4, 1, 16, 16, "f16")
    c = h.upload(be)
    x = up(be, np.ones((5, 1, 16), np.float16), "f16")
    table = up(be, np.array([[0, 7], [-5, 1]], np.int32), "i32")
    for seq, pos in (([0], [4]), ([1], [0]), ([2], [0]), ([-1], [1]), ([0], [8]), ([0], [2 ** 31 - 1])):
        n = len(seq)
        be.kv_append(c, be.external(x.ptr, (n, 1, 16), "f16"), be.external(x.ptr, (n, 1, 16), "f16"), table,
                     up_quietly(be, pos), up_quietly(be, seq))
        with pytest.raises(F.MpcError, match="outside the cache") as e:
            be.device.stream_sync()
        assert e.value.status == F.ERR_INVALID
        be.device.stream_sync()  # reported once
        out = be._alloc((n, 1, 16), "f32"), be._alloc((n, 1, 16), "f32")
        be.device.memset(out[0].ptr, 1, 64 * n)
        be.kv_read(c, table, up_quietly(be, pos), up_quietly(be, seq), dtype="f32", out=out)
        with pytest.raises(F.MpcError, match="outside the cache"):
            be.device.stream_sync()
        assert not be.read_sync(out[0]).data.any()
    assert all(np.array_equal(a, b) for a, b in zip(h.download(be, c)[:2], h.pages))
    assert be.device.status() == F.OK


def up_quietly(be, values):
    return up(be, np.asarray(values, np.int32), "i32")


def test_dtype_of_the_dense_rows_is_kept(be):
    assert NP_STORAGE["bf16"] is np.uint16
    h = HostCache(1, 4, 1, 8, 8, "bf16")
    c = h.upload(be)
    k, _ = be.kv_read(c, up_quietly(be, [[0]]), up_quietly(be, [2]))
    assert k.dtype == "bf16"
    assert np.array_equal(from_storage(be.read_sync(k).data.reshape(1, 1, 8), "bf16")[0], h.values(0)[0, :, 2])


class Appends:
    """kv_append of one token on a stream of one's choice, to a good or a bad place; pool memory that is only written."""

    def __init__(self, be):
        from tensor_cuda import _ffi as F
        self.be, self.F = be, F
        self.cache = HostCache(2, 4, 1, 16, 16, "f16").upload(be)
        self.x = up(be, np.ones((1, 1, 16), np.float16), "f16")
        self.table, self.zero = up_quietly(be, [[0, 7]]), up_quietly(be, [0])
        self.bad = up_quietly(be, [4])  # in page 7 of 2
        self.tokens = F.KvTokens(1, 1, 2, F.I64x2(16, 16), F.I64x2(16, 16), F.F16, 0)

    def call(self, stream, pos):
        import ctypes as C
        self.F.call("mpc_kv_append", self.be.device.handle, *self.cache.args, C.byref(self.tokens), C.c_void_p(self.x.ptr),
                    C.c_void_p(self.x.ptr), C.c_void_p(self.table.ptr), C.c_void_p(self.zero.ptr), C.c_void_p(pos.ptr),
                    C.c_void_p(stream))

    def reports(self, sync):
        try:
            sync()
        except self.F.MpcError as e:
            assert e.status == self.F.ERR_INVALID and "token 0" in str(e)
            return True
        return False


def test_every_bad_call_is_reported(be):
    """A call right behind a synchronisation that reported: its own report is not wiped by the clearing of the last."""
    a, dev = Appends(be), be.device
    s = dev.new_stream()
    for _ in range(300):
        for st in (None, s):
            a.call(st, a.bad)
            assert a.reports(lambda: dev.stream_sync(st))
    assert not a.reports(dev.sync)
    dev.destroy_stream(s)


def test_a_bad_place_is_reported_to_its_own_stream(be):
    """The synchronisation of a stream reports that stream's calls; the device's reports any, each once."""
    a, dev = Appends(be), be.device
    s, t = dev.new_stream(), dev.new_stream()
    of = lambda st: a.reports(lambda: dev.stream_sync(st))  # noqa: E731
    try:
        a.call(s, a.bad)
        a.call(t, a.zero)
        dev.stream_sync(t)
        assert not of(t) and not of(None) and of(s) and not of(s)
        a.call(None, a.bad)
        assert not of(s) and of(None) and not of(None)
        a.call(s, a.bad)
        a.call(t, a.bad)
        assert a.reports(dev.sync) and a.reports(dev.sync) and not a.reports(dev.sync) and not of(s) and not of(t)
        a.call(s, a.bad)
        a.call(t, a.bad)
        assert of(t) and a.reports(dev.sync) and not of(s)
    finally:
        dev.destroy_stream(s)
        dev.destroy_stream(t)


def test_bad_places_of_a_destroyed_stream_and_of_many_streams(be):
    """A stream destroyed before it was synchronised leaves its report to the device's synchronisation, not to a
    stream created later; more streams than the table of reports holds still report every one."""
    a, dev = Appends(be), be.device
    s = dev.new_stream()
    a.call(s, a.bad)
    dev.destroy_stream(s)
    later = [dev.new_stream() for _ in range(4)]
    for st in later:
        a.call(st, a.zero)
        assert not a.reports(lambda: dev.stream_sync(st))
        dev.destroy_stream(st)
    assert a.reports(dev.sync) and not a.reports(dev.sync)
    for _ in range(1200):  # places are handed on
        st = dev.new_stream()
        a.call(st, a.zero)
        dev.destroy_stream(st)
    many = [dev.new_stream() for _ in range(300)]
    for st in many:
        a.call(st, a.bad)
        assert a.reports(lambda: dev.stream_sync(st)) and not a.reports(lambda: dev.stream_sync(st))
    for st in many:
        dev.destroy_stream(st)
    assert not a.reports(dev.sync)


def test_a_captured_call_reports_to_the_next_synchronisation(be):
    """A graph may be launched into any stream: its reports go to whichever synchronisation comes next."""
    import torch
    a, dev = Appends(be), be.device
    st, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        a.call(st.cuda_stream, a.bad)
    other = dev.new_stream()
    for sync in (dev.sync, dev.stream_sync, lambda: dev.stream_sync(other)):
        g.replay()
        torch.cuda.synchronize()
        assert a.reports(sync) and not a.reports(dev.sync)
    dev.destroy_stream(other)

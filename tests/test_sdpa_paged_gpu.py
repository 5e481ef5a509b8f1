"""sdpa_paged on the B200 against softmax(scale q k^T) v in f64, per element within the bound of an f32
evaluation (tests/_paged.py) plus the rounding of the output and, on the tensor cores, of the weights."""
import math

import numpy as np
import pytest

from _paged import EPS, HostCache, attention, from_storage, shuffled_table, to_storage

pytestmark = pytest.mark.gpu

# Weights enter the tensor cores as two numbers of the type, the second the first's rounding error: each
# weight is off by at most (eps / 2)^2 of itself (f16 weights also by 2^-25 of the largest, which the
# slack for exp2 covers); f32 rows stay on the CUDA cores.
WEIGHT = {"f32": 0.0, "f16": 2.0 ** -21, "bf16": 2.0 ** -16, "e4m3": 2.0 ** -20}


@pytest.fixture(scope="module")
def be():
    from tensor_cuda.backend import CudaBackend
    from tensor_cuda.runtime import Device
    return CudaBackend(Device.shared(0))


def up(be, arr, dtype):
    from tensor_cuda.backend import host
    return be.from_host_sync(host(dtype, arr.shape, arr))


def check(be, h, q_dtype, cache, group, ps, hk, d, dv, lengths, seed=0, scale=None, host_cache=None, wide=None, q_mag=1.0):
    pages = sum(-(-n // ps) for n in lengths) + 1
    hc = host_cache or HostCache(pages, ps, hk, d, dv, cache, seed=seed)
    table = shuffled_table(lengths, ps, pages, seed=seed + 1, wide=wide)
    B = len(lengths)
    qs, q = to_storage(np.random.default_rng(seed + 2).standard_normal((B, h, d)) * q_mag, q_dtype)
    scale = 1 / math.sqrt(d) if scale is None else scale
    c = hc.upload(be)
    args = up(be, qs, q_dtype), c, up(be, table, "i32"), up(be, np.array(lengths, np.int32), "i32"), scale
    o, z = be.sdpa_paged(*args, lse=True)
    o2 = be.sdpa_paged(*args)
    got_raw, lse = be.read_sync(o), be.read_sync(z).data.reshape(B, h)
    assert np.array_equal(got_raw.data, be.read_sync(o2).data)  # the same bits again, with and without lse
    got = from_storage(got_raw.data.reshape(B, h, dv), q_dtype)
    for b, n in enumerate(lengths):
        if n == 0:
            assert not got[b].any() and np.all(np.isneginf(lse[b]))
            continue
        want, wz, bo, bz = attention(q[b], hc.rows(0, table[b], n), hc.rows(1, table[b], n), scale)
        spread = np.repeat(np.abs(hc.rows(1, table[b], n)).max(1), group, 0)
        tol = bo + (EPS[q_dtype] / 2) * np.abs(want) * 1.01 + 2 * WEIGHT[cache] * spread + 1e-30
        if q_dtype == "f16":
            tol = tol + 2.0 ** -25  # subnormal outputs
        off = np.abs(got[b] - want) / tol
        assert off.max() <= 1, (b, n, off.max())
        assert np.all(np.abs(lse[b] - wz) <= bz), (b, n, np.abs(lse[b] - wz).max(), bz.min())
    c.dispose()


CASES = [  # q, cache, h, hk, page, d, dv, lengths
    ("bf16", "bf16", 12, 12, 16, 64, 64, [1, 1024, 63, 64, 65, 0, 500]),
    ("f16", "f16", 8, 2, 16, 128, 128, [1, 2, 15, 16, 17, 31, 129, 700]),
    ("bf16", "bf16", 16, 2, 32, 128, 128, [1000, 3, 257]),
    ("f16", "f16", 16, 1, 64, 64, 64, [300, 0, 1]),
    ("bf16", "bf16", 48, 2, 8, 128, 128, [77, 200]),
    ("f16", "f16", 6, 2, 24, 80, 72, [100, 49, 24]),
    ("bf16", "bf16", 5, 5, 1, 96, 96, [33, 7]),
    ("bf16", "bf16", 4, 2, 128, 256, 256, [300, 129, 128]),
    ("f16", "f16", 20, 2, 16, 256, 64, [90, 5]),
    ("f16", "f16", 4, 4, 7, 32, 248, [50, 8]),
    ("bf16", "bf16", 3, 3, 5, 33, 5, [40, 6]),
    ("f16", "f16", 2, 1, 16, 8, 8, [300]),
    ("f32", "f32", 10, 5, 24, 80, 72, [3, 500, 1]),
    ("f32", "f32", 16, 2, 16, 128, 128, [130, 64]),
    ("f32", "f32", 4, 1, 16, 256, 256, [70]),
    ("f32", "f32", 3, 3, 3, 7, 9, [20, 0]),
    ("bf16", "e4m3", 32, 4, 16, 128, 128, [500, 1, 64, 1025]),
    ("f16", "e4m3", 12, 12, 16, 64, 64, [200, 31]),
    ("f32", "e4m3", 8, 2, 64, 128, 128, [400, 65]),
    ("bf16", "e4m3", 16, 1, 24, 80, 72, [99, 25]),
    ("f32", "e4m3", 2, 2, 16, 256, 256, [50]),
    ("bf16", "e4m3", 3, 1, 5, 20, 12, [31]),
    ("f16", "e4m3", 5, 1, 32, 248, 128, [130]),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:7])))
def test_against_the_definition(be, case):
    qd, cache, h, hk, ps, d, dv, lengths = case
    check(be, h, qd, cache, h // hk, ps, hk, d, dv, lengths)


@pytest.mark.parametrize("qd,cache,n,b", [("bf16", "bf16", 20000, 1), ("bf16", "e4m3", 33333, 1), ("f16", "f16", 5000, 3),
                                          ("f32", "f32", 9000, 1)])
def test_long_caches_split_and_joined(be, qd, cache, n, b):
    check(be, 8, qd, cache, 4, 16, 2, 64, 64, [n - 7 * i for i in range(b)])


def test_many_short_sequences(be):
    """More sequences than a block scans at once, empty ones among them."""
    check(be, 2, "bf16", "bf16", 1, 4, 2, 64, 64, [(i * 37) % 23 for i in range(400)])


@pytest.mark.parametrize("qd,cache", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "e4m3")])
def test_sharp_scores(be, qd, cache):
    """Scores far apart: the maximum moves along the cache and most weights vanish."""
    check(be, 8, qd, cache, 4, 16, 2, 64, 64, [700, 90], q_mag=6.0, seed=5)


def test_scale_bytes_far_apart(be):
    """8-bit rows whose scales span 2^40: the rows of small values still count where the large ones
    have no weight."""
    hc = HostCache(5, 16, 1, 64, 64, "e4m3", seed=7)
    r = np.random.default_rng(8)
    hc.scales[1][:] = r.integers(100, 141, hc.scales[1].shape)
    check(be, 4, "bf16", "e4m3", 4, 16, 1, 64, 64, [64], host_cache=hc, seed=7, q_mag=2.0)


@pytest.mark.parametrize("cache,qd", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("e4m3", "f16")])
def test_rows_behind_the_length_do_not_count(be, cache, qd):
    """NaN in every row behind a sequence's length, inside its last page and in other pages."""
    ps, lengths = 16, [5, 17, 40, 0]
    pages = sum(-(-n // ps) for n in lengths) + 1
    hc = HostCache(pages, ps, 2, 64, 64, cache, seed=3)
    table = shuffled_table(lengths, ps, pages, seed=4)
    live = np.zeros((pages, ps), bool)
    for b, n in enumerate(lengths):
        for p in range(n):
            live[table[b, p // ps], p % ps] = True
    nan = {"bf16": 0x7FC0, "e4m3": 127}.get(cache, np.nan)
    for w in (0, 1):
        hc.pages[w][np.broadcast_to(~live[:, None, :], hc.pages[w].shape[:3])] = nan
        if cache == "e4m3":
            hc.scales[w][np.broadcast_to(~live[:, None, :], hc.scales[w].shape)] = 255
    check(be, 4, qd, cache, 2, ps, 2, 64, 64, lengths, seed=3, host_cache=hc)


@pytest.mark.parametrize("cache", ["bf16", "f32", "e4m3"])
def test_not_a_number_in_a_live_row_shows(be, cache):
    qd = "bf16" if cache == "e4m3" else cache
    hc = HostCache(2, 16, 1, 64, 64, cache, seed=1)
    hc.pages[1][0, 0, 3, 10] = {"bf16": 0x7FC0, "e4m3": 127}.get(cache, np.nan)
    c = hc.upload(be)
    qs, _ = to_storage(np.random.default_rng(2).standard_normal((1, 2, 64)), qd)
    o = be.sdpa_paged(up(be, qs, qd), c, up(be, np.array([[0, 1]], np.int32), "i32"), up(be, np.array([20], np.int32), "i32"), 0.1)
    got = from_storage(be.read_sync(o).data.reshape(2, 64), qd)
    assert np.all(np.isnan(got[:, 10])) and not np.isnan(np.delete(got, 10, 1)).any()


def test_shared_pages_and_packed_queries(be):
    """Two sequences reading one prefix page; queries and output of a packed projection."""
    hk, g, d = 2, 3, 64
    hc = HostCache(3, 16, hk, d, d, "bf16", seed=1)
    c = hc.upload(be)
    table = np.array([[2, 0], [2, 1]], np.int32)
    lengths = [20, 31]
    qkv, exact = to_storage(np.random.default_rng(2).standard_normal((2, (hk * g + 2 * hk) * d)), "bf16")
    dev = up(be, qkv, "bf16"), c, up(be, table, "i32"), up(be, np.array(lengths, np.int32), "i32"), 0.125
    o = be.sdpa_paged_packed(*dev)
    assert o.shape == (2, hk * g * d)
    q = np.ascontiguousarray(qkv[:, : hk * g * d]).reshape(2, hk * g, d)
    o2 = be.sdpa_paged(up(be, q, "bf16"), *dev[1:])
    assert np.array_equal(be.read_sync(o).data, be.read_sync(o2).data)
    for b, n in enumerate(lengths):
        want, _, bo, _ = attention(from_storage(q, "bf16")[b], hc.rows(0, table[b], n), hc.rows(1, table[b], n), 0.125)
        got = from_storage(be.read_sync(o2).data.reshape(2, hk * g, d), "bf16")[b]
        assert np.all(np.abs(got - want) <= bo + 2.0 ** -8 * 1.01 * np.abs(want) + 2.0 ** -15 * 4)


@pytest.mark.parametrize("cache,qd", [("bf16", "bf16"), ("f32", "f32")])
def test_bad_pages_and_lengths_are_reported(be, cache, qd):
    """Pages outside the cache are left out, lengths are cut to the table; the next synchronisation says so."""
    from tensor_cuda import _ffi as F
    hc = HostCache(3, 16, 1, 64, 64, cache, seed=1)
    c = hc.upload(be)
    qs, q = to_storage(np.random.default_rng(2).standard_normal((1, 1, 64)), qd)

    def run(table, length):
        o = be._alloc((1, 1, 64), qd)
        be.sdpa_paged(up(be, qs, qd), c, up(be, np.array([table], np.int32), "i32"),
                      up(be, np.array([length], np.int32), "i32"), 0.125, out=o)
        with pytest.raises(F.MpcError, match="sequence 0") as e:
            be.device.stream_sync()
        assert e.value.status == F.ERR_INVALID
        be.device.stream_sync()
        return from_storage(be.read_sync(o).data.reshape(1, 64), qd)

    full = np.concatenate([hc.values(i)[[0, 2]].reshape(1, 1, 32, 64) for i in (0, 1)])
    want, _, bo, _ = attention(q[0], full[0], full[1], 0.125)
    tol = bo + EPS[qd] * np.abs(want) + 2.0 ** -14
    for bad in (3, -1, 2 ** 31 - 1):
        assert np.all(np.abs(run([0, bad, 2], 48) - want) <= tol)
    assert not run([3, 9], 20).any()
    assert not run([0, 2], -4).any()
    assert np.all(np.abs(run([0, 2], 1000) - want) <= tol)
    assert be.device.status() == F.OK


def test_workspace_of_the_caller_on_another_stream(be):
    """The C entry with a workspace and a stream of its own gives the same bits; one too small is refused."""
    import ctypes as C
    from tensor_cuda import _ffi as F
    dev = be.device
    hc = HostCache(80, 16, 2, 128, 128, "f16", seed=1)
    c = hc.upload(be)
    table = shuffled_table([1200], 16, 80)
    qs, _ = to_storage(np.random.default_rng(2).standard_normal((1, 8, 128)), "f16")
    q, t, n = up(be, qs, "f16"), up(be, table, "i32"), up(be, np.array([1200], np.int32), "i32")
    want = be.read_sync(be.sdpa_paged(q, c, t, n, 0.1)).data
    d = F.SdpaPagedDesc()
    d.b, d.h, d.max_pages, d.dtype, d.scale = 1, 8, table.shape[1], F.F16, 0.1
    d.q_stride[:] = d.o_stride[:] = (8 * 128, 128)
    need = C.c_size_t()
    F.call("mpc_sdpa_paged_workspace", dev.handle, c.args[0], C.byref(d), C.byref(need))
    ws, o = dev.alloc(need.value), dev.alloc(8 * 128 * 2)
    dev.memset(ws.ptr, 0, ws.nbytes)
    dev.stream_sync()
    s = dev.new_stream()

    def call(ws_ptr, nbytes):
        F.call("mpc_sdpa_paged", dev.handle, *c.args, C.byref(d), C.c_void_p(q.ptr), C.c_void_p(t.ptr), C.c_void_p(n.ptr),
               C.c_void_p(o.ptr), None, C.c_void_p(ws_ptr), nbytes, C.c_void_p(s))

    for args in ((ws.ptr, need.value), (ws.ptr, need.value), (None, 0)):  # the workspace is ready for the next call
        dev.memset(o.ptr, 255, o.nbytes, stream=s)
        call(*args)
        assert np.array_equal(dev.download(o.ptr, o.nbytes, np.float16, (8 * 128,), stream=s), want)
    for args in ((ws.ptr, need.value - 1), (ws.ptr + 8, need.value)):
        with pytest.raises(F.MpcError, match="workspace"):
            call(*args)
    dev.destroy_stream(s)


@pytest.mark.parametrize("qd", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [2, 6, 40])
def test_cancelling_rows_show_the_weights(be, qd, n):
    """8-bit V rows in pairs (v, -v) under nearly equal weights: the outputs are differences of weights, so that
    an error of a weight shows against the output's own rounding (a weight of one f16 number would be off by up
    to 2^-11 of itself; the bound here is about 2^-17 of the rows)."""
    hc = HostCache(4, 16, 2, 64, 64, "e4m3", seed=n)
    hc.pages[1][:, :, 1::2] = hc.pages[1][:, :, ::2] ^ 0x80
    hc.scales[1][:, :, 1::2] = hc.scales[1][:, :, ::2]
    check(be, 16, qd, "e4m3", 8, 16, 2, 64, 64, [n], seed=n, scale=1.0, host_cache=hc, q_mag=2.0 ** -10)

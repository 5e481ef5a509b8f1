"""The paged cache, its attention and sampling without a GPU: struct layouts, the refusals of the host side
and of the C entries, the block table's bookkeeping, and the tests' own 8-bit arithmetic."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from _paged import _POSITIVE, e4m3_codes, e4m3_values, quantised, scale_bytes

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class NoDevice:
    """A device whose handle is null: every C call on it is refused, nothing runs."""
    handle = None

    def alloc(self, nbytes):
        raise AssertionError("a refused call allocated memory")


@pytest.fixture()
def be():
    from tensor_cuda.backend import CudaBackend
    return CudaBackend(NoDevice())


def cache_of(be, dtype="bf16", hk=2, d=64, dv=None, ps=16):
    from tensor_cuda.kv_cache import PagedKVCache
    return PagedKVCache(be, 4, ps, hk, d, dtype, head_dim_v=dv, pools=(16, 16, 16, 16))


def t(be, shape, dtype="bf16"):
    return be.external(16, shape, dtype)


def test_struct_layouts_match_the_header(tmp_path):
    from tensor_cuda import _ffi as F
    names = {"mpc_kv_desc": F.KvDesc, "mpc_kv_tokens": F.KvTokens, "mpc_sdpa_paged_desc": F.SdpaPagedDesc,
             "mpc_sample_desc": F.SampleDesc}
    lines = []
    for n, s in names.items():
        lines.append(f'printf("%zu", sizeof({n}));')
        lines += [f'printf(" %zu", offsetof({n}, {f[0]}));' for f in s._fields_] + ['printf("\\n");']
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mathplus_cuda.h"\nint main(void) {\n' + "\n".join(lines)
                   + '\nprintf("%d\\n", (int)MPC_E4M3);\nreturn 0;\n}\n')
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "t")], check=True)
    out = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.splitlines()
    for line, s in zip(out, names.values()):
        assert [int(v) for v in line.split()] == [C.sizeof(s)] + [getattr(s, f[0]).offset for f in s._fields_]
    assert int(out[-1]) == F.E4M3


def test_the_c_entries_refuse_a_null_device():
    from tensor_cuda import _ffi as F
    lib = F.load()
    for name in ("mpc_kv_append", "mpc_kv_read", "mpc_sdpa_paged", "mpc_sdpa_paged_workspace", "mpc_sample"):
        zeros = [0 if a in (C.c_size_t, C.c_int32) else None for a in F.SIGNATURES[name]]
        assert getattr(lib, name)(*zeros) == F.ERR_INVALID
        assert "null device" in F.last_error()


def test_append_and_read_refusals(be):
    c = cache_of(be)
    table, pos = t(be, (3, 4), "i32"), t(be, (3,), "i32")
    k = t(be, (3, 2, 64))
    bad = [
        (ValueError, dict(k=t(be, (3, 1, 64)))), (ValueError, dict(v=t(be, (2, 2, 64)))),
        (ValueError, dict(k=t(be, (3, 2, 32)))), (ValueError, dict(k=t(be, (6, 64)))),
        (TypeError, dict(v=t(be, (3, 2, 64), "f16"))), (TypeError, dict(k=t(be, (3, 2, 64), "f16"), v=t(be, (3, 2, 64), "f16"))),
        (TypeError, dict(table=t(be, (3, 4), "f32"))), (TypeError, dict(table=t(be, (12,), "i32"))),
        (TypeError, dict(pos=t(be, (3,), "f32"))), (ValueError, dict(pos=t(be, (2,), "i32"))),
        (ValueError, dict(seq=t(be, (4,), "i32"))), (ValueError, dict(table=t(be, (2, 4), "i32"))),
    ]
    for err, change in bad:
        args = dict(k=k, v=k, table=table, pos=pos, seq=None)
        args.update(change)
        with pytest.raises(err, match="tensor-cuda"):
            be.kv_append(c, **args)
    with pytest.raises(TypeError, match="float"):
        be.kv_read(c, table, pos, dtype="i32")
    with pytest.raises(ValueError, match="out is"):
        be.kv_read(c, table, pos, out=(k, t(be, (3, 2, 65))))
    with pytest.raises(ValueError, match="qkv"):
        be.kv_append_packed(c, t(be, (3, 5 * 64)), table, pos)  # one query head over two K/V heads
    with pytest.raises(ValueError, match="qkv"):
        be.kv_append_packed(cache_of(be, dv=32), t(be, (3, 6 * 64)), table, pos)
    k.disposed = True
    with pytest.raises(RuntimeError, match="dispose"):
        be.kv_append(c, k, k, table, pos)
    c.dispose()
    with pytest.raises(RuntimeError, match="cache used after dispose"):
        be.kv_read(c, table, pos)


def test_tensors_and_caches_of_another_device_are_refused(be):
    from tensor_cuda.backend import CudaBackend
    other = CudaBackend(NoDevice())
    c = cache_of(be)
    table, n = t(be, (2, 4), "i32"), t(be, (2,), "i32")
    with pytest.raises(ValueError, match="another device"):
        be.sdpa_paged(t(other, (2, 2, 64)), c, table, n, 1.0)
    with pytest.raises(ValueError, match="another device"):
        be.sdpa_paged(t(be, (2, 2, 64)), cache_of(other), table, n, 1.0)
    with pytest.raises(ValueError, match="another device"):
        be.kv_read(c, t(other, (2, 4), "i32"), n)
    with pytest.raises(ValueError, match="another device"):
        be.sample(t(be, (2, 9), "f32"), t(other, (2,), "f32"))


def test_attention_refusals(be):
    c = cache_of(be)
    table, n, q = t(be, (2, 4), "i32"), t(be, (2,), "i32"), t(be, (2, 4, 64))
    for err, a in ((ValueError, (t(be, (2, 4, 32)), c, table, n)), (ValueError, (t(be, (2, 3, 64)), c, table, n)),
                   (TypeError, (t(be, (2, 4, 64), "f16"), c, table, n)), (ValueError, (q, c, t(be, (3, 4), "i32"), n)),
                   (TypeError, (q, c, table, t(be, (2,), "f32"))), (ValueError, (q, c, table, t(be, (3,), "i32")))):
        with pytest.raises(err, match="tensor-cuda"):
            be.sdpa_paged(*a, 1.0)
    with pytest.raises(ValueError, match="out is"):
        be.sdpa_paged(q, c, table, n, 1.0, out=t(be, (2, 4, 64), "f32"))
    with pytest.raises(ValueError, match="out is"):
        be.sdpa_paged(q, c, table, n, 1.0, lse=True, out=(q, t(be, (2, 2), "f32")))


def test_sampling_refusals(be):
    x, u = t(be, (2, 9), "f32"), t(be, (2,), "f32")
    for err, a in ((ValueError, (t(be, (9,), "f32"), u)), (ValueError, (t(be, (2, 0), "f32"), u)),
                   (TypeError, (t(be, (2, 9), "i32"), u)), (TypeError, (x, t(be, (3,), "f32"))), (TypeError, (x, 0.5)),
                   (TypeError, (x, u, t(be, (2,), "f16"))), (TypeError, (x, u, 1.0, t(be, (2,), "f32")))):
        with pytest.raises(err, match="tensor-cuda"):
            be.sample(*a)
    with pytest.raises(ValueError, match="out is"):
        be.sample(x, u, out=u)


def test_cache_refusals(be):
    from tensor_cuda.kv_cache import PagedKVCache
    for err, a in ((TypeError, (4, 16, 2, 64, "i32")), (ValueError, (4, 0, 2, 64)), (ValueError, (-1, 16, 2, 64)),
                   (NotImplementedError, (4, 16, 2, 257))):
        with pytest.raises(err, match="tensor-cuda"):
            PagedKVCache(be, *a)
    with pytest.raises(ValueError, match="pools"):
        PagedKVCache(be, 4, 16, 2, 64, "e4m3", pools=(16, 16, None, None))


def test_block_table(be):
    from tensor_cuda.kv_cache import BlockTable
    bt = BlockTable(be, 3, 10, 16, max_pages=6)
    bt.reserve([1, 16, 33])
    assert bt.free_pages == 5
    used = bt.host[bt.host >= 0]
    assert len(set(used.tolist())) == 5 and [(bt.host[b] >= 0).sum() for b in range(3)] == [1, 1, 3]
    before = bt.host.copy()
    bt.reserve([16, 2, 48])  # enough already: pages stay
    assert np.array_equal(bt.host, before)
    bt.reserve([17, 16, 33])
    assert bt.free_pages == 4 and bt.host[0, 0] == before[0, 0] and bt.host[0, 1] >= 0
    kept = bt.host.copy()
    with pytest.raises(ValueError, match="needs 7 pages"):
        bt.reserve([0, 16 * 7, 0])
    with pytest.raises(MemoryError, match="4 of 10 free"):
        bt.reserve([96, 96, 96])
    with pytest.raises(ValueError, match="lengths"):
        bt.reserve([1, 2])
    assert np.array_equal(bt.host, kept) and bt.free_pages == 4
    bt.release(2)
    assert bt.free_pages == 7 and not (bt.host[2] >= 0).any()
    bt.release(2)
    bt.reserve([17, 16, 96])
    assert bt.free_pages == 1 and len(set(bt.host[bt.host >= 0].tolist())) == 9


def test_eight_bit_arithmetic_of_the_tests():
    """The host's rounding is to the nearest of the 8-bit numbers, at their midpoints to the even code."""
    assert _POSITIVE[-1] == 448 and _POSITIVE[1] == 2.0 ** -9 and np.all(np.diff(_POSITIVE) > 0)
    mid = (_POSITIVE[1:] + _POSITIVE[:-1]) / 2
    even = np.arange(126) + np.arange(126) % 2
    assert np.array_equal(e4m3_codes(mid), even)
    assert np.array_equal(e4m3_codes(-mid), even + 128)
    assert np.array_equal(e4m3_codes(np.nextafter(mid, 1e9)), np.arange(1, 127))
    assert np.array_equal(e4m3_codes(np.nextafter(mid, 0)), np.arange(126))
    assert np.array_equal(e4m3_codes([np.inf, 1e9, -np.inf]), [126, 126, 254]) and np.isnan(e4m3_values(e4m3_codes(np.nan)))
    assert scale_bytes(np.array([[448.0], [449.0], [224.0], [225.0], [0.0]])).tolist() == [127, 128, 126, 127, 1]
    x = np.random.default_rng(0).standard_normal((100, 64)) * 1e3
    codes, b = quantised(x)
    back = np.ldexp(e4m3_values(codes), (b.astype(int) - 127)[:, None])
    assert np.all(np.abs(back - x) <= np.maximum(2.0 ** -4 * np.abs(x), np.ldexp(1.0, b.astype(int) - 137)[:, None]))


def test_block_table_uploads_again_where_its_tensor_is_gone():
    """A table first uploaded inside a scope is released with it; the next use uploads it anew."""
    from tensor_cuda.backend import CudaBackend
    from tensor_cuda.kv_cache import BlockTable

    class Uploads(CudaBackend):
        def from_host_sync(self, h):
            return self.external(16, h.shape, h.dtype)

    be = Uploads(NoDevice())
    bt = BlockTable(be, 2, 8, 16, max_pages=4)
    bt.reserve([5, 20])
    inside = []
    be.scope(lambda: inside.append(bt.device))
    assert inside[0].disposed
    again = bt.device
    assert not again.disposed and again is not inside[0] and bt.device is again
    bt.dispose()

"""Append, attention and sampling captured together into a CUDA graph and replayed: positions, lengths and inputs
are read on the device, so one graph serves every step; two graphs with a workspace each run side by side."""
import ctypes as C

import numpy as np
import pytest

from _paged import HostCache, attention, from_storage, to_storage

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    from tensor_cuda.backend import CudaBackend
    from tensor_cuda.runtime import Device
    return CudaBackend(Device.shared(0))


class Step:
    """One decode step's buffers (torch memory) and its three C calls on a stream."""

    def __init__(self, be, seed, B=3, hk=2, g=2, d=64, ps=8, pages=40):
        import torch
        from tensor_cuda import _ffi as F
        self.F, self.be, self.torch = F, be, torch
        self.B, self.hk, self.h, self.d, self.ps = B, hk, hk * g, d, ps
        self.host = HostCache(pages, ps, hk, d, d, "bf16", seed=seed)
        self.cache = self.host.upload(be)
        r = np.random.default_rng(seed)
        self.table = r.permutation(pages)[: B * 12].reshape(B, 12).astype(np.int32)
        self.width = (self.h + 2 * hk) * d
        i32 = dict(device="cuda", dtype=torch.int32)
        self.t_table = torch.from_numpy(self.table).cuda()
        self.t_pos, self.t_len = torch.zeros(B, **i32), torch.zeros(B, **i32)
        self.t_qkv = torch.zeros((B, self.width), device="cuda", dtype=torch.bfloat16)
        self.t_out = torch.zeros((B, self.h, d), device="cuda", dtype=torch.bfloat16)
        self.t_u = torch.zeros(B, device="cuda")
        self.t_tok = torch.zeros(B, **i32)
        self.tokens = F.KvTokens(B, B, 12, F.I64x2(self.width, d), F.I64x2(self.width, d), F.BF16, 0)
        self.desc = F.SdpaPagedDesc(B, self.h, 12, F.I64x2(self.width, d), F.I64x2(self.h * d, d), F.BF16, 0.125)
        self.sdesc = F.SampleDesc(B, self.h * d, self.h * d, F.BF16, 40, 0.7, 0.9, 0.0, 0)
        need = C.c_size_t()
        F.call("mpc_sdpa_paged_workspace", be.device.handle, self.cache.args[0], C.byref(self.desc), C.byref(need))
        self.ws = torch.zeros(need.value, device="cuda", dtype=torch.uint8)

    def calls(self, stream):
        F, dev = self.F, self.be.device.handle
        base = self.t_qkv.data_ptr()
        k = base + self.h * self.d * 2
        F.call("mpc_kv_append", dev, *self.cache.args, C.byref(self.tokens), k, k + self.hk * self.d * 2,
               self.t_table.data_ptr(), None, self.t_pos.data_ptr(), stream)
        F.call("mpc_sdpa_paged", dev, *self.cache.args, C.byref(self.desc), base, self.t_table.data_ptr(),
               self.t_len.data_ptr(), self.t_out.data_ptr(), None, self.ws.data_ptr(), self.ws.numel(), stream)
        F.call("mpc_sample", dev, C.byref(self.sdesc), self.t_out.data_ptr(), self.t_u.data_ptr(), None, None, None, None,
               self.t_tok.data_ptr(), None, None, stream)

    def set(self, lengths, seed):
        """Inputs of a step after which the sequences have these lengths (0: the row is padding)."""
        torch = self.torch
        r = np.random.default_rng(seed)
        bits, self.qkv = to_storage(r.standard_normal((self.B, self.width)), "bf16")
        self.lengths = lengths
        self.t_qkv.copy_(torch.from_numpy(bits.view(np.int16)).view(torch.bfloat16))
        self.t_len.copy_(torch.tensor(lengths, dtype=torch.int32))
        self.t_pos.copy_(torch.tensor(lengths, dtype=torch.int32) - 1)
        self.t_u.copy_(torch.from_numpy(r.random(self.B).astype(np.float32)))
        for b, n in enumerate(lengths):
            if n:
                page, off = self.table[b, (n - 1) // self.ps], (n - 1) % self.ps
                for w in (0, 1):
                    at = (self.h + w * self.hk) * self.d
                    self.host.pages[w][page, :, off] = bits[b, at:at + self.hk * self.d].reshape(self.hk, self.d)

    def check(self):
        got = self.t_out.float().cpu().numpy().astype(np.float64)
        for b, n in enumerate(self.lengths):
            if n == 0:
                assert not got[b].any()
                continue
            q = self.qkv[b, : self.h * self.d].reshape(self.h, self.d)
            k, v = (self.host.rows(w, self.table[b], n) for w in (0, 1))
            want, _, bo, _ = attention(q, k, v, 0.125)
            assert np.all(np.abs(got[b] - want) <= bo + 2.0 ** -8 * 1.01 * np.abs(want) + 2.0 ** -15 * np.abs(v).max()), b
        eager = self.be.sample(self.be.external(self.t_out.data_ptr(), (self.B, self.h * self.d), "bf16"),
                               self.be.external(self.t_u.data_ptr(), (self.B,), "f32"), 0.7, 40, 0.9)
        assert np.array_equal(self.be.read_sync(eager).data, self.t_tok.cpu().numpy())


def test_one_graph_serves_every_step(be):
    import torch
    s = Step(be, 1)
    st = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        s.calls(st.cuda_stream)
    for i, lengths in enumerate(([1, 40, 96], [2, 41, 0], [3, 0, 7], [0, 0, 0], [96, 95, 64])):
        s.set(lengths, 10 + i)
        torch.cuda.synchronize()
        g.replay()
        g.replay()  # the same step again: the same places, the same answer
        torch.cuda.synchronize()
        s.check()
    be.device.sync()


def test_two_graphs_side_by_side(be):
    import torch
    steps = [Step(be, 2), Step(be, 3)]
    streams = [torch.cuda.Stream() for _ in steps]
    graphs = []
    torch.cuda.synchronize()
    for s, st in zip(steps, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            for _ in range(5):
                s.calls(st.cuda_stream)
        graphs.append(g)
    for i in range(3):
        for s in steps:
            s.set([5 + i, 90 - i, 33], 20 + i)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for s in steps:
            s.check()
    be.device.sync()


def test_a_captured_call_needs_a_workspace(be):
    """Without one the call is refused before it allocates; the capture goes on."""
    import torch
    from tensor_cuda import _ffi as F
    s = Step(be, 4)
    s.set([4, 5, 6], 1)
    st = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        with pytest.raises(F.MpcError, match="workspace"):
            F.call("mpc_sdpa_paged", be.device.handle, *s.cache.args, C.byref(s.desc), s.t_qkv.data_ptr(),
                   s.t_table.data_ptr(), s.t_len.data_ptr(), s.t_out.data_ptr(), None, None, 0, st.cuda_stream)
        s.calls(st.cuda_stream)
    g.replay()
    torch.cuda.synchronize()
    s.check()


def test_misaligned_pages_take_the_other_path(be):
    """Pages at an odd 2-byte address, a workspace sized for either path."""
    import torch
    from tensor_cuda import _ffi as F
    from tensor_cuda.kv_cache import PagedKVCache
    hc = HostCache(4, 16, 2, 64, 64, "f16", seed=1)
    bufs = [torch.zeros(a.size + 8, device="cuda", dtype=torch.float16) for a in hc.pages]
    for t, a in zip(bufs, hc.pages):
        t[1:1 + a.size].copy_(torch.from_numpy(a.reshape(-1)))
    c = PagedKVCache(be, 4, 16, 2, 64, "f16", pools=(bufs[0].data_ptr() + 2, bufs[1].data_ptr() + 2, None, None))
    r = np.random.default_rng(0)
    qs, q = to_storage(r.standard_normal((1, 4, 64)), "f16")
    tq = torch.from_numpy(qs).cuda()
    table, lens = torch.tensor([[2, 0, 3]], dtype=torch.int32, device="cuda"), torch.tensor([40], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    o = be.sdpa_paged(be.external(tq.data_ptr(), (1, 4, 64), "f16"), c, be.external(table.data_ptr(), (1, 3), "i32"),
                      be.external(lens.data_ptr(), (1,), "i32"), 0.125)
    got = from_storage(be.read_sync(o).data.reshape(4, 64), "f16")
    want, _, bo, _ = attention(q[0], hc.rows(0, [2, 0, 3], 40), hc.rows(1, [2, 0, 3], 40), 0.125)
    assert np.all(np.abs(got - want) <= bo + 2.0 ** -11 * 1.01 * np.abs(want) + 2.0 ** -20)
    k, v = be.kv_read(c, be.external(table.data_ptr(), (1, 3), "i32"),
                      be.from_host_sync(__import__("tensor_cuda.backend", fromlist=["host"]).host("i32", (1,), np.array([39], np.int32))))
    assert np.array_equal(from_storage(be.read_sync(k).data.reshape(2, 64), "f16"), hc.rows(0, [2, 0, 3], 40)[:, 39])

"""A GPT-2-small-shaped forward pass on the device, composed from the Backend ops of the GEMM /
attention path.

The block is the reference's pre-norm transformer layer (``TransformerEncoderLayer.forward`` with
``normFirst``, packages/tensor-autograd/src/transformer.ts:320-333: ``x = x + sa(norm1(x))``,
``x = x + ff(norm2(x))``, exact-erf GELU) with causal self-attention laid out like its
``MultiheadAttention`` (transformer.ts:173-242: packed ``in_proj_weight [3E, E]``, heads split as
``[N, L, H, D] -> [N, H, L, D]``, ``out_proj`` on the merged heads). GPT-2's token + position
embeddings lead in and a final LayerNorm and the tied LM head (``linear`` with the token table)
lead out.

Every step is one device op: ``embedding``, ``add``, ``layerNorm``, ``linear`` (bias, GELU for the
first MLP projection and the residual adds in the GEMM's epilogue) and ``sdpa_packed`` (causal
attention reading Q / K / V straight from the packed in-projection and writing the heads merged). Activations and weight matrices are bf16; biases and LayerNorm
parameters f32; every GEMM accumulates in f32.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import numpy as np

from . import _ffi as F
from .backend import CudaBackend, CudaTensor, host
from .kv_cache import BlockTable, PagedKVCache


@dataclass(frozen=True)
class GPT2Config:
    n_layer: int = 12
    d_model: int = 768
    n_head: int = 12
    d_ff: int = 3072
    vocab: int = 50257
    n_ctx: int = 1024
    eps: float = 1e-5

    @property
    def head_dim(self) -> int:
        return self.d_model // self.n_head

    def forward_flop(self, batch: int, seq: int) -> float:
        """Dense FLOP of one forward: the four linears per layer, causal attention (half of
        4*L^2*D per head) and the LM head."""
        d, f = self.d_model, self.d_ff
        per_token = self.n_layer * 2 * (d * 3 * d + d * d + 2 * d * f) + 2 * d * self.vocab
        attn = self.n_layer * 0.5 * 4 * seq * seq * d  # per sequence, all heads
        return batch * (seq * per_token + attn)


def _bf16_bits(x: np.ndarray) -> np.ndarray:
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def random_weights(cfg: GPT2Config, seed: int = 0, std: float = 0.02) -> dict:
    """Host weights: matrices ~ N(0, std) rounded to bf16 (uint16 bits), biases ~ N(0, std) and
    LayerNorm weight 1 / bias 0 in f32. Keys follow GPT-2's parameter names."""
    rng = np.random.default_rng(seed)
    d, f = cfg.d_model, cfg.d_ff
    mat = lambda *shape: _bf16_bits(rng.standard_normal(shape, dtype=np.float32) * std)
    vec = lambda n: (rng.standard_normal(n, dtype=np.float32) * std).astype(np.float32)
    w = {"wte": mat(cfg.vocab, d), "wpe": mat(cfg.n_ctx, d),
         "ln_f.weight": np.ones(d, np.float32), "ln_f.bias": np.zeros(d, np.float32)}
    for i in range(cfg.n_layer):
        p = f"h.{i}."
        w[p + "ln_1.weight"] = np.ones(d, np.float32)
        w[p + "ln_1.bias"] = np.zeros(d, np.float32)
        w[p + "attn.in_proj_weight"] = mat(3 * d, d)
        w[p + "attn.in_proj_bias"] = vec(3 * d)
        w[p + "attn.out_proj.weight"] = mat(d, d)
        w[p + "attn.out_proj.bias"] = vec(d)
        w[p + "ln_2.weight"] = np.ones(d, np.float32)
        w[p + "ln_2.bias"] = np.zeros(d, np.float32)
        w[p + "mlp.fc.weight"] = mat(f, d)
        w[p + "mlp.fc.bias"] = vec(f)
        w[p + "mlp.proj.weight"] = mat(d, f)
        w[p + "mlp.proj.bias"] = vec(d)
    return w


class GPT2:
    """The model's weights resident on one device and its forward pass."""

    def __init__(self, backend: CudaBackend, cfg: GPT2Config, weights: dict):
        """``weights``: host arrays (uint16 = bf16 bits, else f32), uploaded here, or device
        tensors (``CudaTensor``, e.g. from ``safetensors.gpt2_device_weights``), taken as they are."""
        self.backend, self.cfg = backend, cfg
        self.w: dict[str, CudaTensor] = {}
        for name, arr in weights.items():
            if isinstance(arr, CudaTensor):
                self.w[name] = arr
                continue
            dtype = "bf16" if arr.dtype == np.uint16 else "f32"
            self.w[name] = backend.from_host_sync(host(dtype, arr.shape, arr))
        self._pos: dict[int, CudaTensor] = {}

    @classmethod
    def from_safetensors(cls, backend: CudaBackend, cfg: GPT2Config, source) -> "GPT2":
        """A Hugging Face GPT-2 checkpoint (a ``.safetensors`` path or its bytes) on the device."""
        from .safetensors import gpt2_device_weights
        return cls(backend, cfg, gpt2_device_weights(source, backend, cfg.n_layer))

    def _positions(self, seq: int) -> CudaTensor:
        if seq not in self._pos:
            self._pos[seq] = self.backend.from_host_sync(host("i32", (seq,), np.arange(seq, dtype=np.int32)))
        return self._pos[seq]

    def forward(self, ids: CudaTensor, stop_after: int | None = None) -> CudaTensor:
        """ids i32 [B, L] -> logits bf16 [B, L, vocab]; with ``stop_after`` = n, the residual stream
        bf16 [B, L, d_model] after the first n blocks instead (no final LayerNorm or LM head)."""
        be, cfg, w = self.backend, self.cfg, self.w
        B, L = ids.shape
        if L > cfg.n_ctx:
            raise ValueError(f"GPT2: sequence of {L} tokens is longer than the context ({cfg.n_ctx})")
        if stop_after is not None and not 0 <= stop_after <= cfg.n_layer:
            raise ValueError(f"GPT2: stop_after={stop_after} outside 0..{cfg.n_layer}")
        D, H, Dh = cfg.d_model, cfg.n_head, cfg.head_dim
        tok = be.embedding(w["wte"], ids)                      # [B, L, D]
        pos = be.embedding(w["wpe"], self._positions(L))      # [L, D]
        s = be.add(tok, pos)
        x = be.reshape(s, (B * L, D))
        for t in (tok, pos, s):
            be.dispose(t)
        for i in range(cfg.n_layer if stop_after is None else stop_after):
            p = f"h.{i}."
            x = self._block(x, p, B, L, D, H, Dh)
        if stop_after is not None:
            out = be.reshape(x, (B, L, D))
            be.dispose(x)
            return out
        h = be.layerNorm(x, w["ln_f.weight"], w["ln_f.bias"], cfg.eps)
        be.dispose(x)
        logits = be.linear(h, w["wte"])                        # tied LM head: x . wte^T
        out = be.reshape(logits, (B, L, cfg.vocab))
        be.dispose(logits)
        be.dispose(h)
        return out

    def _block(self, x: CudaTensor, p: str, B: int, L: int, D: int, H: int, Dh: int, attend=None) -> CudaTensor:
        """One block over x [B*L, D]; ``attend(qkv)`` replaces the causal self-attention over the L tokens
        (a session's, over its cache)."""
        be, w, eps = self.backend, self.w, self.cfg.eps
        tmp = []
        h = be.layerNorm(x, w[p + "ln_1.weight"], w[p + "ln_1.bias"], eps)
        qkv = be.linear(h, w[p + "attn.in_proj_weight"], w[p + "attn.in_proj_bias"])      # [B*L, 3D]
        qkv3 = be.reshape(qkv, (B, L, 3 * D))                                              # [B, L, 3, H, Dh]
        a = be.sdpa_packed(qkv3, H, 1.0 / math.sqrt(Dh), causal=True) if attend is None else attend(qkv3)  # [B, L, H*Dh]
        merged = be.reshape(a, (B * L, D))
        o = be.linear(merged, w[p + "attn.out_proj.weight"], w[p + "attn.out_proj.bias"])
        x1 = be.add(x, o)
        tmp += [h, qkv, qkv3, a, merged, o]
        h2 = be.layerNorm(x1, w[p + "ln_2.weight"], w[p + "ln_2.bias"], eps)
        f = be.linear(h2, w[p + "mlp.fc.weight"], w[p + "mlp.fc.bias"], activation="gelu")  # [B*L, d_ff]
        g = be.linear(f, w[p + "mlp.proj.weight"], w[p + "mlp.proj.bias"])
        x2 = be.add(x1, g)
        tmp += [h2, f, g, x1, x]
        for t in tmp:
            be.dispose(t)
        return x2

    def session(self, n_seq: int, n_pages: int | None = None, page_size: int = 16, cache_dtype: str = "bf16") -> "GPT2Session":
        """A serving session of ``n_seq`` sequences (see ``GPT2Session``)."""
        return GPT2Session(self, n_seq, n_pages, page_size, cache_dtype)


class GPT2Session:
    """Sequences answered token by token: the model's K and V of every token seen are kept in paged caches
    (one per layer, one block table), so a step computes its new tokens only.

    ``step(ids, counts)`` takes the next tokens of every sequence and returns the logits that follow the last
    of each. Its attention is causal ``sdpa_packed`` for the sequences' first tokens, ``sdpa_paged`` for one new
    token each, and ``sdpa`` over the cache read back (``kv_read``) for several more. ``generate`` draws tokens
    with ``CudaBackend.sample``. ``cache_dtype="e4m3"`` holds the cache in 8 bits."""

    def __init__(self, model: GPT2, n_seq: int, n_pages: int | None = None, page_size: int = 16, cache_dtype: str = "bf16"):
        if n_seq <= 0:
            raise ValueError(f"GPT2Session: {n_seq} sequences")
        if cache_dtype not in ("bf16", "e4m3"):
            raise TypeError(f"GPT2Session: a cache of {cache_dtype} (bf16, as the activations, or e4m3)")
        self.model, self.n_seq = model, n_seq
        cfg, be = model.cfg, model.backend
        per_seq = -(-cfg.n_ctx // page_size)
        n_pages = n_seq * per_seq if n_pages is None else n_pages
        self.table = BlockTable(be, n_seq, n_pages, page_size, max_pages=per_seq)
        self.caches = [PagedKVCache(be, n_pages, page_size, cfg.n_head, cfg.head_dim, cache_dtype) for _ in range(cfg.n_layer)]
        self.lengths = [0] * n_seq

    def step(self, ids, counts=None) -> CudaTensor:
        """ids i32 [n_seq, n] (a host array, or a device tensor such as ``sample``'s result as [n_seq, 1]): the next
        tokens, ``counts[b]`` of them for sequence b (default all n; the rest of a row is padding). Every sequence
        gets at least one. Returns logits bf16 [n_seq, vocab] after each sequence's last token. Pages are taken
        from the pool first: when it is exhausted or the context is full nothing has changed."""
        be, cfg = self.model.backend, self.model.cfg
        on_device = isinstance(ids, CudaTensor)
        ids = ids if on_device else np.ascontiguousarray(ids, np.int32)
        if len(ids.shape) != 2 or ids.shape[0] != self.n_seq or ids.shape[1] == 0:
            raise ValueError(f"GPT2Session: ids [{','.join(map(str, ids.shape))}] for {self.n_seq} sequences")
        B, n = ids.shape
        counts = [n] * B if counts is None else [int(c) for c in counts]
        if len(counts) != B or not all(0 < c <= n for c in counts):
            raise ValueError(f"GPT2Session: counts {counts} of rows of {n} tokens")
        start = list(self.lengths)
        after = [s + c for s, c in zip(start, counts)]
        if max(after) > cfg.n_ctx:
            raise ValueError(f"GPT2Session: {max(after)} tokens are more than the context ({cfg.n_ctx})")
        self.table.reserve(after)
        i = np.arange(n)
        live = i[None, :] < np.asarray(counts)[:, None]
        pos = np.where(live, np.asarray(start)[:, None] + i[None, :], -1).astype(np.int32)
        up = lambda a: be.from_host_sync(host("i32", a.shape, a))  # noqa: E731
        tmp = [up(pos.reshape(-1)), up(np.repeat(np.arange(B), n).astype(np.int32)), up(np.asarray(after, np.int32)),
               up(np.maximum(pos, 0)), up((np.arange(B) * n + np.asarray(counts) - 1).astype(np.int32))]
        d_pos, d_seq, d_len, d_wpe, d_last = tmp
        if not on_device:
            ids = up(ids)
            tmp.append(ids)
        D, H, Dh = cfg.d_model, cfg.n_head, cfg.head_dim
        w, table = self.model.w, self.table.device
        attend = self._attention(n, start, after, pos, d_len, tmp)
        tok, place = be.embedding(w["wte"], ids), be.embedding(w["wpe"], d_wpe)
        s = be.add(tok, place)
        x = be.reshape(s, (B * n, D))
        tmp += [tok, place, s]
        for layer, cache in enumerate(self.caches):
            def over_cache(qkv, cache=cache):
                flat = be.reshape(qkv, (B * n, 3 * D))
                be.kv_append_packed(cache, flat, table, d_pos, d_seq)
                be.dispose(flat)
                return attend(qkv, cache)

            x = self.model._block(x, f"h.{layer}.", B, n, D, H, Dh, over_cache)
        last = be.embedding(x, d_last) if n > 1 else x  # the rows that are followed by new tokens
        h = be.layerNorm(last, w["ln_f.weight"], w["ln_f.bias"], cfg.eps)
        logits = be.linear(h, w["wte"])
        _ = logits.ptr
        for t in tmp + [x, last, h]:
            be.dispose(t)
        self.lengths = after
        return logits

    def _attention(self, n: int, start, after, pos, d_len, tmp):
        """The attention of a step: qkv [B, n, 3D] and a layer's cache (the new rows in it) -> [B, n, D]."""
        be, cfg, B = self.model.backend, self.model.cfg, self.n_seq
        H, Dh, D = cfg.n_head, cfg.head_dim, cfg.d_model
        scale, table = 1.0 / math.sqrt(Dh), self.table.device
        if not any(start) and n > 1:
            return lambda qkv, cache: be.sdpa_packed(qkv, H, scale, causal=True)
        if n == 1:
            def one(qkv, cache):
                flat = be.reshape(qkv, (B, 3 * D))
                o = be.sdpa_paged_packed(flat, cache, table, d_len, scale)
                out = be.reshape(o, (B, 1, D))
                be.dispose(flat)
                be.dispose(o)
                return out
            return one
        # Several tokens behind a cached prefix: the whole sequences read back, new token i of sequence b seeing
        # positions 0 .. start[b] + i.
        L = max(after)
        j = np.arange(L)
        all_pos = np.where(j[None, :] < np.asarray(after)[:, None], j[None, :], -1).astype(np.int32).reshape(-1)
        seen = (j[None, None, None, :] <= pos[:, None, :, None])
        up = lambda dt, a: be.from_host_sync(host(dt, a.shape, a))  # noqa: E731
        d_pos, d_seq = up("i32", all_pos), up("i32", np.repeat(np.arange(B), L).astype(np.int32))
        mask = up("bool", seen)
        tmp += [d_pos, d_seq, mask]

        def several(qkv, cache):
            k, v = be.kv_read(cache, table, d_pos, d_seq, dtype="bf16")
            q = be.slice(qkv, [0, 0, 0], [B, n, D])
            heads = [be.reshape(q, (B, n, H, Dh)), be.reshape(k, (B, L, H, Dh)), be.reshape(v, (B, L, H, Dh))]
            by_head = [be.transpose(t, (0, 2, 1, 3)) for t in heads]
            o = be.sdpa(*by_head, mask, scale)
            rows = be.transpose(o, (0, 2, 1, 3))
            out = be.reshape(rows, (B, n, D))
            for t in [k, v, q, o, rows] + heads + by_head:
                be.dispose(t)
            return out
        return several

    def generate(self, prompts, max_new: int, u=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> list:
        """Continues every prompt (a list of token lists, one per sequence) by ``max_new`` tokens drawn with
        ``CudaBackend.sample`` from the uniform numbers u [n_seq, max_new] (none needed with temperature 0: the
        best token). Returns the new tokens. The session goes on from there; the last token drawn has not been
        fed yet, so the next ids begin with it. Settings are checked and pages for all of it are taken first: when a
        setting is refused, or the pool or the context is too small, nothing has changed."""
        be, n_ctx = self.model.backend, self.model.cfg.n_ctx
        if len(prompts) != self.n_seq or not all(len(p) for p in prompts):
            raise ValueError(f"GPT2Session: {len(prompts)} prompts for {self.n_seq} sequences, none of them empty")
        if u is None:
            if not isinstance(temperature, (int, float)) or temperature > 0:
                raise ValueError("GPT2Session: drawing needs the uniform numbers u")
            u = np.zeros((self.n_seq, max_new))
        u = np.asarray(u, np.float32)
        if u.shape != (self.n_seq, max_new):
            raise ValueError(f"GPT2Session: u [{','.join(map(str, u.shape))}] for {self.n_seq} sequences of {max_new} tokens")
        be._sample_settings(F.SampleDesc(), self.n_seq, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        if max_new:
            after = [s + len(p) + max_new - 1 for s, p in zip(self.lengths, prompts)]
            if max(after) > n_ctx:
                raise ValueError(f"GPT2Session: {max(after)} tokens are more than the context ({n_ctx})")
            self.table.reserve(after)
        longest = max(len(p) for p in prompts)
        ids = np.zeros((self.n_seq, longest), np.int32)
        for row, p in zip(ids, prompts):
            row[: len(p)] = p
        draws = be.from_host_sync(host("f32", (max_new, self.n_seq), u.T))
        by_step = be.split(draws, max_new) if max_new else []
        tokens, step, counts = [], ids, [len(p) for p in prompts]
        for i in range(max_new):
            logits = self.step(step, counts)
            draw = be.reshape(by_step[i], (self.n_seq,))
            tokens.append(be.sample(logits, draw, temperature, top_k, top_p, min_p))
            for t in (logits, draw) + ((step,) if i else ()):
                be.dispose(t)
            step, counts = be.reshape(tokens[-1], (self.n_seq, 1)), None
        if max_new:
            be.dispose(step)
        out = np.stack([be.read_sync(t).data for t in tokens], 1) if max_new else np.zeros((self.n_seq, 0), np.int32)
        for t in tokens + by_step + [draws]:
            be.dispose(t)
        return out.tolist()

    def release(self, b: int) -> None:
        """Ends sequence b: its pages go back to the pool and the next tokens start it anew."""
        self.table.release(b)
        self.lengths[b] = 0

    def dispose(self) -> None:
        for c in self.caches:
            c.dispose()
        self.table.dispose()

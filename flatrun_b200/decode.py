"""Device-resident greedy decode of a Qwen2/Llama-architecture model.

Every operator of a decode token runs on the GPU, stream-ordered, with no
host round trip between layers, and the whole token is captured in one CUDA
graph that replays for every token (the token's position and id live in
device memory):

  embedding row                       frc_embed_row
  per layer:
    RMSNorm + q, k, v projections     frc_gemv_ex (norm inside the launch;
                                      one launch per quant group)
    bias + RoPE + KV append           frc_rope_append
    GQA attention over the cache      frc_attention_decode (split positions)
    o projection + residual           frc_gemv_ex, FRC_GEMV_ACCUMULATE
    RMSNorm + gate, up projections    frc_gemv_ex (one fused launch)
    SwiGLU + down + residual          frc_gemv_ex: x = silu(gate) * up, accumulate
  final RMSNorm + lm_head, argmax     frc_gemv_ex, frc_argmax

This is the reference forwarder's decode step (flatrun/model/qwen2.py
``make_qwen2_forwarder``: :1510-1646 attention, :1648-1751 MLP, :2238-2297
head) with the NumPy work moved onto the device; the projections are the
same B200 kernels the ``cuda`` backend slot calls.  PyTorch is used only to
allocate device memory and for the stream and graph plumbing (and, in
``prefill``, for the elementwise steps between the kernels).

``kv_bits=4`` keeps the cache in 4 bits (5 with its scales, against 32): the
attention steps are then ``flatrun_b200.attention``'s:

    bias + RoPE                         frc_qk_norm_rope (in place)
    quantise and append                 frc_kv_append_q4
    attention over the 4-bit cache      frc_attention_decode_q4

``prefill`` takes a whole prompt at once: batched projections, rotation,
``frc_attention_prefill`` in fp16, and the prompt's keys and values into the
cache of either kind.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import numpy as np

from . import _lib

_PROJ = ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj",
         "mlp.up_proj", "mlp.down_proj")


@dataclass(frozen=True)
class DecoderConfig:
    hidden: int
    ffn: int
    vocab: int
    layers: int
    heads: int
    kv_heads: int
    eps: float
    rope_theta: float
    max_pos: int
    rope_scaling: dict | None = None  # of attention.rope_tables_scaled; None: the reference's fp32 tables

    @property
    def head_dim(self) -> int:
        return self.hidden // self.heads


def rope_tables(head_dim: int, theta: float, max_pos: int) -> tuple[np.ndarray, np.ndarray]:
    """cos/sin tables [max_pos][head_dim / 2] in fp32, computed as the
    reference does (qwen2.py:398-476): inv_freq = 1 / theta^(2i / d),
    angles = positions x inv_freq."""
    inv_freq = 1.0 / (theta ** (np.arange(0, head_dim, 2, dtype=np.float32) / head_dim))
    freqs = np.outer(np.arange(max_pos, dtype=np.float32), inv_freq)
    return np.cos(freqs).astype(np.float32), np.sin(freqs).astype(np.float32)


def _half_operands(q, k, v):
    """q, the parts of k and the parts of v (fp32, (tokens, heads, head_dim)) as fp16 operands
    of prompt attention: (q, k, v, up), the result being `up` times what they give.

    Where something lies beyond 2^15 it is taken down by a power of two; v's is `up`, and
    q and k take over each other's as far as they stay below 2^15 themselves, so that the
    scores are the same.  (Where both are that large the scores come down with them: by less
    than what their fp16 roundings leave open, which stays far above one.)  Decided on the
    device: the factors are 1 for what fp16 holds."""
    import torch

    def beyond(parts):  # exponent of the largest, and how far it is above 15
        top = torch.stack([torch.linalg.vector_norm(x, float("inf")) if x.numel() else x.new_zeros(()) for x in parts]).amax()
        e = torch.frexp(top)[1].float()
        e = torch.where(torch.isfinite(top), e, torch.zeros_like(e))
        return e, (e - 15).clamp(min=0)

    (eq, a), (ek, b), (_, c) = beyond([q]), beyond(k), beyond(v)
    fq = torch.exp2(torch.minimum(b, 15 - eq.clamp(max=15)) - a)
    fk = torch.exp2(torch.minimum(a, 15 - ek.clamp(max=15)) - b)
    k, v = (torch.cat([(x * f).half() for x in parts]) for parts, f in ((k, fk), (v, torch.exp2(-c))))
    return (q * fq).half(), k, v, torch.exp2(c)


class DecodeEngine:
    """Greedy decode of one sequence with every weight and the KV cache in HBM.

    `weights` maps the reference's tensor names to host arrays or device
    tensors: raw GGUF block bytes (uint8, with `quant_of(name)` -> (n, k,
    quant)) for the projections and the head, fp32 arrays for norms, biases
    and an fp32 embedding table (or raw bytes with its quant).  `kv_prefill` optionally
    maps a layer to (keys, values) of shape (positions, kv_heads, head_dim)
    already in the cache before the first token.  `kv_bits` is 32 or 4 (pages
    of `kv_page` tokens, a multiple of 16).
    """

    def __init__(self, cfg: DecoderConfig, weights: dict, quant_of, device: int = 0, kv_prefill=None,
                 attn_splits: int = 0, kv_bits: int = 32, kv_page: int = 64):
        import torch

        if kv_bits not in (32, 4):
            raise ValueError(f"kv_bits must be 32 or 4, not {kv_bits}")

        self.torch = torch
        self.cfg = cfg
        self.lib = _lib.load()
        self.device = device
        self._dev = torch.device("cuda", device)
        self.stream = torch.cuda.Stream(device=self._dev)
        c = cfg
        hd, kvd = c.head_dim, c.kv_heads * c.head_dim
        f32 = torch.float32

        def up(a, dtype):
            # host arrays are copied in; device tensors (a streamed GGUF
            # file, gguf_stream.load_decoder) are used where they are
            if isinstance(a, torch.Tensor):
                return a.to(self._dev).reshape(-1).view(torch.uint8) if dtype is np.uint8 \
                    else a.to(self._dev, torch.float32)
            a = np.asarray(a, dtype)
            return torch.from_numpy(np.ascontiguousarray(a.reshape(-1) if dtype is np.uint8 else a)).to(self._dev)

        self._w = {}  # name -> (device tensor, quant id, n, k)
        for name, arr in weights.items():
            q = quant_of(name)
            if q is not None:
                n, k, quant = q
                self._w[name] = (up(arr, np.uint8), _lib.QUANT_IDS[quant], n, k)
        self._norm = {name: up(a, np.float32) for name, a in weights.items() if name.endswith("norm.weight")}
        self._bias = {}
        for i in range(c.layers):
            p = f"model.layers.{i}.self_attn"
            if f"{p}.q_proj.bias" in weights:
                self._bias[i] = torch.cat([up(weights[f"{p}.{n}.bias"], np.float32).reshape(-1)
                                           for n in ("q_proj", "k_proj", "v_proj")])
        emb = weights["model.embed_tokens.weight"]
        eq = quant_of("model.embed_tokens.weight")
        self._emb_quant = 0 if eq is None else _lib.QUANT_IDS[eq[2]]
        self._emb = up(emb, np.float32 if eq is None else np.uint8)
        if c.rope_scaling is None:
            cos, sin = rope_tables(hd, c.rope_theta, c.max_pos)
        else:
            from .attention import rope_tables_scaled
            cos, sin = rope_tables_scaled(hd, c.rope_theta, c.max_pos, c.rope_scaling)
        self._cos, self._sin = up(cos, np.float32), up(sin, np.float32)
        self.kv_bits = kv_bits
        if kv_bits == 4:
            from . import attention
            self._attn = attention
            pages = -(-c.max_pos // kv_page)
            self.q4_cache = [attention.kv_cache_q4(pages, kv_page, c.kv_heads, hd, self._dev) for _ in range(c.layers)]
            self._table = torch.arange(pages, dtype=torch.int32, device=self._dev).reshape(1, -1)
            self._q4_joins = attention._decode_q4_kernels(1, c.heads, c.kv_heads, pages * kv_page) - 1
        else:
            self.k_cache, self.v_cache = (
                [torch.zeros((c.max_pos, c.kv_heads, hd), dtype=f32, device=self._dev) for _ in range(c.layers)]
                for _ in range(2))
        start = 0
        for i, (kp, vp) in (kv_prefill or {}).items():
            start = kp.shape[0]
            if start > c.max_pos:
                raise ValueError(f"kv_prefill holds {start} positions, max_pos is {c.max_pos}")
            self._store(i, 0, up(kp, np.float32).reshape(kp.shape), up(vp, np.float32).reshape(vp.shape))
        self.pos = torch.tensor([start], dtype=torch.int32, device=self._dev)
        self._filled = start  # the position, known to the host: a token at max_pos would lie behind tables and caches
        if kv_bits == 4:  # the token's slot, and the number of tokens with it
            self._slot = torch.tensor([start], dtype=torch.int64, device=self._dev)
            self._length = torch.tensor([start + 1], dtype=torch.int32, device=self._dev)
        self.tok_in = torch.zeros(1, dtype=torch.int32, device=self._dev)
        self.tok_out = torch.zeros(1, dtype=torch.int32, device=self._dev)
        self.h = torch.zeros(c.hidden, dtype=f32, device=self._dev)
        self.x = torch.zeros(c.hidden, dtype=f32, device=self._dev)
        self.qkv = torch.zeros(c.hidden + 2 * kvd, dtype=f32, device=self._dev)
        self.ctx = torch.zeros(c.hidden, dtype=f32, device=self._dev)
        self.gate = torch.zeros(c.ffn, dtype=f32, device=self._dev)
        self.upb = torch.zeros(c.ffn, dtype=f32, device=self._dev)
        self.logits = torch.zeros(c.vocab, dtype=f32, device=self._dev)
        # one attention CTA per SM and KV head: each of its eight warps keeps
        # eight K (or V) rows in flight
        sm = torch.cuda.get_device_properties(self._dev).multi_processor_count
        self.splits = attn_splits or max(1, sm // c.kv_heads)
        ws = ctypes.c_size_t()
        _lib.check(self.lib.frc_attention_workspace(c.heads, hd, self.splits, ctypes.byref(ws)), self.lib)
        self.part = torch.zeros(int(ws.value), dtype=f32, device=self._dev)
        _lib.check(self.lib.frc_argmax_workspace(c.vocab, ctypes.byref(ws)), self.lib)
        self.argmax_ws = torch.zeros(int(ws.value), dtype=torch.uint8, device=self._dev)
        self._graph = None
        self.launches_per_token = 0
        # what was filled and stored above ran on the caller's stream, tokens run on the engine's
        torch.cuda.current_stream(self._dev).synchronize()

    def _store(self, layer: int, start: int, k, v) -> None:
        """Keys and values (tokens, kv_heads, head_dim) into the layer's cache from position `start` on."""
        end = start + k.shape[0]
        if self.kv_bits == 4:
            slots = self.torch.arange(start, end, dtype=self.torch.int64, device=self._dev)
            self._attn.kv_append_q4(self.q4_cache[layer], k, v, slots)
        else:
            self.k_cache[layer][start:end] = k
            self.v_cache[layer][start:end] = v

    # ---- launches ------------------------------------------------------------
    def _gemv(self, names, x, ys, x_mul=None, norm=None, accumulate=False):
        ws = [self._w[nm] for nm in names]
        cnt = len(ws)
        rc = self.lib.frc_gemv_ex(ws[0][1], cnt, (ctypes.c_void_p * cnt)(*[w[0].data_ptr() for w in ws]),
                                  (ctypes.c_size_t * cnt)(*[w[0].numel() for w in ws]),
                                  (ctypes.c_int64 * cnt)(*[w[2] for w in ws]), ws[0][3], x.data_ptr(),
                                  x_mul.data_ptr() if x_mul is not None else None,
                                  norm.data_ptr() if norm is not None else None, self.cfg.eps,
                                  _lib.FRC_GEMV_ACCUMULATE if accumulate else 0,
                                  (ctypes.c_void_p * cnt)(*[y.data_ptr() for y in ys]), self._st)
        _lib.check(rc, self.lib)
        self.launches_per_token += 1

    def _groups(self, names):
        """Consecutive names grouped by quant (one fused launch per group)."""
        out = []
        for nm in names:
            if out and self._w[out[-1][0]][1] == self._w[nm][1] and len(out[-1]) < 4:
                out[-1].append(nm)
            else:
                out.append([nm])
        return out

    def _mlp(self, p: str) -> None:
        ln2 = self._norm[f"{p}.post_attention_layernorm.weight"]
        gu = [f"{p}.mlp.gate_proj.weight", f"{p}.mlp.up_proj.weight"]
        for grp in self._groups(gu):
            self._gemv(grp, self.h, [self.gate if g.endswith("gate_proj.weight") else self.upb for g in grp],
                       norm=ln2)
        self._gemv([f"{p}.mlp.down_proj.weight"], self.gate, [self.h], x_mul=self.upb, accumulate=True)

    def _attention_q4(self, layer: int, bias) -> None:
        """The token's attention over the 4-bit cache (on the current stream, which is the engine's)."""
        c, hd, cache = self.cfg, self.cfg.head_dim, self.q4_cache[layer]
        row = self.qkv.view(1, -1)
        q, k, v = (part.view(1, -1, hd) for part in row.split((c.heads * hd, c.kv_heads * hd, c.kv_heads * hd), dim=1))
        self._attn.qk_norm_rope(row, c.heads, c.kv_heads, self._cos, self._sin, self.pos, bias=bias, out=(q, k, v))
        self._attn.kv_append_q4(cache, k, v, self._slot)
        self._attn.attention_decode_q4(q, cache, self._table, self._length, scale=float(np.float32(1.0 / np.sqrt(hd))),
                                       out=self.ctx.view(1, c.heads, hd))
        self.launches_per_token += 3 + self._q4_joins

    def _token(self) -> None:
        """Enqueue one decode token (the graph body)."""
        c, lib, st = self.cfg, self.lib, self._st
        hd, kvd = c.head_dim, c.kv_heads * c.head_dim
        self.launches_per_token = 0

        def chk(rc: int, kernels: int = 1) -> None:
            _lib.check(rc, lib)
            self.launches_per_token += kernels

        chk(lib.frc_embed_row(self._emb_quant, self._emb.data_ptr(), c.hidden, self.tok_in.data_ptr(),
                              self.h.data_ptr(), st))
        q_out = self.qkv[:c.hidden]
        k_out = self.qkv[c.hidden:c.hidden + kvd]
        v_out = self.qkv[c.hidden + kvd:]
        outs = {"self_attn.q_proj": q_out, "self_attn.k_proj": k_out, "self_attn.v_proj": v_out}
        scale = float(np.float32(1.0 / np.sqrt(hd)))
        for i in range(c.layers):
            p = f"model.layers.{i}"
            ln1 = self._norm[f"{p}.input_layernorm.weight"]
            for grp in self._groups([f"{p}.{nm}.weight" for nm in _PROJ[:3]]):
                self._gemv(grp, self.h, [outs[g[len(p) + 1:-len(".weight")]] for g in grp], norm=ln1)
            bias = self._bias.get(i)
            if self.kv_bits == 4:
                self._attention_q4(i, bias)
                self._gemv([f"{p}.self_attn.o_proj.weight"], self.ctx, [self.h], accumulate=True)
                self._mlp(p)
                continue
            chk(lib.frc_rope_append(self.qkv.data_ptr(), bias.data_ptr() if bias is not None else None, c.heads,
                                    c.kv_heads, hd, self._cos.data_ptr(), self._sin.data_ptr(), self.pos.data_ptr(),
                                    self.k_cache[i].data_ptr(), self.v_cache[i].data_ptr(), st))
            chk(lib.frc_attention_decode(q_out.data_ptr(), self.k_cache[i].data_ptr(), self.v_cache[i].data_ptr(),
                                         self.pos.data_ptr(), c.heads, c.kv_heads, hd, scale, self.splits,
                                         self.part.data_ptr(), self.ctx.data_ptr(), st), kernels=2)
            self._gemv([f"{p}.self_attn.o_proj.weight"], self.ctx, [self.h], accumulate=True)
            self._mlp(p)
        self._gemv(["lm_head.weight"], self.h, [self.logits], norm=self._norm["model.norm.weight"])
        chk(lib.frc_argmax(self.logits.data_ptr(), c.vocab, self.tok_out.data_ptr(), self.argmax_ws.data_ptr(), st))
        chk(lib.frc_pos_advance(self.pos.data_ptr(), st))
        if self.kv_bits == 4:  # (the slot is below 2^31: its low word)
            chk(lib.frc_pos_advance(self._length.data_ptr(), st))
            chk(lib.frc_pos_advance(self._slot.data_ptr(), st))
        # the greedy pick is the next token's input unless step() overrides it
        self.tok_in.copy_(self.tok_out)
        self.launches_per_token += 1

    @property
    def _st(self):
        return ctypes.c_void_p(self.stream.cuda_stream)

    def capture(self) -> None:
        """Record one token as a CUDA graph (replayed by step()).  The position,
        the last token's logits and its pick stay as they are."""
        torch = self.torch
        self._room(1)  # the eager token below writes its cache row
        with torch.cuda.stream(self.stream):
            # one eager token first: lazy module loading and launch
            # configuration happen outside the capture; then undo its effects
            state = [self.pos, self.tok_in, self.tok_out, self.h, self.logits] + ([self._slot, self._length] if self.kv_bits == 4 else [])
            before = [t.clone() for t in state]
            self._token()
            self.stream.synchronize()
            for t, b in zip(state, before):
                t.copy_(b)
            self._graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self._graph, stream=self.stream):
                self._token()
        self.stream.synchronize()

    def step(self, token: int | None = None) -> None:
        """One token: feed `token` (None: the previous step's argmax) and
        advance the position.  Asynchronous on the engine's stream.  Raises
        ValueError where max_pos tokens are there already, or for a token that
        the vocabulary does not have."""
        torch = self.torch
        self._room(1)
        if token is not None and not 0 <= int(token) < self.cfg.vocab:
            raise ValueError(f"token ids must lie in 0 .. {self.cfg.vocab - 1}, not {token}")
        with torch.cuda.stream(self.stream):
            if token is not None:
                self.tok_in.fill_(int(token))
            if self._graph is None:
                self._token()
            else:
                self._graph.replay()
        self._filled += 1

    def _room(self, tokens: int) -> None:
        if self._filled + tokens > self.cfg.max_pos:
            raise ValueError(f"{tokens} tokens from position {self._filled} on pass max_pos {self.cfg.max_pos}")

    def prefill(self, tokens) -> None:
        """Feed a prompt at once, behind what the cache holds: afterwards `logits`
        and `argmax_host()` are those of its last token, and `step()` goes on.
        The projections run batched (above 16 tokens with fp16 operands, as
        frc_gemv's), the attention on fp16 queries, keys and values (scaled
        by powers of two where they lie beyond fp16's range);
        asynchronous on the engine's stream."""
        from . import attention

        torch, c, lib, f32 = self.torch, self.cfg, self.lib, self.torch.float32
        ids = np.asarray(tokens, np.int32).reshape(-1)
        n, hd = ids.size, c.head_dim
        kvd = c.kv_heads * hd
        if hd not in (64, 128):
            raise ValueError(f"prompt attention needs a head_dim of 64 or 128, not {hd}")
        if n == 0:
            raise ValueError("an empty prompt")
        if ids.min() < 0 or ids.max() >= c.vocab:
            raise ValueError(f"token ids must lie in 0 .. {c.vocab - 1}")
        self._room(n)
        start = self._filled
        with torch.cuda.stream(self.stream):
            ids_dev = torch.from_numpy(ids).to(self._dev)
            h = torch.empty((n, c.hidden), dtype=f32, device=self._dev)
            for t in range(n):
                _lib.check(lib.frc_embed_row(self._emb_quant, self._emb.data_ptr(), c.hidden, ids_dev[t:].data_ptr(),
                                             h[t].data_ptr(), self._st), lib)

            def norm(x, w):
                y = torch.empty_like(x)
                _lib.check(lib.frc_rmsnorm(x.data_ptr(), w.data_ptr(), n, x.shape[1], c.eps, y.data_ptr(), self._st),
                           lib)
                return y

            def project(name, x):
                # rows scaled by powers of two to below 2, so that none leaves fp16's range in the GEMM
                w, quant, rows, k = self._w[name]
                up = torch.exp2(torch.floor(torch.log2(x.abs().amax(dim=1, keepdim=True).clamp(min=1e-30))))
                x = x / up
                y = torch.empty((n, rows), dtype=f32, device=self._dev)
                _lib.check(lib.frc_gemv(quant, w.data_ptr(), w.numel(), rows, k, x.data_ptr(), n, y.data_ptr(), self._st),
                           lib)
                return y.mul_(up)

            pos = torch.arange(start, start + n, dtype=torch.int32, device=self._dev)
            cu_q, cu_k = (torch.tensor([0, m], dtype=torch.int32, device=self._dev) for m in (n, start + n))
            for i in range(c.layers):
                p = f"model.layers.{i}"
                x = norm(h, self._norm[f"{p}.input_layernorm.weight"])
                qkv = torch.cat([project(f"{p}.{m}.weight", x) for m in _PROJ[:3]], dim=1)
                parts = tuple(t.unflatten(1, (-1, hd)) for t in qkv.split((c.hidden, kvd, kvd), dim=1))
                q, k, v = attention.qk_norm_rope(qkv, c.heads, c.kv_heads, self._cos, self._sin, pos,
                                                 bias=self._bias.get(i), out=parts)
                self._store(i, start, k, v)
                k, v = [k], [v]
                if start:
                    if self.kv_bits == 4:
                        slots = torch.arange(start, dtype=torch.int64, device=self._dev)
                        past = attention.kv_read_q4(self.q4_cache[i], slots)
                    else:
                        past = (self.k_cache[i][:start], self.v_cache[i][:start])
                    k, v = ([x] + y for x, y in zip(past, (k, v)))
                q, k, v, up = _half_operands(q, k, v)
                ctx = attention.attention_prefill(q, k, v, cu_q, cu_k, scale=float(np.float32(1.0 / np.sqrt(hd))))
                h += project(f"{p}.self_attn.o_proj.weight", ctx.reshape(n, c.hidden).float().mul_(up))
                x = norm(h, self._norm[f"{p}.post_attention_layernorm.weight"])
                gate = torch.nn.functional.silu(project(f"{p}.mlp.gate_proj.weight", x))
                h += project(f"{p}.mlp.down_proj.weight", gate * project(f"{p}.mlp.up_proj.weight", x))
            self.h.copy_(h[-1])
            launches = self.launches_per_token  # a token's, which the prompt is not
            self._gemv(["lm_head.weight"], self.h, [self.logits], norm=self._norm["model.norm.weight"])
            self.launches_per_token = launches
            _lib.check(lib.frc_argmax(self.logits.data_ptr(), c.vocab, self.tok_out.data_ptr(), self.argmax_ws.data_ptr(),
                                      self._st), lib)
            self.tok_in.copy_(self.tok_out)
            self.pos += n
            if self.kv_bits == 4:
                self._slot += n
                self._length += n
        self._filled += n

    def logits_host(self) -> np.ndarray:
        self.stream.synchronize()
        return self.logits.cpu().numpy()

    def argmax_host(self) -> int:
        self.stream.synchronize()
        return int(self.tok_out.item())

    def close(self) -> None:
        self._graph = None
        self.stream.synchronize()


__all__ = ["DecoderConfig", "DecodeEngine", "rope_tables"]

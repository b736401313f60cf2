"""KV-cache generation for the Llama family on the gfx950 kernels (serving / evaluation of a trained chart).

Prefill runs the prompt through the training forward's kernels (fused residual + RMSNorm, one QKV GEMM, RoPE
in place, the flash-attention forward, SwiGLU MLP) and writes each layer's rotated K and V into a
preallocated cache; every decode step then pushes one token per sequence through the same projections with
RoPE at the sequence's position and the split-K decode-attention kernel (``csrc/decode_attn.hip``) over the
cache. MI355X-first sizing: the cache is one contiguous [B, Hkv, Smax, D] bf16 tensor per layer for K and for
V (each (sequence, KV head) a contiguous slab the decode kernel streams) (Llama-3-8B: 128 KiB per token across its 32 layers, so 288 GB of HBM minus 16 GB of weights holds ~2M
cached tokens, e.g. 256 sequences x 8k context), allocated once, never reshaped or copied between steps.

Many requests on one model. A prompt that every request starts with is prefilled once (``set_prefix``): its K / V are held
once, every step reads them once for the whole batch, and the sequences' own caches start behind it
(``kf.prefix_attention``). Requests can bring low-rank adapters (``set_adapters``, one index per cache slot): each
projection adds its rows' own (``kf.lora_add``). ``extend`` pushes several tokens per sequence through one step, and
``speculate`` uses it to check the tokens that a small draft model proposes (``kf.verify_draft``): the outputs are the
large model's own samples, several per step of it.

Weights are the model's own parameters (views into a trainer's flat store, or any loaded Llama module); the
generator adds no autograd state (``torch.no_grad``). On CPU every op falls back to its PyTorch reference.
"""
from __future__ import annotations

import math
import os

import torch

from ..models.llama import Llama
from ..ops import functional as kf
from ..ops import reference as ref


class KVCache:
    def __init__(self, n_layers: int, batch: int, max_seq: int, n_kv_heads: int, head_dim: int, device,
                 dtype=torch.bfloat16):
        shape = (batch, n_kv_heads, max_seq, head_dim)
        self.k = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        self.v = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.host_lens = [0] * batch  # host mirror of lens: sizes the decode kernel's split grid without a sync
        self.batch, self.max_seq = batch, max_seq

    @property
    def max_len(self) -> int:
        return max(self.host_lens)

    def release(self, slot: int) -> None:
        """Free a sequence slot (continuous batching): its next prefill overwrites the stale rows."""
        self.host_lens[slot] = 0
        self.lens[slot] = 0

    def truncate(self, lens: list) -> None:
        """Forget what rows [0, len(lens)) hold past the given lengths (drafted tokens that were refused)."""
        if len(lens) > self.batch or any(not 0 <= n <= h for n, h in zip(lens, self.host_lens)):
            raise ValueError("truncate can only shorten the cached sequences")
        self.host_lens[: len(lens)] = [int(n) for n in lens]
        self.lens[: len(lens)] = torch.tensor(lens, dtype=torch.int32).to(self.lens.device)

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.k + self.v)


class LoraAdapters:
    """Low-rank adapters of many requests for the block projections, stacked so that one launch serves a mixed batch: per
    layer and projection a [n, rank, in] and b [n, out, rank] in bf16 (``ops.lora_add``), and one scale per adapter.
    ``rank``: a multiple of 8 (pad smaller adapters with zeros). New adapters are zero: ``set`` fills one in."""

    TARGETS = ("wqkv", "wo", "w_gate_up", "w_down")

    def __init__(self, cfg, n: int, rank: int, device, targets=TARGETS):
        if n < 1 or rank < 8 or rank % 8 or rank > 128 or not targets or any(t not in self.TARGETS for t in targets):
            raise ValueError("n >= 1 adapters, a rank that is a multiple of 8 up to 128, targets among " + ", ".join(self.TARGETS))
        D, H, F = cfg.head_dim, cfg.hidden, cfg.ffn_hidden
        shape = {"wqkv": ((cfg.n_heads + 2 * cfg.n_kv_heads) * D, H), "wo": (H, cfg.n_heads * D), "w_gate_up": (2 * F, H),
                 "w_down": (H, F)}
        self.n, self.rank, self.targets = n, rank, tuple(targets)
        self.scale = torch.ones(n, dtype=torch.float32, device=device)
        self.layers = [{t: (torch.zeros(n, rank, shape[t][1], dtype=torch.bfloat16, device=device),
                            torch.zeros(n, shape[t][0], rank, dtype=torch.bfloat16, device=device)) for t in targets}
                       for _ in range(cfg.n_layers)]

    def set(self, i: int, layer: int, target: str, a: torch.Tensor, b: torch.Tensor) -> None:
        """Adapter ``i`` of one projection: a [r, in], b [out, r] with r <= rank (the rest is zero)."""
        A, B = self.layers[layer][target]
        if not 0 <= i < self.n or a.shape[0] > self.rank or b.shape[1] != a.shape[0] or a.shape[1] != A.shape[2] \
                or b.shape[0] != B.shape[1]:
            raise ValueError("adapter index or shape")
        A[i].zero_()
        B[i].zero_()
        A[i, : a.shape[0]] = a.to(A)
        B[i, :, : a.shape[0]] = b.to(B)

    def state_dict(self) -> dict:
        out = {"scale": self.scale}
        for li, layer in enumerate(self.layers):
            for t, (a, b) in layer.items():
                out[f"layers.{li}.{t}.a"], out[f"layers.{li}.{t}.b"] = a, b
        return out

    @classmethod
    def load(cls, cfg, path: str, device) -> "LoraAdapters":
        """From a file of ``torch.save(adapters.state_dict(), path)`` (read with ``weights_only=True``)."""
        sd = torch.load(path, map_location=device, weights_only=True)
        targets = [t for t in cls.TARGETS if f"layers.0.{t}.a" in sd]
        if not targets or "scale" not in sd:
            raise ValueError(f"{path} holds no adapters")
        n, rank, _ = sd[f"layers.0.{targets[0]}.a"].shape
        self = cls(cfg, n, rank, device, targets)
        mine = self.state_dict()
        if mine.keys() != sd.keys() or any(mine[k].shape != sd[k].shape for k in mine):
            raise ValueError(f"{path}: adapters of another model")
        for k in mine:
            mine[k].copy_(sd[k])
        return self


class LlamaGenerator:
    """``graph``: replay each decode step as one captured HIP graph (``torch.cuda.CUDAGraph`` is a hipGraph on
    ROCm) -- a decode step is ~400 small launches whose host-side cost dominates at small batch. The graph's
    decode-attention grid then covers the whole cache (splits past a sequence's length exit at once)."""

    def __init__(self, model: Llama, max_batch: int, max_seq: int, graph: bool = False, fp8: bool = False):
        """``fp8``: E4M3 copies of the four block projections (per-tensor scale) are attached to the model's
        weights (``w.w8``, read by ``ops.functional`` linear / swiglu_mlp): decode steps then read half the weight
        bytes. Serving-only models: a trainer would pick the copies up too (``drop_fp8`` removes them)."""
        if not isinstance(model, Llama) or model.tp.enabled:
            raise ValueError("the generator serves single-GPU Llama models")
        self.model = model
        if fp8:
            from ..ops import fp8 as f8

            with torch.no_grad():
                for blk in model.layers:
                    for w in (blk.wqkv, blk.wo, blk.w_gate_up, blk.w_down):
                        w.w8, w.w8_scale = f8.quantize(w.detach())
        c = model.cfg
        self.cfg = c
        self.device = model.tok_emb.device
        self.cache = KVCache(c.n_layers, max_batch, max_seq, c.n_kv_heads, c.head_dim, self.device)
        self.cos, self.sin = ref.rope_cache(max_seq, c.head_dim, c.rope_theta, device=self.device)
        self.scale = 1.0 / math.sqrt(c.head_dim)
        self.prefix_len = 0
        self.prefix: list = []  # per layer (K, V) [Hkv, P, D] of the prompt that every sequence starts with
        self.adapters: LoraAdapters | None = None
        self.slot_adapter = torch.full((max_batch,), -1, dtype=torch.int32, device=self.device)  # -1: none
        self.graph = graph and self.device.type == "cuda"
        self._graphs: dict = {}  # batch -> (graph, static token input, static logits output)
        # decode projections of <= GEMV_ROWS token rows through the HIP GEMV (csrc/gemv.hip); KOP_DECODE_GEMV=0: GEMMs
        self._gemv = self.device.type == "cuda" and os.environ.get("KOP_DECODE_GEMV", "1") != "0"

    def drop_fp8(self) -> None:
        for blk in self.model.layers:
            for w in (blk.wqkv, blk.wo, blk.w_gate_up, blk.w_down):
                for a in ("w8", "w8_scale"):
                    if hasattr(w, a):
                        delattr(w, a)

    def _head(self):
        return self.model.tok_emb if self.cfg.tie_embeddings else self.model.lm_head

    # rows routed to the GEMV: Llama-3-8B decode at batch 1 runs 4.35 vs 4.77 ms per step (+9.6 %), but at
    # batch 4 / 8 the library GEMM is 15-20 % faster (profiles/r3_decode_gemv_ab.jsonl); the kernel takes up to 8
    GEMV_ROWS = 1

    def _gemv_ok(self, x, w) -> bool:
        return (self._gemv and x.shape[0] <= self.GEMV_ROWS and x.shape[-1] % 1024 == 0
                and w.dtype == torch.bfloat16 and not hasattr(w, "w8"))

    def _lin(self, x, w):
        """x . w^T: a decode step reads every weight once, so for a few token rows the HIP GEMV (weight rows
        streamed at HBM rate) replaces the library GEMM's small-M tiles; FP8 weights and larger batches keep
        ``kf.linear``."""
        if self._gemv_ok(x, w):
            from ..ops import load

            return load().gemv(x, w)
        return kf.linear(x, w)

    def _proj(self, x, i: int, name: str, rows):
        """Projection ``name`` of layer i, with the rows' adapters added (``rows``: each row's adapter, or None)."""
        y = self._lin(x, getattr(self.model.layers[i], name))
        if rows is not None and name in self.adapters.targets:
            a, b = self.adapters.layers[i][name]
            y = kf.lora_add(y, x, a, b, rows, self.adapters.scale, out=y)
        return y

    def _adapter_rows(self, slots: torch.Tensor, tokens: int):
        """Adapter index of every row of a batch of ``tokens`` rows per slot (None: no adapters are set)."""
        if self.adapters is None:
            return None
        idx = self.slot_adapter[slots]
        return idx.repeat_interleave(tokens) if tokens > 1 else idx

    def _mlp(self, blk, y2, i: int = 0, rows=None):
        if rows is not None:
            return self._proj(kf.swiglu(self._proj(y2, i, "w_gate_up", rows)), i, "w_down", rows)
        if self._gemv_ok(y2, blk.w_gate_up) and self._gemv_ok(y2, blk.w_down):
            return self._lin(kf.swiglu(self._lin(y2, blk.w_gate_up)), blk.w_down)
        return kf.swiglu_mlp(y2, blk.w_gate_up, blk.w_down)

    def set_adapters(self, adapters: LoraAdapters | None) -> None:
        """Serve with these adapters (``prefill(adapters=)`` chooses each sequence's); None: without."""
        self.adapters = adapters
        self.slot_adapter.fill_(-1)
        self._graphs.clear()  # captured steps hold the launches of the old set

    @torch.no_grad()
    def set_prefix(self, ids: torch.Tensor | None) -> None:
        """The tokens [P] that every sequence starts with (a system prompt), prefilled here once and for all: prompts given
        to ``prefill`` from now on are what follows it, and ``max_seq`` bounds that part alone. None: no prefix. Empties the
        cache. The prefix is the base model's: adapters apply to what follows."""
        c = self.cfg
        P = 0 if ids is None else int(ids.numel())
        if P and self.device.type == "cuda" and c.head_dim not in (64, 128):
            raise ValueError("a shared prefix needs a head dim of 64 or 128")
        self._graphs.clear()
        self.prefix_len, self.prefix = 0, []
        self.cache.host_lens = [0] * self.cache.batch
        self.cache.lens.zero_()
        if P:
            # through a cache of its own, as long as the prefill pads to
            tmp = LlamaGenerator(self.model, 1, -(-P // 128) * 128)
            tmp.prefill(ids.reshape(1, P).to(self.device))
            self.prefix = [(k[0, :, :P].contiguous(), v[0, :, :P].contiguous()) for k, v in zip(tmp.cache.k, tmp.cache.v)]
            self.prefix_len = P
        cos, sin = ref.rope_cache(P + self.cache.max_seq, c.head_dim, c.rope_theta, device=self.device)
        self.cos, self.sin = cos[P:].contiguous(), sin[P:].contiguous()  # own positions start behind the prefix

    def _attend(self, i: int, q, k, v, lens, max_len: int, tokens: int):
        """Attention of ``tokens`` new rows per sequence over its cached keys, and the prefix if there is one."""
        if not self.prefix_len and tokens == 1:
            return kf.decode_attention(q, k, v, lens, max_len, self.scale)
        pk, pv = self.prefix[i] if self.prefix_len else (k[0, :, :0], v[0, :, :0])
        return kf.prefix_attention(q, pk, pv, k, v, lens, max_len, tokens, self.scale)

    @torch.no_grad()
    def prefill(self, ids: torch.Tensor, slot: int = 0, lengths: list | None = None,
                slots: list | None = None, adapters: list | None = None) -> torch.Tensor:
        """Prompts ``ids`` [B, S] into cache rows [slot, slot + B) (or the listed ``slots``) -> logits of each
        prompt's last position [B, vocab] (fp32). ``lengths``: real lengths of right-padded rows (default S):
        causal attention keeps every real position independent of the padding after it. ``adapters``: each sequence's
        adapter index (-1: none; default none)."""
        c, m = self.cfg, self.model
        B, S = ids.shape
        slots = list(range(slot, slot + B)) if slots is None else list(slots)
        lengths = [S] * B if lengths is None else list(lengths)
        if len(slots) != B or len(lengths) != B or max(slots) >= self.cache.batch or S > self.cache.max_seq:
            raise ValueError("prompt batch / length exceeds the cache")
        if adapters is not None and (self.adapters is None or len(adapters) != B
                                     or any(not -1 <= int(x) < self.adapters.n for x in adapters)):
            raise ValueError("adapters: one index in [-1, n) per prompt, with adapters set")
        contiguous = slots == list(range(slots[0], slots[0] + B))
        rows = slice(slots[0], slots[0] + B) if contiguous else torch.tensor(slots, device=self.device)
        if ids.is_cuda and S % 128 and not self.prefix_len and S + 128 - S % 128 <= self.cache.max_seq:
            # right-pad to the HIP flash forward's 128-row tiles: causal attention keeps the real positions
            # independent of the padding, whose cache rows lie past lens and are overwritten by decode steps
            ids = torch.cat([ids, ids.new_zeros(B, 128 - S % 128)], dim=1)
            S = ids.shape[1]
        Hq, Hkv, D = c.n_heads, c.n_kv_heads, c.head_dim
        a, kc = Hq * D, (Hq + Hkv) * D
        ad = full = None
        if self.adapters is not None:
            slot_t = torch.tensor(slots, device=self.device)
            self.slot_adapter[slot_t] = torch.tensor(adapters if adapters is not None else [-1] * B, dtype=torch.int32,
                                                     device=self.device)
            ad = self._adapter_rows(slot_t, S) if adapters is not None else None
        if self.prefix_len:  # every row of a (padded) prompt sees the prefix and the rows before it
            full = torch.full((B,), S, dtype=torch.int32, device=self.device)
        x = kf.embedding(ids.reshape(-1), m.tok_emb)
        pending = None
        for i, blk in enumerate(m.layers):
            if pending is None:
                y, x1 = kf.rms_norm(x, blk.attn_norm, c.norm_eps), x
            else:
                y, x1 = kf.rms_norm(x, blk.attn_norm, c.norm_eps, residual=pending)
            qkv = kf.linear(y, blk.wqkv) if ad is None else self._proj(y, i, "wqkv", ad)
            if qkv.is_cuda:
                from ..ops import load

                load().rope_(qkv, self.cos, self.sin, None, S, Hq + Hkv, D, False)
            else:
                qkv = ref.rope_ref(qkv, self.cos, self.sin, S, Hq + Hkv, D)
            q, k, v = qkv[:, :a], qkv[:, a:kc], qkv[:, kc:]
            kh, vh = k.reshape(B, S, Hkv, D).transpose(1, 2), v.reshape(B, S, Hkv, D).transpose(1, 2)
            if contiguous:  # a slice of the cache: copy in place
                self.cache.k[i][rows, :, :S].copy_(kh)
                self.cache.v[i][rows, :, :S].copy_(vh)
            else:  # index tensor: advanced indexing returns a COPY, so write through index_put_ (assignment)
                self.cache.k[i][rows, :, :S] = kh
                self.cache.v[i][rows, :, :S] = vh
            if self.prefix_len:
                o = self._attend(i, q, kh.contiguous(), vh.contiguous(), full, S, S)
            elif q.is_cuda and S % 128 == 0:  # the HIP flash forward's tile constraint
                o, _ = kf.flash_attention(q, k, v, B, S, Hq, Hkv, D, causal=True, scale=self.scale)
            else:
                o, _ = ref.attention_ref(q, k, v, B, S, Hq, Hkv, D, True, self.scale)
            y2, x = kf.rms_norm(x1, blk.mlp_norm, c.norm_eps, residual=self._proj(o, i, "wo", ad))
            pending = self._mlp(blk, y2, i, ad)
        y, _ = kf.rms_norm(x, m.final_norm, c.norm_eps, residual=pending)
        lt = torch.tensor(lengths, dtype=torch.int32)
        self.cache.lens[rows] = lt.to(self.device)
        for r, n in zip(slots, lengths):
            self.cache.host_lens[r] = int(n)
        last = y.view(B, S, -1)[torch.arange(B, device=y.device), (lt.long() - 1).to(y.device)]
        return torch.mm(last, self._head().t()).float()

    @torch.no_grad()
    def decode(self, tok: torch.Tensor, active: list | None = None) -> torch.Tensor:
        """One new token per sequence ``tok`` [B] (cache rows [0, B)) at position lens[b] -> next-token logits
        [B, vocab] (fp32). ``active`` (host list of bools, continuous batching): only those rows advance; the
        others compute throw-away rows of the same batched GEMMs."""
        B = tok.shape[0]
        rows = range(B) if active is None else [r for r in range(B) if active[r]]
        if max((self.cache.host_lens[r] for r in rows), default=0) + 1 > self.cache.max_seq:
            raise ValueError("KV cache is full")
        max_len = max(self.cache.host_lens[:B]) + 1
        if active is not None:
            act = torch.tensor([bool(x) for x in active[:B]], dtype=torch.int32).to(self.device, non_blocking=True)
            out = self._decode(tok, max_len, act)
        elif not self.graph:
            out = self._decode(tok, max_len)
        else:
            if B not in self._graphs:
                self._capture(B, tok)
            g, static_tok, static_out = self._graphs[B]
            static_tok.copy_(tok)
            g.replay()
            out = static_out.clone()
        for r in rows:
            self.cache.host_lens[r] += 1
        return out

    @torch.no_grad()
    def extend(self, tok: torch.Tensor) -> torch.Tensor:
        """Several new tokens per sequence ``tok`` [B, T] (cache rows [0, B)) at positions lens[b] .. lens[b] + T - 1 ->
        the logits after each of them [B, T, vocab] (fp32): T decode steps in one pass over the weights and the caches.
        ``cache.truncate`` takes tokens back."""
        B, T = tok.shape
        if B < 1 or T < 1 or B > self.cache.batch or max(self.cache.host_lens[:B]) + T > self.cache.max_seq:
            raise ValueError("KV cache is full")
        out = self._decode(tok, max(self.cache.host_lens[:B]) + T)
        for r in range(B):
            self.cache.host_lens[r] += T
        return out.view(B, T, -1)

    def _capture(self, B: int, tok: torch.Tensor) -> None:
        static_tok = tok.clone()
        lens0 = self.cache.lens.clone()
        s = torch.cuda.Stream(device=self.device)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):  # warm-up outside capture (library handles, workspaces); state restored below
            self._decode(static_tok, self.cache.max_seq)
        torch.cuda.current_stream().wait_stream(s)
        self.cache.lens.copy_(lens0)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            static_out = self._decode(static_tok, self.cache.max_seq)
        self.cache.lens.copy_(lens0)  # capture does not run the kernels, but keep the state exact either way
        self._graphs[B] = (g, static_tok, static_out)

    def _decode(self, tok: torch.Tensor, max_len: int, active: torch.Tensor | None = None) -> torch.Tensor:
        """Device-side body of a decode step (no host reads: capturable); ``max_len`` sizes the split grid. ``tok`` [B], or
        [B, T] for T tokens per sequence (rows b * T + t)."""
        c, m = self.cfg, self.model
        B = tok.shape[0]
        T = tok.shape[1] if tok.dim() == 2 else 1
        Hq, Hkv, D = c.n_heads, c.n_kv_heads, c.head_dim
        a, kc = Hq * D, (Hq + Hkv) * D
        pos = self.cache.lens[:B].clone()
        rows = self._rows(B)
        pls = [(pos + t) for t in range(T)] if T > 1 else [pos]
        lens = pos + T
        ad = self._adapter_rows(rows, T)
        x = kf.embedding(tok.reshape(-1), m.tok_emb)
        pending = None
        for i, blk in enumerate(m.layers):
            if pending is None:
                y, x1 = kf.rms_norm(x, blk.attn_norm, c.norm_eps), x
            else:
                y, x1 = kf.rms_norm(x, blk.attn_norm, c.norm_eps, residual=pending)
            qkv = self._proj(y, i, "wqkv", ad)
            by_tok = qkv.view(B, T, -1)
            for t, pt in enumerate(pls):
                row = by_tok[:, t]
                if qkv.is_cuda:  # one kernel: RoPE at pos on Q / K + K / V rows appended to the cache
                    from ..ops import load

                    load().decode_rope_append_(row, self.cos, self.sin, pt, self.cache.k[i], self.cache.v[i], Hq)
                else:
                    kf.rope_positions_(row, self.cos, self.sin, pt, Hq + Hkv, D)
                    self.cache.k[i][rows, :, pt.long()] = row[:, a:kc].reshape(B, Hkv, D)
                    self.cache.v[i][rows, :, pt.long()] = row[:, kc:].reshape(B, Hkv, D)
            o = self._attend(i, qkv[:, :a], self.cache.k[i][:B], self.cache.v[i][:B], lens, max_len, T)
            y2, x = kf.rms_norm(x1, blk.mlp_norm, c.norm_eps, residual=self._proj(o, i, "wo", ad))
            pending = self._mlp(blk, y2, i, ad)
        y, _ = kf.rms_norm(x, m.final_norm, c.norm_eps, residual=pending)
        self.cache.lens[:B] = lens if active is None else pos + active
        return self._lin(y, self._head()).float() if self._gemv_ok(y, self._head()) else \
            torch.mm(y, self._head().t()).float()

    def _rows(self, B: int) -> torch.Tensor:
        key = ("rows", B)
        if key not in self._graphs:
            self._graphs[key] = torch.arange(B, device=self.device)
        return self._graphs[key]

    @torch.no_grad()
    def generate(self, ids: torch.Tensor, max_new_tokens: int, adapters: list | None = None) -> torch.Tensor:
        """Greedy continuation: [B, S] prompt -> [B, S + max_new_tokens] tokens. ``adapters`` as in ``prefill``: each
        sequence's index, default none."""
        out = [ids]
        logits = self.prefill(ids, adapters=adapters)
        for _ in range(max_new_tokens):
            nxt = logits.argmax(-1)
            out.append(nxt.unsqueeze(1).to(ids.dtype))
            if len(out) - 1 == max_new_tokens:
                break
            logits = self.decode(nxt)
        return torch.cat(out, dim=1)

    @torch.no_grad()
    def speculate(self, draft: "LlamaGenerator", ids: torch.Tensor, max_new_tokens: int, drafts: int = 4,
                  temperature: float = 0.0, generator: torch.Generator | None = None, adapters: list | None = None):
        """Continuation of ``ids`` [B, S] through a small draft model: it proposes ``drafts`` tokens per round, one ``extend`` of
        this model scores them all, and ``ops.verify_draft`` keeps the first ones and draws the token after them. With
        ``temperature`` 0 the result is this model's greedy continuation, otherwise it is distributed as this model's
        samples (uniform numbers from ``generator``). ``adapters`` as in ``prefill``: each sequence's index into this model's
        adapters, default none; the draft proposes without any. Returns ([B, S + max_new_tokens] tokens, kept drafts per round);
        both caches then hold all of them but the last, as after ``generate``."""
        B, S = ids.shape
        if draft.cfg.vocab_size != self.cfg.vocab_size or not 1 <= drafts <= 32 or max_new_tokens < 1:
            raise ValueError("the draft needs this model's vocabulary; 1 to 32 drafts per round")
        if draft is self:
            raise ValueError("the draft needs a generator (a cache) of its own")
        if draft.prefix_len != self.prefix_len:
            raise ValueError("give the draft the same prefix")
        for g in (self, draft):  # a finished sequence, all but its last token cached, goes through rounds of drafts + 1 more
            if B > g.cache.batch or S + max_new_tokens + drafts > g.cache.max_seq:
                raise ValueError("KV cache too small for the continuation and one round of drafts")

        def uniform(*shape):
            return torch.rand(*shape, device=self.device, generator=generator)

        def sample(logits):  # one token per row, as verify_draft draws it: no drafted tokens to check
            none = torch.empty(B, 0, dtype=torch.long, device=self.device)
            return kf.verify_draft(logits.unsqueeze(1), None, none, uniform(B, 1), temperature)[0][:, 0]

        out: list = [[] for _ in range(B)]

        def add(new: list, last: torch.Tensor):
            """Each unfinished sequence's new tokens into ``out``; the tokens that the next round starts with (a finished sequence
            computes rows that are thrown away: any token will do)."""
            for o, more in zip(out, new):
                if len(o) >= max_new_tokens:
                    continue
                o += more
                if o[:max_new_tokens][-1] < 0:
                    raise RuntimeError("a row of the model's logits gives no token any probability")
            return last.clamp(min=0)

        cur = sample(self.prefill(ids, adapters=adapters))
        draft.prefill(ids)
        cur = add([[t] for t in cur.tolist()], cur)
        rounds = []
        while min(len(o) for o in out) < max_new_tokens:
            start = self.cache.host_lens[:B]
            tok, toks, qs = cur, [], []
            for _ in range(drafts):
                q = draft.decode(tok)
                toks.append(sample(q))  # -1 (no token has any probability) is refused below
                tok = toks[-1].clamp(min=0)
                qs.append(q)
            draft.decode(tok)  # the last one's keys: all of them may be kept
            proposed = torch.stack(toks, 1)
            p = self.extend(torch.cat([cur.unsqueeze(1), proposed.clamp(min=0)], 1))
            new, kept = kf.verify_draft(p, torch.stack(qs, 1), proposed, uniform(B, drafts + 1), temperature)
            last = new.gather(1, kept.long().unsqueeze(1)).squeeze(1)
            kept = kept.tolist()
            rounds.append(kept)
            cur = add([row[: k + 1] for row, k in zip(new.tolist(), kept)], last)
            # everything but the last token; a finished sequence's rows from then on are thrown away
            lens = [min(n + k + 1, S + max_new_tokens - 1) for n, k in zip(start, kept)]
            for g in (self, draft):
                g.cache.truncate(lens)
        res = torch.tensor([o[:max_new_tokens] for o in out], dtype=ids.dtype, device=ids.device)
        return torch.cat([ids, res], dim=1), rounds

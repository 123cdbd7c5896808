"""Batched greedy decoding of a Hugging-Face-shaped Llama whose linear layers were quantised with
quantize_model_mxfp4 (the reference's README scenario: Llama-2-7B, batch 128; src/mxfp4/utils/model_utils.py:8-73 swaps
the layers, the model's own PyTorch code runs them).

The reference owns only the linear layers of such a model; everything between them is the model's code.  This runner
keeps that split but runs the part the library owns as one fused chain per layer (mxfp4.gemm.FusedChain): the RMS norms
(with their learned weights), the residual adds and silu*mul end directly in MXFP4 activations, the row-parallel sums of
tensor parallelism run inside those same kernels over peer memory, q|k|v and gate|up are one GEMM each.  Attention itself
(rotary embedding, KV cache, softmax(QK^T)V) is torch's scaled_dot_product_attention on a preallocated cache: it is not part
of this library.  A decode step has fixed shapes and is replayed from a CUDA graph.

Tensor parallelism: q/k/v/gate/up are split by output rows (whole heads per rank), o and down by input columns; every
rank holds the KV cache of its own heads.  The only exchange is the row-parallel sum, which runs inside mxfp4_act_fused:
a decode step contains no NCCL call.

With `page_size` the keys and values live in paged caches instead and attention is this library's too (mxfp4.serving): one
launch turns q and k and appends k and v, paged_attention reads the pages, sequences may have their own lengths, and a prefix
given to set_prefix() is held once and attended once for the whole batch.  set_sampling() replaces the greedy choice by
sample_tokens() on given uniform numbers, with either cache.
"""
from typing import Optional

import torch
import torch.nn.functional as F

from . import _capi
from . import gemm as _gemm
from . import serving as _serving
from .parallel import _PeerSum, _group_info, shard_quantized


class LlamaMXDecoder:
    def __init__(self, model, max_batch: int, max_len: int, group=None, page_size: Optional[int] = None, max_prefix: int = 0):
        """`model`: transformers LlamaForCausalLM (or the same module layout) after quantize_model_mxfp4, on a CUDA
        device; the quantised buffers are sliced for this rank, nothing is re-quantised.  page_size: paged caches of pages of so many
        tokens (a power of two from 16), with room for max_len tokens of every sequence and max_prefix of a shared prefix."""
        cfg = model.config
        self.world, self.rank = _group_info(group)
        self.group = group
        base = model.model
        self.dev = base.embed_tokens.weight.device
        self.hidden = cfg.hidden_size
        self.n_heads, self.n_kv = cfg.num_attention_heads, cfg.num_key_value_heads
        self.head_dim = getattr(cfg, "head_dim", None) or cfg.hidden_size // cfg.num_attention_heads
        if self.n_heads % self.world or self.n_kv % self.world:
            raise ValueError(f"{self.n_heads} heads / {self.n_kv} KV heads do not divide over {self.world} ranks")
        self.h_l, self.kv_l = self.n_heads // self.world, self.n_kv // self.world
        self.eps = cfg.rms_norm_eps
        self.B, self.S = max_batch, max_len
        w, r = self.world, self.rank

        def rows(layer):                      # column-parallel: output rows of this rank
            return shard_quantized(layer.packed_weight, layer.weight_scales, 0, w, r)

        def cols(layer):                      # row-parallel: input columns of this rank
            return shard_quantized(layer.packed_weight, layer.weight_scales, 1, w, r)

        self.layers = []
        for L in base.layers:
            a, m = L.self_attn, L.mlp
            for lin in (a.q_proj, a.k_proj, a.v_proj, a.o_proj, m.gate_proj, m.up_proj, m.down_proj):
                if not getattr(lin, "is_quantized", False) or lin.bias is not None:
                    raise ValueError("LlamaMXDecoder needs bias-free projections quantised by quantize_model_mxfp4")
            q, k, v, g, u = rows(a.q_proj), rows(a.k_proj), rows(a.v_proj), rows(m.gate_proj), rows(m.up_proj)
            o, d = cols(a.o_proj), cols(m.down_proj)
            self.layers.append(dict(
                qkv=(torch.cat([q[0], k[0], v[0]], 0), torch.cat([q[1], k[1], v[1]], 0)),
                gateup=(torch.cat([g[0], u[0]], 0), torch.cat([g[1], u[1]], 0)),
                o=o, down=d,
                g1=L.input_layernorm.weight.detach().to(torch.bfloat16).contiguous(),
                g2=L.post_attention_layernorm.weight.detach().to(torch.bfloat16).contiguous()))
        self.g_final = base.norm.weight.detach().to(torch.bfloat16).contiguous()
        self.embed = base.embed_tokens.weight.detach()
        head = model.lm_head
        if not getattr(head, "is_quantized", False):
            raise ValueError("LlamaMXDecoder needs a quantised lm_head")
        self.vocab = head.packed_weight.shape[0]
        # the vocabulary projection stays whole on every rank: its input (the residual stream) is replicated, so every
        # rank gets the full logits and picks the same token without any exchange (70 MB of weights per step at 7B size)
        self.head = (head.packed_weight, head.weight_scales)
        inv_freq = base.rotary_emb.inv_freq.to(self.dev)
        scaling = float(getattr(base.rotary_emb, "attention_scaling", 1.0))
        self.page_size = page_size
        if page_size is None:
            if max_prefix:
                raise ValueError("a shared prefix needs paged caches (page_size)")
            # rotary tables as the model computes them (float32 angles, cast to the activations' dtype)
            ang = torch.arange(max_len, device=self.dev).float()[:, None] * inv_freq.float()[None, :]
            emb = torch.cat([ang, ang], -1)
            self.cos, self.sin = (emb.cos() * scaling).to(torch.bfloat16), (emb.sin() * scaling).to(torch.bfloat16)
            kv_shape = (max_batch, self.kv_l, max_len, self.head_dim)
            self.k_cache = [torch.zeros(kv_shape, dtype=torch.bfloat16, device=self.dev) for _ in self.layers]
            self.v_cache = [torch.zeros(kv_shape, dtype=torch.bfloat16, device=self.dev) for _ in self.layers]
        else:
            self.inv_freq, self.rope_scaling = inv_freq.double(), scaling
            own, shared = -(-max_len // page_size), -(-max_prefix // page_size)
            total = max(max_batch * own + shared, 1)
            self.pages = [_serving.PagedKVCache(total, page_size, self.kv_l, self.head_dim, torch.bfloat16, self.dev) for _ in self.layers]
            ids = torch.arange(total, dtype=torch.int32, device=self.dev)
            self.table, self.prefix_pages = ids[:max_batch * own].view(max_batch, own), ids[max_batch * own:]
            self.lens = torch.zeros(max_batch, dtype=torch.int32, device=self.dev)          # own tokens of every sequence in the cache
            self.prefix_len = torch.zeros(1, dtype=torch.int32, device=self.dev)
        self.max_prefix = max_prefix
        self.sampling, self.u = None, torch.zeros(max_batch, device=self.dev)
        self.chain = _gemm.FusedChain(self.dev)
        # two peer-visible partial buffers serve all layers: the o and down sums alternate, so a buffer is never used
        # twice in a row and the "everybody has finished reading" handshake can be skipped
        self.peers = None
        if w > 1:
            self.peers = (_PeerSum(group), _PeerSum(group))
            for p in self.peers:
                p.interleaved = True
        self.pos = torch.zeros(1, dtype=torch.int64, device=self.dev)
        self.ids = torch.zeros(max_batch, dtype=torch.int64, device=self.dev)
        self.graph = None

    # ------------------------------------------------------------------------------------------------
    def _row_parallel(self, weight, which, M):
        """GEMM of a row-parallel layer into the chain's buffer (one rank) or this rank's peer-visible partial."""
        if self.world == 1:
            self.chain.gemm(*weight)
            return None
        peer = self.peers[which]
        part = peer.partial_view(M, self.hidden, self.dev)
        if part is None:
            raise _capi.MXFP4BackendError("mxfp4: the decoder's tensor parallelism needs the peer-memory reduction (symmetric memory)")
        self.chain.gemm(*weight, out=part)
        return peer

    def _rope(self, x, cos, sin):
        half = x.shape[-1] // 2
        rot = torch.cat((-x[..., half:], x[..., :half]), dim=-1)
        return x * cos + rot * sin

    def _paged_plan(self, B, T, batch0, prefix):
        """What rope_append and paged_attention need besides the tensors, the same for every layer."""
        n = torch.arange(T, device=self.dev)
        p = dict(q_starts=None, prefix_pages=None, prefix_len=None)
        if prefix:                                    # the prefix itself, as one sequence on the shared pages
            table, place, p["lens"] = self.prefix_pages[None], n[None], torch.full((1,), T, dtype=torch.int32, device=self.dev)
            p["positions"] = n
        else:
            table = self.table[batch0:batch0 + B]
            if T > 1:
                place, p["lens"] = n[None].expand(B, T), torch.full((B,), T, dtype=torch.int32, device=self.dev)
            else:
                place = self.lens[batch0:batch0 + B, None]
                p["lens"] = self.lens[batch0:batch0 + B] + 1
            p["positions"] = (place + self.prefix_len).reshape(-1).long()
            if self.max_prefix:
                p.update(prefix_pages=self.prefix_pages, prefix_len=self.prefix_len)
        if T > 1:
            p["q_starts"] = torch.arange(B + 1, dtype=torch.int32, device=self.dev) * T
        p["table"], p["slots"] = table, self.pages[0].slots(table, place).reshape(-1)
        return p

    def _attend_paged(self, li, qkv, plan):
        M, D, nq = qkv.shape[0], self.head_dim, self.h_l * self.head_dim
        q, k = qkv[:, :nq].view(M, self.h_l, D), qkv[:, nq:nq + self.kv_l * D].view(M, self.kv_l, D)
        v, cache = qkv[:, nq + self.kv_l * D:].view(M, self.kv_l, D), self.pages[li]
        q = _serving.rope_append(q, k, v, cache.k, cache.v, plan["positions"], plan["slots"], self.inv_freq, scaling=self.rope_scaling, q_out=q)
        att = _serving.paged_attention(q, cache.k, cache.v, plan["table"], plan["lens"], q_starts=plan["q_starts"], prefix_pages=plan["prefix_pages"],
                                       prefix_len=plan["prefix_len"])
        return att.view(M, nq)

    def _forward(self, ids, T, pos0=None, batch0=0, prefix=False):
        """Logits of the LAST position of every sequence: ids [B, T]; T > 1 is a prefill from position 0 (written into
        cache rows batch0..batch0+B), T == 1 a decode step at the device-side position self.pos (paged: behind each
        sequence's own tokens) for the whole batch.  prefix: ids [1, T] are the shared prefix."""
        c = self.chain
        c.src = None                                  # the first step of a pass has no GEMM in front
        B = ids.shape[0]
        M = B * T
        hid = self.embed.index_select(0, ids.reshape(-1)).to(torch.bfloat16)       # [M, hidden]: the residual stream
        if self.page_size is not None:
            plan = self._paged_plan(B, T, batch0, prefix)
        elif T > 1:
            cos, sin = self.cos[:T][None, None], self.sin[:T][None, None]
        else:
            cos, sin = self.cos.index_select(0, self.pos)[None, None], self.sin.index_select(0, self.pos)[None, None]
            mask = (torch.arange(self.S, device=self.dev) <= self.pos)[None, None, None, :]
        nq, nkv, D = self.h_l * self.head_dim, self.kv_l * self.head_dim, self.head_dim
        qkv = torch.empty(M, nq + 2 * nkv, dtype=torch.bfloat16, device=self.dev)
        peer_prev = None
        for li, L in enumerate(self.layers):
            c.act(_capi.ACT_RMSNORM, M, self.hidden, residual=hid, hidden_out=hid, gamma=L["g1"], eps=self.eps, peer=peer_prev)
            c.gemm(*L["qkv"], out=qkv)
            if self.page_size is None:
                q = qkv[:, :nq].view(B, T, self.h_l, D).transpose(1, 2)
                k = qkv[:, nq:nq + nkv].view(B, T, self.kv_l, D).transpose(1, 2)
                v = qkv[:, nq + nkv:].view(B, T, self.kv_l, D).transpose(1, 2)
                q, k = self._rope(q, cos, sin), self._rope(k, cos, sin)
            if self.page_size is not None:
                att = self._attend_paged(li, qkv, plan)
            elif T > 1:
                self.k_cache[li][batch0:batch0 + B, :, :T] = k
                self.v_cache[li][batch0:batch0 + B, :, :T] = v
                att = F.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=self.h_l != self.kv_l)
            else:
                kc, vc = self.k_cache[li][:B], self.v_cache[li][:B]      # the batch may be smaller than the cache
                kc.index_copy_(2, self.pos, k)
                vc.index_copy_(2, self.pos, v)
                att = F.scaled_dot_product_attention(q, kc, vc, attn_mask=mask, enable_gqa=self.h_l != self.kv_l)
            c.feed(att if self.page_size is not None else att.transpose(1, 2).reshape(M, nq))
            c.act(_capi.ACT_IDENTITY, M, nq)
            peer_o = self._row_parallel(L["o"], 0, M)
            c.act(_capi.ACT_RMSNORM, M, self.hidden, residual=hid, hidden_out=hid, gamma=L["g2"], eps=self.eps, peer=peer_o)
            n = c.gemm(*L["gateup"])
            c.act(_capi.ACT_SILU_MUL, M, n // 2)
            peer_prev = self._row_parallel(L["down"], 1, M)
        c.act(_capi.ACT_RMSNORM, M, self.hidden, residual=hid, hidden_out=hid, gamma=self.g_final, eps=self.eps, peer=peer_prev,
              quantize=(T == 1))
        if T > 1:
            # only the last position of every sequence feeds the vocabulary projection
            last = hid.view(B, T, self.hidden)[:, -1]
            x = (self.g_final * F.rms_norm(last.float(), (self.hidden,), eps=self.eps).to(torch.bfloat16)).contiguous()
            c.feed(x)
            c.act(_capi.ACT_IDENTITY, B, self.hidden)
        logits = torch.empty(B, self.vocab, dtype=torch.bfloat16, device=self.dev)
        c.gemm(*self.head, out=logits)
        return logits

    def _next_tokens(self, logits, b0=0):
        if self.sampling is None:
            return logits.float().argmax(dim=-1)
        at = slice(b0, b0 + logits.shape[0])
        heat, most, mass, least = (t[at] for t in self.sampling)
        return _serving.sample_tokens(logits, self.u[at], temperature=heat, top_k=most, top_p=mass, min_p=least)

    def set_sampling(self, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        """Tokens are drawn by sample_tokens() from here on: each setting a number, or a tensor with one value per sequence
        (temperature 0: greedy).  prefill() and decode() then take the uniform numbers.  temperature=None: greedy again, by argmax."""
        if temperature is None:
            self.sampling, self.graph = None, None
            return
        values = [torch.as_tensor(v, dtype=d, device=self.dev).expand(self.B) if not isinstance(v, torch.Tensor) or v.dim() == 0
                  else torch.cat([v.to(self.dev, d), torch.zeros(self.B - len(v), dtype=d, device=self.dev)])
                  for v, d in ((temperature, torch.float32), (top_k, torch.int32), (top_p, torch.float32), (min_p, torch.float32))]
        if self.sampling is None:
            self.sampling, self.graph = [v.clone() for v in values], None
        else:                                         # a captured step reads these tensors
            for mine, v in zip(self.sampling, values):
                mine.copy_(v)

    def _uniforms(self, uniforms, shape, name):
        if self.sampling is None:
            return None
        if uniforms is None or tuple(uniforms.shape) != shape:
            raise ValueError(f"{name}() draws tokens (set_sampling) and needs uniforms of shape {shape}")
        return uniforms.to(self.dev, torch.float32)

    @torch.no_grad()
    def set_prefix(self, prefix_ids: torch.Tensor):
        """Fills the shared pages with the prefix [P] that every sequence of the next prefill() continues; an empty one: none."""
        if self.page_size is None:
            raise ValueError("a shared prefix needs paged caches (page_size)")
        P = prefix_ids.numel()
        if P > self.max_prefix:
            raise ValueError(f"a prefix of {P} tokens, room for {self.max_prefix}")
        self.lens.zero_()                             # what the caches held behind another prefix means nothing now
        self.prefix_len.zero_()
        if P:
            self._forward(prefix_ids.reshape(1, -1).to(self.dev), P, prefix=True)
        self.prefix_len.fill_(P)

    @torch.no_grad()
    def prefill(self, prompt_ids: torch.Tensor, chunk: int = 16, uniforms: Optional[torch.Tensor] = None):
        """Fills the KV cache from the prompts [B, T] (sequence chunks bound the activation buffers) and returns the first
        generated token of every sequence.  uniforms: [B], where tokens are drawn."""
        B, T = prompt_ids.shape
        assert B <= self.B and T < self.S
        u = self._uniforms(uniforms, (B,), "prefill")
        if u is not None:
            self.u[:B].copy_(u)
        if self.page_size is not None:
            self.lens.zero_()
        out = []
        for b0 in range(0, B, chunk):
            ids = prompt_ids[b0:b0 + chunk].to(self.dev)
            out.append(self._next_tokens(self._forward(ids, T, batch0=b0), b0))
        self.pos.fill_(T)
        if self.page_size is not None:
            self.lens[:B].fill_(T)
        if getattr(self, "nb", None) != B:
            self.graph = None                      # a captured decode step is tied to its batch size
        self.nb, self.used = B, T
        nxt = torch.cat(out)
        self.ids[:B].copy_(nxt)
        return nxt

    @torch.no_grad()
    def _step(self):
        nxt = self._next_tokens(self._forward(self.ids[:self.nb, None], 1))
        self.ids[:self.nb].copy_(nxt)
        self.pos.add_(1)
        if self.page_size is not None:
            self.lens[:self.nb].add_(1)
        return nxt

    @torch.no_grad()
    def decode(self, new_tokens: int, use_graph: bool = True, uniforms: Optional[torch.Tensor] = None):
        """Decoding after prefill(): returns [B, new_tokens] (the first column is prefill's token).  uniforms: [B, new_tokens - 1],
        where tokens are drawn."""
        toks = [self.ids[:self.nb].clone()]
        u = self._uniforms(uniforms, (self.nb, new_tokens - 1), "decode") if new_tokens > 1 else None
        if new_tokens <= 1:
            return torch.stack(toks, 1)
        if self.used + new_tokens - 1 > self.S:
            raise ValueError(f"{self.used} tokens in the cache and {new_tokens - 1} steps: room for {self.S}")
        self.used += new_tokens - 1
        if use_graph and self.graph is None:
            # one eager step allocates every buffer (and sets up the peer buffers) before the capture
            keep = [t for t in (self.pos, self.ids, self.lens if self.page_size is not None else None) if t is not None]
            held = [t.clone() for t in keep]
            side = torch.cuda.Stream(self.dev)
            side.wait_stream(torch.cuda.current_stream(self.dev))
            with torch.cuda.stream(side):
                self._step()
                for t, v in zip(keep, held):
                    t.copy_(v)
                torch.cuda.synchronize(self.dev)
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=side):
                    self._graph_out = self._step()
            torch.cuda.current_stream(self.dev).wait_stream(side)
            for t, v in zip(keep, held):
                t.copy_(v)
            self.graph = g
        for i in range(new_tokens - 1):
            if u is not None:
                self.u[:self.nb].copy_(u[:, i])
            if use_graph:
                self.graph.replay()
                toks.append(self._graph_out.clone())
            else:
                toks.append(self._step().clone())
        return torch.stack(toks, 1)

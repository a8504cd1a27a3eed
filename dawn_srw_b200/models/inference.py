"""Inference and analysis API of the SRW models.

Functions (reference: models/dawn_spatial_v41_exp.py — prefill/decode_step
:1772-1957, vectorized_eval :1964-2070, vectorized_neuron_health and
vectorized_weight_analysis :2073-2133, analysis_forward :2136-2243,
build_suppressed_forward :2246-2338):

* ``prefill(model, ids)`` -> ``(logits [B,S,V], cache_K, cache_V, S)`` with
  caches ``[L, B, H, max_seq, d_head]``;
* ``decode_step(model, tok, cache_K, cache_V, length)`` -> ``(logits [B,V],
  cache_K, cache_V, length + 1)``;
* ``generate(model, ids, ...)``: KV-cache sampler with temperature / top-k;
* ``PagedSession(model, max_seqs, ...)``: sequences of their own lengths over one paged cache (bf16, e4m3 or
  int8), prompts in chunks, single tokens in a CUDA graph, an optional attention window with sinks (no
  counterpart in the reference, whose caches are dense, fp32 and of one length for the batch);
* ``vectorized_eval(model, batches)`` -> ``(avg_loss, ppl, acc %, n_valid)``;
  note its valid mask is ``label > 0`` (pad id 0), unlike training's
  ``label != -100`` — kept as in the reference and documented;
* ``analysis_forward(model, ids, mode)``: per-layer gates ``[L,B,S,N]``
  (normalised; ``mode='full'`` adds raw) and per-layer output norms;
* ``build_suppressed_forward(model, masks)`` -> ``forward_fn(ids) -> logits``
  with per-pool boolean unit masks zeroing gates.  The reference's version of
  this function still evaluates an older gate (z*Phi(z) with sum of z+ as
  denominator) inside its newest model file; here the model's own gate is used;
* ``neuron_health`` / ``weight_analysis``: pool norm statistics, dead counts,
  cosine-similarity and effective-rank summaries.

No dropout, no load-balance terms.  Everything runs through the model's
backend (sm_100a kernels on a GPU, plain torch on CPU).
"""
from __future__ import annotations

import math
from contextlib import contextmanager
from typing import Callable, Dict, Iterable, List, Optional, Tuple

import torch

from ..ops import reference as R
from ..ops.backend import ParallelCtx
from ..ops.paged import PAGE_DTYPES


def _be(model, device):
    return model._backend(device)


def _pools(model, be):
    """Prepared pools (compute copies, Gram statistics) for inference.  They
    depend only on the pool parameters, so they are kept until a parameter
    changes (its autograd version or storage moves) instead of being rebuilt
    for every decoded token."""
    ps = model.neuron_pool
    key = tuple((p.data_ptr(), p._version, p.device) for p in ps.parameters()) + (id(be),)
    hit = getattr(model, "_inference_pools", None)
    if hit is not None and hit[0] == key:
        return hit[1]
    with torch.no_grad():
        pools = model.prepare_pools(be)
    model._inference_pools = (key, pools)
    return pools


def _srw(model, be, x, h, tau, pools, name, *, return_gates=False, unit_mask=None):
    return be.srw(x, h, tau, pools[name], model.gate, pctx=model.pctx(name), want_diag=False,
                  return_gates=return_gates, unit_mask=unit_mask)


def _fast_infer(model, be) -> bool:
    """Forward-only kernels path: unsharded pools on a backend that has it."""
    return hasattr(be, "srw_infer") and model.shard_group is None


def _layer_qkv(model, be, normed, pools, masks=None, return_gates=False):
    """normed [T,D] -> Q,K,V [T,D] (+ gates)."""
    rt, r = model.router, model.d_route
    T = normed.shape[0]
    m = masks or {}
    if hasattr(be, "linear_cat") and not torch.is_grad_enabled():
        h_all, tau_all = be.linear_cat(normed, (rt.proj_attn, rt.tau_attn))
    else:
        h_all = be.linear(normed, rt.proj_attn.weight, rt.proj_attn.bias)
        tau_all = be.linear(normed, rt.tau_attn.weight, rt.tau_attn.bias).float()
    if not m and not return_gates and _fast_infer(model, be):
        q, k = be.srw_infer(normed, h_all[:, :2 * r].reshape(T, 2, r), tau_all[:, 0:2], pools["qk"],
                            model.gate, n_total=model.n_qk, out_scale=model.pool_scale("qk"))
        (v,) = be.srw_infer(normed, h_all[:, 2 * r:].reshape(T, 1, r), tau_all[:, 2:3], pools["v"],
                            model.gate, n_total=model.n_v, out_scale=model.pool_scale("v"))
        return q, k, v, None, None
    rq = _srw(model, be, normed, h_all[:, :2 * r].reshape(T, 2, r), tau_all[:, 0:2], pools, "qk",
              return_gates=return_gates, unit_mask=m.get("qk"))
    rv = _srw(model, be, normed, h_all[:, 2 * r:].reshape(T, 1, r), tau_all[:, 2:3], pools, "v",
              return_gates=return_gates, unit_mask=m.get("v"))
    qs, vs = model.pool_scale("qk"), model.pool_scale("v")
    return rq.route(0) * qs, rq.route(1) * qs, rv.route(0) * vs, rq, rv


def _know(model, be, normed, pools, masks=None, return_gates=False):
    rt = model.router
    T = normed.shape[0]
    if hasattr(be, "linear_cat") and not torch.is_grad_enabled():
        h, tau = be.linear_cat(normed, (rt.proj_know, rt.tau_know))
    else:
        h = be.linear(normed, rt.proj_know.weight, rt.proj_know.bias)
        tau = be.linear(normed, rt.tau_know.weight, rt.tau_know.bias).float()
    if not masks and not return_gates and _fast_infer(model, be):
        (out,) = be.srw_infer(normed, h.reshape(T, 1, model.d_route), tau, pools["know"], model.gate,
                              n_total=model.n_know, out_scale=model.pool_scale("know"))
        return out, None
    res = _srw(model, be, normed, h.reshape(T, 1, model.d_route), tau, pools, "know",
               return_gates=return_gates, unit_mask=(masks or {}).get("know"))
    return res.route(0) * model.pool_scale("know"), res


def _is_dense(model) -> bool:
    return getattr(model, "version", "") == "baseline"


def _dense_layer_cached(model, be, x, lyr, li, cache_k, cache_v, pos0: int, decode: bool):
    """One layer of the dense baseline on x [B,S,D] whose first position is
    ``pos0``; K / V of the new positions are written into the caches
    (reference: vanilla_cached_forward, models/baseline_transformer_jax.py)."""
    import torch.nn.functional as F
    B, S, D = x.shape
    H = model.n_heads
    dh = D // H
    a = lyr.attn
    n = be.layer_norm(x, lyr.norm1.weight, lyr.norm1.bias).reshape(B * S, D)
    heads = lambda t: t.float().reshape(B, S, H, dh).transpose(1, 2)
    q = heads(be.linear(n, a.q_proj.weight, a.q_proj.bias))
    k = heads(be.linear(n, a.k_proj.weight, a.k_proj.bias))
    v = heads(be.linear(n, a.v_proj.weight, a.v_proj.bias))
    cache_k[li, :, :, pos0: pos0 + S] = k
    cache_v[li, :, :, pos0: pos0 + S] = v
    if decode:
        o = R.cached_attention(q, cache_k[li], cache_v[li], pos0 + 1)
    else:
        o = be.attention(q, k, v, 0.0, False)
    o = o.transpose(1, 2).reshape(B * S, D)
    x = x + be.linear(o, a.o_proj.weight, None).reshape(B, S, D)
    n = be.layer_norm(x, lyr.norm2.weight, lyr.norm2.bias).reshape(B * S, D)
    hdn = F.gelu(be.linear(n, lyr.ffn.w_up.weight, lyr.ffn.w_up.bias), approximate="tanh")
    return x + be.linear(hdn, lyr.ffn.w_down.weight, lyr.ffn.w_down.bias).reshape(B, S, D)


def _dense_prefill(model, input_ids):
    B, S = input_ids.shape
    dev = input_ids.device
    be = _be(model, dev)
    L, H, D = model.n_layers, model.n_heads, model.d_model
    cache_k = torch.zeros(L, B, H, model.max_seq_len, D // H, device=dev)
    cache_v = torch.zeros_like(cache_k)
    x = be.embed(input_ids, model.token_emb.weight, model.pos_emb.weight).float()
    for li, lyr in enumerate(model.layers):
        x = _dense_layer_cached(model, be, x, lyr, li, cache_k, cache_v, 0, False)
    x = be.layer_norm(x, model.norm.weight, model.norm.bias)
    return be.logits(x, model.token_emb.weight), cache_k, cache_v, S


def _dense_decode(model, token, cache_k, cache_v, length):
    B = token.shape[0]
    be = _be(model, token.device)
    D = model.d_model
    x = (model.token_emb.weight[token] + model.pos_emb.weight[length]).float().reshape(B, 1, D)
    for li, lyr in enumerate(model.layers):
        x = _dense_layer_cached(model, be, x, lyr, li, cache_k, cache_v, length, True)
    x = be.layer_norm(x, model.norm.weight, model.norm.bias)
    return be.logits(x, model.token_emb.weight)[:, 0], cache_k, cache_v, length + 1


@torch.no_grad()
def prefill(model, input_ids: torch.Tensor):
    B, S = input_ids.shape
    if S > model.max_seq_len:
        raise ValueError(f"Sequence length {S} exceeds max_seq_len")
    if _is_dense(model):
        return _dense_prefill(model, input_ids)
    dev = input_ids.device
    be = _be(model, dev)
    pools = _pools(model, be)
    L, H, D = model.n_layers, model.n_heads, model.d_model
    dh = D // H
    cache_k = torch.zeros(L, B, H, model.max_seq_len, dh, device=dev)
    cache_v = torch.zeros_like(cache_k)
    x = be.embed(input_ids, model.token_emb.weight, model.pos_emb.weight).float()
    heads = lambda t: t.reshape(B, S, H, dh).transpose(1, 2)
    for li, blk in enumerate(model.layers):
        n = be.layer_norm(x, blk.norm1.weight, blk.norm1.bias).reshape(B * S, D)
        q, k, v, _, _ = _layer_qkv(model, be, n, pools)
        if hasattr(be, "prompt_attention"):
            o = be.prompt_attention(q, k, v, cache_k[li], cache_v[li], B, S)
        else:
            qh, kh, vh = heads(q), heads(k), heads(v)
            cache_k[li, :, :, :S] = kh
            cache_v[li, :, :, :S] = vh
            o = be.attention(qh, kh, vh, 0.0, False).transpose(1, 2).reshape(B * S, D)
        x = x + be.linear(o, blk.attn.expand_O.weight, None).reshape(B, S, D)
        n = be.layer_norm(x, blk.norm2.weight, blk.norm2.bias).reshape(B * S, D)
        ko, _ = _know(model, be, n, pools)
        x = x + ko.reshape(B, S, D)
    x = be.layer_norm(x, model.norm.weight, model.norm.bias)
    return be.logits(x, model.token_emb.weight), cache_k, cache_v, S


@torch.no_grad()
def decode_step(model, token: torch.Tensor, cache_k, cache_v, length: int):
    """token [B] (ids of the newest position) -> logits [B,V] for the next one."""
    B = token.shape[0]
    if length >= model.max_seq_len:
        raise ValueError("KV cache is full")
    if _is_dense(model):
        return _dense_decode(model, token, cache_k, cache_v, length)
    dev = token.device
    be = _be(model, dev)
    pools = _pools(model, be)
    H, D = model.n_heads, model.d_model
    dh = D // H
    x = (model.token_emb.weight[token] + model.pos_emb.weight[length]).float().reshape(B, 1, D)
    for li, blk in enumerate(model.layers):
        n = be.layer_norm(x, blk.norm1.weight, blk.norm1.bias).reshape(B, D)
        q, k, v, _, _ = _layer_qkv(model, be, n, pools)
        cache_k[li, :, :, length] = k.reshape(B, H, dh)
        cache_v[li, :, :, length] = v.reshape(B, H, dh)
        o = R.cached_attention(q.reshape(B, H, 1, dh), cache_k[li], cache_v[li], length + 1)
        o = o.reshape(B, D)
        x = x + be.linear(o, blk.attn.expand_O.weight, None).reshape(B, 1, D)
        n = be.layer_norm(x, blk.norm2.weight, blk.norm2.bias).reshape(B, D)
        ko, _ = _know(model, be, n, pools)
        x = x + ko.reshape(B, 1, D)
    x = be.layer_norm(x, model.norm.weight, model.norm.bias)
    return be.logits(x, model.token_emb.weight)[:, 0], cache_k, cache_v, length + 1


class DecodeSession:
    """KV-cache decoding with the whole per-token step captured in a CUDA graph.

    One decoded token is about forty small launches per layer (LayerNorm, router
    GEMMs, statistics, three gate kernels, three split-K write GEMMs, cache
    attention, O projection, ...).  At batch 1 the kernels of the 400M model stream
    about 12 GB of pool weights per token, i.e. a couple of milliseconds of HBM
    time, which is less than the time the host needs to issue those launches one
    by one; a graph replays them in one submission.  For that the step must have
    static shapes and addresses: the position is a device scalar (position
    embedding by ``index_select``, cache write by ``index_copy_``, attention over
    the whole cache under a position mask), the token ids arrive in a fixed buffer.

    ``session = DecodeSession(model, cache_k, cache_v, length)`` after ``prefill``;
    ``logits = session.step(tokens)`` per new token.  On CPU, for the dense baseline
    or with ``use_graph=False`` it runs the same step eagerly."""

    def __init__(self, model, cache_k, cache_v, length: int, use_graph: Optional[bool] = None):
        self.model, self.cache_k, self.cache_v = model, cache_k, cache_v
        dev = cache_k.device
        self.B = cache_k.shape[1]
        self.length = int(length)
        self.tok = torch.zeros(self.B, dtype=torch.long, device=dev)
        self.pos = torch.full((1,), self.length, dtype=torch.long, device=dev)
        self.be = _be(model, dev)
        self.pools = None if _is_dense(model) else _pools(model, self.be)
        if use_graph is None:
            use_graph = dev.type == "cuda" and not _is_dense(model) and _fast_infer(model, self.be)
        self.graph, self.out = None, None
        self.use_graph = bool(use_graph)

    @torch.no_grad()
    def _step_static(self):
        m, be, pools = self.model, self.be, self.pools
        B, H, D = self.B, m.n_heads, m.d_model
        dh = D // H
        x = (m.token_emb.weight.index_select(0, self.tok)
             + m.pos_emb.weight.index_select(0, self.pos)).float().reshape(B, 1, D)
        n_valid = self.pos + 1                                   # cache positions in use
        fused_attn = (hasattr(be, "decode_attention") and self.cache_k.is_cuda
                      and self.cache_k.dtype == torch.float32 and self.cache_k[0].is_contiguous()
                      and dh <= 128)
        for li, blk in enumerate(m.layers):
            n = be.layer_norm(x, blk.norm1.weight, blk.norm1.bias).reshape(B, D)
            q, k, v, _, _ = _layer_qkv(m, be, n, pools)
            if fused_attn:
                o = be.decode_attention(q, k, v, self.cache_k[li], self.cache_v[li], self.pos, H)
            else:
                self.cache_k[li].index_copy_(2, self.pos, k.reshape(B, H, 1, dh).to(self.cache_k.dtype))
                self.cache_v[li].index_copy_(2, self.pos, v.reshape(B, H, 1, dh).to(self.cache_v.dtype))
                o = R.cached_attention(q.reshape(B, H, 1, dh), self.cache_k[li], self.cache_v[li], n_valid)
            x = x + be.linear(o.reshape(B, D), blk.attn.expand_O.weight, None).reshape(B, 1, D)
            n = be.layer_norm(x, blk.norm2.weight, blk.norm2.bias).reshape(B, D)
            ko, _ = _know(m, be, n, pools)
            x = x + ko.reshape(B, 1, D)
        x = be.layer_norm(x, m.norm.weight, m.norm.bias)
        return be.logits(x, m.token_emb.weight)[:, 0]

    @torch.no_grad()
    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """tokens [B] -> logits [B, V] of the next position."""
        if self.length >= self.model.max_seq_len:
            raise ValueError("KV cache is full")
        if not self.use_graph:
            lg, self.cache_k, self.cache_v, self.length = decode_step(
                self.model, tokens, self.cache_k, self.cache_v, self.length)
            return lg
        self.tok.copy_(tokens)
        self.pos.fill_(self.length)
        if self.graph is None:
            # warm up on a side stream (lazy initialisation must not happen during capture),
            # then capture; the warm-up writes the same cache slot the replay writes again
            side = torch.cuda.Stream(device=self.tok.device)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                for _ in range(2):
                    self._step_static()
            torch.cuda.current_stream().wait_stream(side)
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.out = self._step_static()
        self.graph.replay()
        self.length += 1
        return self.out.clone()


class _Watched:
    """A model's parameters and buffers as they are now.  It holds their storages, so that an address is never that of
    another one in the meantime."""

    def __init__(self, model):
        dicts = [d for m in model.modules() for d in (m._modules, m._parameters, m._buffers) if d]
        tensors = [*model.parameters(), *model.buffers()]
        self.sizes = [(d, len(d)) for d in dicts]
        self.links = [(d, k, v) for d in dicts for k, v in d.items()]
        self.seen = [(p, p._version, p.data_ptr()) for p in tensors]
        self.held = [p.detach() for p in tensors]

    def same(self) -> bool:
        """Nothing written to, pointed elsewhere (``p.data = ..``) or replaced since.  Asked for every token: plain
        loops, a third of what a walk over the modules takes."""
        for d, n in self.sizes:
            if len(d) != n:
                return False
        for d, k, v in self.links:
            if d.get(k) is not v:
                return False
        for p, version, address in self.seen:
            if p._version != version or p.data_ptr() != address:
                return False
        return True


class PagedSession:
    """Decoding of up to ``max_seqs`` sequences, each of its own length, over one paged key/value cache.

    Keys and values live in pages ``[n_layers, n_pages, H, page_size, dh]`` in bf16, or as e4m3 / int8 codes
    with an fp32 scale for each position and head (``kv_dtype``); a sequence takes pages from a common pool
    as it grows and gives them back when it is freed.  With ``window`` a token attends to the last
    ``window`` positions and the first ``sinks`` ones only, and pages that no later token can see go back
    to the pool early.

        s = PagedSession(model, max_seqs=8, kv_dtype="e4m3")
        a, b = s.open(), s.open()
        logits = s.extend({a: ids_a, b: ids_b})     # prompts, or further chunks of them: [2, V], last tokens
        logits = s.step({a: tok_a, b: tok_b})       # one token each: a CUDA graph on a GPU
        s.close(a)

    Attention reads what the pages hold, so the logits are those of the rounded cache.  Dense and SRW models;
    pools must not be sharded.  A kernel that gives up (a wait that ran out, a page outside the pool) is reported
    by RuntimeError in the call after the one that launched it, or by ``check()``, which waits for the GPU."""

    def __init__(self, model, max_seqs: int, *, n_pages: Optional[int] = None, page_size: int = 16,
                 kv_dtype: str = "bf16", window: Optional[int] = None, sinks: int = 0,
                 use_graph: Optional[bool] = None):
        if kv_dtype not in PAGE_DTYPES:
            raise ValueError(f"kv_dtype {kv_dtype!r} is none of {sorted(PAGE_DTYPES)}")
        if max_seqs < 1 or page_size < 16 or page_size > 256 or page_size & (page_size - 1):
            raise ValueError("max_seqs must be positive and page_size a power of two from 16 to 256")
        if window is not None and window < 1 or sinks < 0:
            raise ValueError("window must be at least 1 (None: no window), sinks not negative")
        if sinks and window is None:
            raise ValueError("sinks belong to a window")
        if not _is_dense(model) and model.shard_group is not None:
            raise ValueError("a paged session needs unsharded pools")
        self.model, self.page_size, self.window, self.sinks = model, page_size, window, sinks
        dev = model.token_emb.weight.device
        self.be = _be(model, dev)
        L, H = model.n_layers, model.n_heads
        dh = model.d_model // H
        self.width = -(-model.max_seq_len // page_size)
        self.be.paged_supported(H, dh, max_seqs, self.width * page_size)
        n_pages = max_seqs * self.width if n_pages is None else int(n_pages)
        dtype = PAGE_DTYPES[kv_dtype]
        shape = (L, n_pages, H, page_size, dh)
        self.k_pages, self.v_pages = torch.zeros(shape, dtype=dtype, device=dev), torch.zeros(shape, dtype=dtype, device=dev)
        scaled = dtype != torch.bfloat16
        self.k_scale = torch.ones(shape[:4], device=dev) if scaled else None
        self.v_scale = torch.ones(shape[:4], device=dev) if scaled else None
        self._layers = [(self.k_pages[l], self.v_pages[l],
                         dict(k_scale=self.k_scale[l] if scaled else None, v_scale=self.v_scale[l] if scaled else None))
                        for l in range(L)]
        self.free_pages = list(range(n_pages - 1, -1, -1))
        self.pages: List[Optional[List[int]]] = [None] * max_seqs      # of each open sequence; -1: given back
        self.lengths = [0] * max_seqs
        self.max_seqs = max_seqs
        z = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=dev)
        self._table, self._len, self._tok = z(max_seqs, self.width), z(max_seqs), z(max_seqs).long()
        self._graph = self._out = None
        self._pools = self._watched = None
        self.use_graph = dev.type == "cuda" if use_graph is None else bool(use_graph)

    # ---- sequences and pages -------------------------------------------
    def open(self) -> int:
        """A new, empty sequence; its number."""
        for s, p in enumerate(self.pages):
            if p is None:
                self.pages[s], self.lengths[s] = [], 0
                return s
        raise RuntimeError(f"all {self.max_seqs} sequences are open")

    def close(self, seq: int) -> None:
        """The sequence ends; its pages go back to the pool."""
        self._check(seq)
        self.free_pages.extend(p for p in self.pages[seq] if p >= 0)
        self.pages[seq], self.lengths[seq] = None, 0

    def _check(self, seq: int) -> None:
        if not 0 <= seq < self.max_seqs or self.pages[seq] is None:
            raise ValueError(f"sequence {seq} is not open")

    def _check_ids(self, ids: torch.Tensor) -> None:
        """Before anything changes: an index outside the embedding would end the process's use of a GPU."""
        if ids.numel() and bool(((ids < 0) | (ids >= self.model.vocab_size)).any()):
            raise ValueError(f"a token id is outside the vocabulary of {self.model.vocab_size}")

    @contextmanager
    def _grown(self, new: Dict[int, int]):
        """Room for ``new`` tokens of each sequence while what is inside succeeds; an error changes nothing."""
        before = {s: self.lengths[s] for s in new if 0 <= s < self.max_seqs}
        taken = self._grow(new)
        try:
            yield
        except BaseException:
            for s, n in before.items():
                self.lengths[s] = n
                del self.pages[s][-(-n // self.page_size):]
            self.free_pages.extend(reversed(taken))
            raise

    def _grow(self, new: Dict[int, int]) -> List[int]:
        """Room for ``new`` tokens of each sequence, or an error that changes nothing; the pages that it took."""
        need = 0
        for s, n in new.items():
            self._check(s)
            if n < 1:
                raise ValueError(f"sequence {s}: no new token")
            if self.lengths[s] + n > self.model.max_seq_len:
                raise ValueError(f"sequence {s}: {self.lengths[s]} + {n} tokens exceed max_seq_len")
            need += -(-(self.lengths[s] + n) // self.page_size) - len(self.pages[s])
        if need > len(self.free_pages):
            raise RuntimeError(f"paged cache is full: {need} pages wanted, {len(self.free_pages)} free")
        taken = []
        for s, n in new.items():
            self.lengths[s] += n
            while len(self.pages[s]) * self.page_size < self.lengths[s]:
                taken.append(self.free_pages.pop())
                self.pages[s].append(taken[-1])
        return taken

    def _forget(self, seqs) -> None:
        """Pages that no later token sees go back to the pool."""
        if self.window is None:
            return
        first = -(-self.sinks // self.page_size)
        for s in seqs:
            last = max(0, self.lengths[s] + 1 - self.window) // self.page_size      # the next token's first page
            for i in range(first, last):
                if self.pages[s][i] >= 0:
                    self.free_pages.append(self.pages[s][i])
                    self.pages[s][i] = -1

    def _table_of(self, seqs, width: int) -> torch.Tensor:
        t = torch.full((len(seqs), width), -1, dtype=torch.int32)
        for i, s in enumerate(seqs):
            p = self.pages[s] or []
            t[i, : len(p)] = torch.tensor(p, dtype=torch.int32)
        return t

    # ---- forward -------------------------------------------------------
    def _forward(self, x, table, lengths, starts, max_new):
        """Final hidden states [T, D] of packed new tokens x [T, D]."""
        m, be, H = self.model, self.be, self.model.n_heads
        T, D = x.shape
        dh, dense = D // H, _is_dense(m)
        heads = lambda t: t.reshape(T, H, dh)
        for li, blk in enumerate(m.layers):
            kp, vp, scales = self._layers[li]
            n = be.layer_norm(x, blk.norm1.weight, blk.norm1.bias).reshape(T, D)
            if dense:
                q, k, v = (be.linear(n, w.weight, w.bias) for w in (blk.attn.q_proj, blk.attn.k_proj, blk.attn.v_proj))
            else:
                q, k, v, _, _ = _layer_qkv(m, be, n, self._pools)
            be.paged_write(heads(k).float(), heads(v).float(), kp, vp, table, lengths, starts, **scales)
            o = be.paged_attention(heads(q).float(), kp, vp, table, lengths, starts, max_new=max_new,
                                   window=self.window, sinks=self.sinks, **scales).reshape(T, D)
            if dense:
                x = x + be.linear(o, blk.attn.o_proj.weight, None)
                n = be.layer_norm(x, blk.norm2.weight, blk.norm2.bias).reshape(T, D)
                hdn = torch.nn.functional.gelu(be.linear(n, blk.ffn.w_up.weight, blk.ffn.w_up.bias), approximate="tanh")
                x = x + be.linear(hdn, blk.ffn.w_down.weight, blk.ffn.w_down.bias)
            else:
                x = x + be.linear(o, blk.attn.expand_O.weight, None)
                n = be.layer_norm(x, blk.norm2.weight, blk.norm2.bias).reshape(T, D)
                x = x + _know(m, be, n, self._pools)[0]
        return be.layer_norm(x, m.norm.weight, m.norm.bias)

    def _embed(self, ids, pos):
        m = self.model
        return (m.token_emb.weight.index_select(0, ids) + m.pos_emb.weight.index_select(0, pos)).float()

    def _refresh(self) -> None:
        """What is made from the parameters, made again after one was written to or replaced: a captured step reads
        the copies that it was captured with."""
        if self._watched is None or not self._watched.same():
            self._graph = self._out = self._watched = None
            self._pools = None if _is_dense(self.model) else _pools(self.model, self.be)
            self._watched = _Watched(self.model)

    @torch.no_grad()
    def extend(self, new: Dict[int, torch.Tensor], all_logits: bool = False):
        """New tokens (1-D ids) of some sequences, any number each: a prompt, a chunk of one, drafted tokens.
        Logits [len(new), V] of each one's last token, in the order of ``new``; with ``all_logits`` a list of
        [n, V]."""
        if not new:
            raise ValueError("no sequence to extend")
        dev = self._table.device
        ids = {s: torch.as_tensor(t, dtype=torch.long, device=dev).reshape(-1) for s, t in new.items()}
        counts = {s: t.numel() for s, t in ids.items()}
        packed = torch.cat(list(ids.values()))
        self._check_ids(packed)
        with self._grown(counts):
            self._refresh()
            seqs, ns = list(ids), list(counts.values())
            width = max(len(self.pages[s]) for s in seqs)
            table = self._table_of(seqs, width).to(dev)
            lengths = torch.tensor([self.lengths[s] for s in seqs], dtype=torch.int32, device=dev)
            starts = torch.tensor([0] + ns, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(dev)
            pos = torch.cat([torch.arange(self.lengths[s] - n, self.lengths[s]) for s, n in zip(seqs, ns)]).to(dev)
            h = self._forward(self._embed(packed, pos), table, lengths, starts, max(ns))
            if all_logits:
                out = list(self.be.logits(h, self.model.token_emb.weight).split(ns))
            else:
                out = self.be.logits(h[starts[1:].long() - 1].contiguous(), self.model.token_emb.weight)
            self.be.finish_step()
        self._forget(seqs)
        return out

    def _step_static(self):
        pos = (self._len.long() - 1).clamp(min=0)              # an idle slot has no position and attends to nothing
        h = self._forward(self._embed(self._tok, pos), self._table, self._len, None, 1)
        return self.be.logits(h, self.model.token_emb.weight)

    @torch.no_grad()
    def step(self, tokens: Dict[int, int]) -> torch.Tensor:
        """One new token for each of some sequences; logits [len(tokens), V] in their order.  On a GPU the
        whole step, over all ``max_seqs`` slots, is a CUDA graph: sequences come and go between replays."""
        if not tokens:
            raise ValueError("no sequence to extend")
        tokens = {s: int(t) for s, t in tokens.items()}
        self._check_ids(torch.tensor(list(tokens.values())))
        with self._grown({s: 1 for s in tokens}):
            self._refresh()
            dev = self._table.device
            active = list(range(self.max_seqs))
            self._table.copy_(self._table_of(active, self.width))
            self._len.copy_(torch.tensor([self.lengths[s] if s in tokens else 0 for s in active], dtype=torch.int32))
            self._tok.copy_(torch.tensor([tokens.get(s, 0) for s in active]))
            out = self._replay(dev) if self.use_graph else self._step_static()
            out = out[torch.tensor(list(tokens), device=dev)]
            self.be.finish_step()
        self._forget(tokens)
        return out

    def _replay(self, dev) -> torch.Tensor:
        """The captured step, captured first where there is none."""
        if self._graph is None:
            # outside the capture first (lazy initialisation); it writes the slots that the replay writes again
            side = torch.cuda.Stream(device=dev)
            side.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(side):
                for _ in range(2):
                    self._step_static()
            torch.cuda.current_stream(dev).wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = self._step_static()
            self._graph, self._out = graph, out           # only now: a failed capture leaves none
        self._graph.replay()
        return self._out

    def check(self) -> None:
        """Waits for the GPU and raises RuntimeError if a kernel reported a failure."""
        self.be.finish_run()

    @torch.no_grad()
    def dense(self, seqs: Iterable[int]) -> Tuple[torch.Tensor, torch.Tensor]:
        """The caches of some sequences as ``prefill`` returns them: fp32 [L, n, H, max_seq, dh], zeros behind a
        length (sequences without a window, all their pages still there)."""
        seqs = list(seqs)
        for s in seqs:
            self._check(s)
            if any(p < 0 for p in self.pages[s]):
                raise ValueError(f"sequence {s}: pages outside the window are gone")
        dev = self._table.device
        table = self._table_of(seqs, self.width).to(dev)
        lengths = torch.tensor([self.lengths[s] for s in seqs], dtype=torch.int32, device=dev)
        got = [self.be.paged_read(kp, vp, table, lengths, self.model.max_seq_len, dtype=torch.float32, **scales)
               for kp, vp, scales in self._layers]
        return torch.stack([k for k, _ in got]), torch.stack([v for _, v in got])


def sample_token(logits: torch.Tensor, temperature: float = 1.0, top_k: int = 0,
                 top_p: float = 0.0, generator=None) -> torch.Tensor:
    if temperature <= 0:
        return logits.argmax(-1)
    lg = logits.float() / temperature
    if top_k and top_k < lg.shape[-1]:
        kth = lg.topk(top_k, dim=-1).values[..., -1:]
        lg = lg.masked_fill(lg < kth, float("-inf"))
    if top_p and 0.0 < top_p < 1.0:
        srt, idx = lg.sort(dim=-1, descending=True)
        cum = srt.softmax(-1).cumsum(-1)
        drop = cum - srt.softmax(-1) > top_p
        srt = srt.masked_fill(drop, float("-inf"))
        lg = torch.full_like(lg, float("-inf")).scatter(-1, idx, srt)
    return torch.multinomial(lg.softmax(-1), 1, generator=generator).squeeze(-1)


class _PagedBatch:
    """A batch of prompts of one length in a ``PagedSession``, stepped as ``DecodeSession`` is."""

    def __init__(self, model, input_ids, kv_dtype, window, sinks, use_graph, max_new_tokens):
        B, S = input_ids.shape
        if S > model.max_seq_len:
            raise ValueError(f"Sequence length {S} exceeds max_seq_len")
        page = 16
        most = min(model.max_seq_len, S + max_new_tokens)
        self.session = PagedSession(model, B, n_pages=B * -(-most // page), page_size=page, kv_dtype=kv_dtype,
                                    window=window, sinks=sinks, use_graph=use_graph)
        self.seqs = [self.session.open() for _ in range(B)]
        self.first = self.session.extend(dict(zip(self.seqs, input_ids)))
        self.use_graph = self.session.use_graph

    @property
    def length(self) -> int:
        return self.session.lengths[0]

    def step(self, tokens):
        return self.session.step(dict(zip(self.seqs, tokens.tolist())))


@torch.no_grad()
def generate(model, input_ids: torch.Tensor, max_new_tokens: int = 32, temperature: float = 1.0,
             top_k: int = 0, top_p: float = 0.0, stop_ids: Iterable[int] = (), generator=None,
             use_graph: Optional[bool] = None, kv_dtype: Optional[str] = None, window: Optional[int] = None,
             sinks: int = 0) -> Tuple[torch.Tensor, Dict[str, float]]:
    """KV-cache sampling (reference sampler: scripts/analysis/standalone/
    spatial_analysis.py:444-546).  Returns the full sequences and tokens/s.  With ``kv_dtype`` (bf16, e4m3,
    int8) or ``window`` the caches are paged (``PagedSession``), otherwise dense and fp32."""
    import time
    model.eval()
    if kv_dtype is not None or window is not None:
        session = _PagedBatch(model, input_ids, kv_dtype or "bf16", window, sinks, use_graph, max_new_tokens)
        first = session.first
    else:
        if sinks:
            raise ValueError("sinks belong to a window")
        logits, ck, cv, length = prefill(model, input_ids)
        session = DecodeSession(model, ck, cv, length, use_graph=use_graph)
        first = logits[:, -1]
    out = [input_ids]
    nxt = sample_token(first, temperature, top_k, top_p, generator)
    stop = set(int(s) for s in stop_ids)
    sync = torch.cuda.synchronize if input_ids.is_cuda else (lambda: None)
    t0, n, t1 = time.perf_counter(), 0, None
    for _ in range(max_new_tokens):
        out.append(nxt[:, None])
        n += 1
        if session.length >= model.max_seq_len or (stop and all(int(t) in stop for t in nxt)):
            break
        lg = session.step(nxt)
        nxt = sample_token(lg, temperature, top_k, top_p, generator)
        if t1 is None:                 # the first step carries the graph capture
            sync()
            t1 = time.perf_counter()
    sync()
    t2 = time.perf_counter()
    _be(model, input_ids.device).finish_run()          # raises if a kernel gave up
    B = input_ids.shape[0]
    stats = {"new_tokens": n, "tokens_per_sec": n * B / max(t2 - t0, 1e-9),
             "first_step_s": (t1 - t0) if t1 is not None else 0.0, "graph": session.use_graph}
    if t1 is not None and n > 2:
        stats["steady_tokens_per_sec"] = (n - 2) * B / max(t2 - t1, 1e-9)
    return torch.cat(out, dim=1), stats


@torch.no_grad()
def vectorized_eval(model, batches: Iterable[torch.Tensor]):
    """(avg_loss, ppl, accuracy %, n_valid) over ``batches`` of token ids; sums
    stay on the device until the end.  Valid positions are ``label > 0``."""
    model.eval()
    tot = None
    for ids in batches:
        ids = ids.long()
        labels = torch.where(ids > 0, ids, torch.full_like(ids, -100))
        r = model(ids, labels=labels, want_diag=False)
        cur = torch.stack([r["loss"].double() * r["valid_count"], r["correct"].double(),
                           r["valid_count"].double()])
        tot = cur if tot is None else tot + cur
    if tot is None:
        return 0.0, 1.0, 0.0, 0
    loss_sum, correct, valid = tot.tolist()
    avg = loss_sum / max(valid, 1.0)
    return avg, math.exp(min(avg, 50.0)), 100.0 * correct / max(valid, 1.0), int(valid)


@torch.no_grad()
def analysis_forward(model, input_ids: torch.Tensor, mode: str = "light") -> Dict[str, torch.Tensor]:
    """Forward that also returns the gates of every layer.

    ``gate_{Q,K,V,Know}``: [L, B, S, N] gate / sum(gate); with ``mode='full'``
    also ``gate_*_raw``.  ``attn_out_norm`` / ``know_out_norm``: [L]."""
    model.eval()
    B, S = input_ids.shape
    dev = input_ids.device
    be = _be(model, dev)
    pools = _pools(model, be)
    H, D = model.n_heads, model.d_model
    dh = D // H
    x = be.embed(input_ids, model.token_emb.weight, model.pos_emb.weight).float()
    heads = lambda t: t.reshape(B, S, H, dh).transpose(1, 2)
    names = ("Q", "K", "V", "Know")
    norm_g: Dict[str, List] = {n: [] for n in names}
    raw_g: Dict[str, List] = {n: [] for n in names}
    a_norms, k_norms = [], []

    def keep(name, g):                       # g [T, U]
        g = g.reshape(B, S, -1).float()
        norm_g[name].append(g / g.sum(-1, keepdim=True).clamp(min=1e-8))
        if mode == "full":
            raw_g[name].append(g)
    for blk in model.layers:
        n = be.layer_norm(x, blk.norm1.weight, blk.norm1.bias).reshape(B * S, D)
        q, k, v, rq, rv = _layer_qkv(model, be, n, pools, return_gates=True)
        keep("Q", rq.gates[:, 0]); keep("K", rq.gates[:, 1]); keep("V", rv.gates[:, 0])
        o = be.attention(heads(q), heads(k), heads(v), 0.0, False).transpose(1, 2).reshape(B * S, D)
        ao = be.linear(o, blk.attn.expand_O.weight, None)
        a_norms.append(torch.linalg.vector_norm(ao.float(), dim=-1).mean())
        x = x + ao.reshape(B, S, D)
        n = be.layer_norm(x, blk.norm2.weight, blk.norm2.bias).reshape(B * S, D)
        ko, rk = _know(model, be, n, pools, return_gates=True)
        keep("Know", rk.gates[:, 0])
        k_norms.append(torch.linalg.vector_norm(ko.float(), dim=-1).mean())
        x = x + ko.reshape(B, S, D)
    x = be.layer_norm(x, model.norm.weight, model.norm.bias)
    out = {"logits": be.logits(x, model.token_emb.weight),
           "attn_out_norm": torch.stack(a_norms), "know_out_norm": torch.stack(k_norms)}
    for nme in names:
        out[f"gate_{nme}"] = torch.stack(norm_g[nme])
        if mode == "full":
            out[f"gate_{nme}_raw"] = torch.stack(raw_g[nme])
    return out


def build_suppressed_forward(model, masks: Dict[str, torch.Tensor]) -> Callable[[torch.Tensor], torch.Tensor]:
    """``masks``: {'qk' | 'v' | 'know': bool [N]} with True = unit is suppressed.
    Returns ``forward_fn(ids) -> logits`` with those units' gates forced to zero."""
    keep = {k: (~v.bool()).float() for k, v in masks.items()}

    @torch.no_grad()
    def forward_fn(input_ids: torch.Tensor) -> torch.Tensor:
        model.eval()
        B, S = input_ids.shape
        dev = input_ids.device
        be = _be(model, dev)
        pools = _pools(model, be)
        km = {k: v.to(dev) for k, v in keep.items()}
        H, D = model.n_heads, model.d_model
        dh = D // H
        heads = lambda t: t.reshape(B, S, H, dh).transpose(1, 2)
        x = be.embed(input_ids, model.token_emb.weight, model.pos_emb.weight).float()
        for blk in model.layers:
            n = be.layer_norm(x, blk.norm1.weight, blk.norm1.bias).reshape(B * S, D)
            q, k, v, _, _ = _layer_qkv(model, be, n, pools, masks=km)
            o = be.attention(heads(q), heads(k), heads(v), 0.0, False).transpose(1, 2).reshape(B * S, D)
            x = x + be.linear(o, blk.attn.expand_O.weight, None).reshape(B, S, D)
            n = be.layer_norm(x, blk.norm2.weight, blk.norm2.bias).reshape(B * S, D)
            ko, _ = _know(model, be, n, pools, masks=km)
            x = x + ko.reshape(B, S, D)
        x = be.layer_norm(x, model.norm.weight, model.norm.bias)
        return be.logits(x, model.token_emb.weight)
    return forward_fn


@torch.no_grad()
def neuron_health(model, dead_norm: float = 1e-6) -> Dict[str, float]:
    """Norm statistics and dead counts per pool tensor, tau biases."""
    out: Dict[str, float] = {}
    p = model.neuron_pool
    for name in ("qk", "v", "know"):
        n = p.n_valid(name)
        for kind in ("emb", "read", "write"):
            norms = torch.linalg.vector_norm(getattr(p, f"{name}_{kind}")[:n].float(), dim=-1)
            key = f"{name}_{kind}"
            out[f"{key}_norm_mean"] = float(norms.mean())
            out[f"{key}_norm_min"] = float(norms.min())
            out[f"{key}_norm_max"] = float(norms.max())
            out[f"{key}_norm_std"] = float(norms.std(unbiased=False))
            out[f"{key}_dead"] = int((norms < dead_norm).sum())
        if model.gate.learnable_scale:
            out[f"{name}_scale"] = float(getattr(p, f"{name}_scale")[0])
    rt = model.router
    out["tau_know_bias"] = float(rt.tau_know.bias[0])
    for i, nm in enumerate("qkv"):
        out[f"tau_attn_bias_{nm}"] = float(rt.tau_attn.bias[i])
    return out


@torch.no_grad()
def weight_analysis(model, max_rows: int = 2048) -> Dict[str, float]:
    """Cosine-similarity summary (at most ``max_rows`` stride-sampled rows) and
    SVD effective rank (exp of the singular-value entropy) per pool tensor."""
    out: Dict[str, float] = {}
    p = model.neuron_pool
    for name in ("qk", "v", "know"):
        n = p.n_valid(name)
        for kind in ("emb", "read", "write"):
            w = getattr(p, f"{name}_{kind}")[:n].float()
            if w.shape[0] > max_rows:
                w = w[:: w.shape[0] // max_rows][:max_rows]
            u = w / (torch.linalg.vector_norm(w, dim=-1, keepdim=True) + 1e-8)
            sim = u @ u.t()
            m = sim.shape[0]
            off = sim - torch.diag(torch.diagonal(sim))
            key = f"{name}_{kind}"
            out[f"{key}_cos_abs_mean"] = float(off.abs().sum() / (m * m - m))
            out[f"{key}_cos_max"] = float(off.max())
            sv = torch.linalg.svdvals(w.cpu())
            ps = sv / sv.sum()
            out[f"{key}_effective_rank"] = float(torch.exp(-(ps * torch.log(ps + 1e-12)).sum()))
    return out


def estimate_flops_per_token(model, seq_len: Optional[int] = None) -> Dict[str, float]:
    """Forward FLOPs per token (reference estimator: spatial_analysis.py:247-256);
    scores are counted once here (the Gram-matrix statistics need no second pass)."""
    D, r, L, H = model.d_model, model.d_route, model.n_layers, model.n_heads
    S = seq_len or model.max_seq_len
    nq, nv, nk = model.n_qk, model.n_v, model.n_know
    scores = 2 * r * (2 * nq + nv + nk)
    read = 2 * D * (nq + nv + nk)
    write = 2 * D * (2 * nq + nv + nk)
    attn = 4 * S * D / 2 + 2 * D * D
    router = 2 * D * (4 * r + 4)
    per_layer = scores + read + write + attn + router
    head = 2 * D * model.vocab_size
    return {"per_layer": per_layer, "lm_head": head, "total": L * per_layer + head}

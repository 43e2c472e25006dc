"""Greedy-decode harness for a full quantized decoder (Qwen3-32B shape by
default): every decoder linear is a QuantizedLinear with random E8P codes,
the rest of the model (embeddings, norms, rotary tables, lm_head) is the
transformers implementation in bf16 with random weights.  Built on the meta
device and materialized on the GPU, so the 32B-parameter model never exists
densely.  Decoding runs through StaticDecoder (static bf16 KV cache, device
positions, the decode step's own kernels around the quantized linears) so
that each step is one HIP-graph replay.  Reports
prefill time, decode tok/s and, per decoder linear of the first layer, the
forward time and HBM GB/s at each batch size.

    python -m quipsharp_amd.decode --batch 1 8 --prompt 512 --new 256
"""
import argparse
import json
import time

import torch
from torch import nn

from .architectures import get_decoder_layers, get_linear_groups
from .checkpoint import (QuantizedLinear, build_codebook, grouped_forward, grouped_forward_pre,
                         link_sibling_linears, run_preop)
from .hadamard import is_pow2, kron_factor, rademacher

QWEN3_32B = dict(hidden_size=5120, intermediate_size=25600, num_hidden_layers=64, num_attention_heads=64,
                 num_key_value_heads=8, head_dim=128, vocab_size=151936, max_position_embeddings=40960,
                 rms_norm_eps=1e-6, tie_word_embeddings=False)


def _random_qlinear(lin, device, gen, cpu_gen, scale=0.0135):
    n, m = lin.in_features, lin.out_features
    kind = "rht" if is_pow2(n) and is_pow2(m) else "krht"
    if kind == "krht" and (kron_factor(n) is None or kron_factor(m) is None):
        raise ValueError(f"no transform for a {m} x {n} linear")
    q = QuantizedLinear(n, m, 8, kind, has_bias=getattr(lin, "bias", None) is not None)
    q = q.to(device)
    with torch.no_grad():
        q.codes.copy_(torch.randint(-32768, 32768, q.codes.shape, generator=gen, device=device, dtype=torch.int32)
                      .to(torch.int16))
        q.scale.fill_(scale)
        q.su.copy_(rademacher(m, device=device, generator=cpu_gen))
        q.sv.copy_(rademacher(n, device=device, generator=cpu_gen))
        if q.bias is not None:
            q.bias.zero_()
    return q


def random_quantized_model(config, device="cuda", seed=0):
    """transformers causal LM of ``config`` with every decoder linear replaced
    by a random-code QuantizedLinear (linear discovery as
    architectures.get_linear_groups) and random bf16 for the rest."""
    from transformers import AutoModelForCausalLM
    with torch.device("meta"):
        model = AutoModelForCausalLM.from_config(config, dtype=torch.bfloat16)
    gen = torch.Generator(device=device).manual_seed(seed)
    cpu_gen = torch.Generator().manual_seed(seed)
    codebook, _ = build_codebook("2bit", device, seed)
    for i, layer in enumerate(get_decoder_layers(model)):
        for group in get_linear_groups(layer, i):
            for name, lin in group:
                parent_name, _, attr = name.rpartition(".")
                parent = layer.get_submodule(parent_name)
                q = _random_qlinear(lin, device, gen, cpu_gen)
                q.codebook = codebook
                setattr(parent, attr, q)
    # everything still on the meta device gets fresh storage on the GPU
    for mod in model.modules():
        if hasattr(mod, "inv_freq") and getattr(mod, "inv_freq").is_meta:
            fresh = type(mod)(config=mod.config)
            for k, v in fresh.named_buffers(recurse=False):
                setattr(mod, k, v.to(device))
            if hasattr(fresh, "attention_scaling"):
                mod.attention_scaling = fresh.attention_scaling
            continue
        for k, p in list(mod.named_parameters(recurse=False)):
            if p.is_meta:
                if "norm" in type(mod).__name__.lower():
                    t = torch.ones(p.shape, dtype=p.dtype, device=device)
                else:
                    t = torch.randn(p.shape, generator=gen, dtype=torch.float32, device=device).mul_(0.02)
                    t = t.to(p.dtype)
                setattr(mod, k, nn.Parameter(t, requires_grad=False))
        for k, b in list(mod.named_buffers(recurse=False)):
            if b is not None and b.is_meta:
                setattr(mod, k, torch.zeros(b.shape, dtype=b.dtype, device=device))
    model.eval()
    link_sibling_linears(model)
    return model


@torch.no_grad()
def greedy_decode(model, prompt_ids, new_tokens):
    """Prefill ``prompt_ids`` (B, P), then ``new_tokens`` greedy steps with a
    KV cache, by the model's own forward (no adapters run there).  Returns
    (tokens (B, new_tokens), prefill s, decode s)."""
    from transformers import DynamicCache
    cache = DynamicCache()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    out = model(input_ids=prompt_ids, past_key_values=cache, use_cache=True)
    nxt = out.logits[:, -1].argmax(-1, keepdim=True)
    torch.cuda.synchronize()
    t1 = time.perf_counter()
    toks = [nxt]
    for _ in range(new_tokens - 1):
        out = model(input_ids=nxt, past_key_values=cache, use_cache=True)
        nxt = out.logits[:, -1].argmax(-1, keepdim=True)
        toks.append(nxt)
    torch.cuda.synchronize()
    t2 = time.perf_counter()
    return torch.cat(toks, 1), t1 - t0, t2 - t1


class StaticDecoder:
    """A graph-capturable greedy-decode step for Qwen3-style decoders built on
    the transformers modules of ``model`` (embeddings, RMSNorm and q/k-norm
    weights, rotary tables, lm_head) and its QuantizedLinear layers, with a
    static bf16 KV cache of ``max_len`` positions per layer and the position
    passed as a device tensor, so one decode step can be captured once and
    replayed.

    A decode step (one new token per row) runs the layer's own kernels
    (csrc/qs_decoder.hip): q/k norm plus rotary embedding plus the cache
    write in one launch, attention over the filled cache prefix only (splits
    of 64 positions and a combine launch), SiLU * up; q/k/v and gate/up each
    go through one grouped quantized-linear launch that, at one row, also
    does the residual add and the RMSNorm before it
    (checkpoint.grouped_forward_pre; at more rows the norm runs on its own
    launch first).  The prompt
    (several tokens per row), and every step of a model whose activation is
    not SiLU, runs transformers' modules with the same bf16 cache (attention
    in fp32)."""

    def __init__(self, model, batch, max_len, cache=True):
        from . import _lib
        cfg = model.config
        self.model = model
        self.layers = get_decoder_layers(model)
        self.B, self.max_len = batch, max_len
        self.nh, self.nkv = cfg.num_attention_heads, cfg.num_key_value_heads
        self.hd = getattr(cfg, "head_dim", None) or cfg.hidden_size // self.nh
        self.hidden = cfg.hidden_size
        self.eps = float(cfg.rms_norm_eps)
        self.scale = self.hd ** -0.5
        dev = model.lm_head.weight.device
        self.dev = dev
        bf = torch.bfloat16
        if cache:
            if not all(hasattr(L.self_attn, "q_norm") for L in self.layers):
                raise ValueError(f"the static decoder takes layers with q/k norms (Qwen3), not {cfg.model_type}: PagedDecoder "
                                 f"takes Llama and Qwen2 too")
            self.k = [torch.zeros(batch, self.nkv, max_len, self.hd, device=dev, dtype=bf) for _ in self.layers]
            self.v = [torch.zeros(batch, self.nkv, max_len, self.hd, device=dev, dtype=bf) for _ in self.layers]
        self.kpos = torch.arange(max_len, device=dev)
        # rotary tables of every cache position, as transformers computes them
        m = model.model
        with torch.no_grad():
            cos, sin = m.rotary_emb(torch.zeros(1, 1, self.hidden, device=dev, dtype=bf), self.kpos[None])
        self.cos, self.sin = cos[0].to(bf).contiguous(), sin[0].to(bf).contiguous()
        L = _lib.lib()
        self._L, self._lib = L, _lib
        if cache:
            nbytes = L.qs_dec_attention_workspace_bytes(batch, self.nkv, max_len)
            self.attn_ws = torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=dev)
        self.silu = getattr(cfg, "hidden_act", "silu") in ("silu", "swish")  # what the decode step computes
        self.fused_ok = self.hd == 128 and self.nh % self.nkv == 0 and self.nh // self.nkv <= 16 \
            and self.hidden % 8 == 0 and self.silu

    def _weight(self, mod):
        w = mod.weight
        if w.dtype != torch.bfloat16 or not w.is_contiguous():
            raise TypeError("the decode step takes bf16 norm weights")
        return w

    def _adapted(self):
        return any(getattr(mod, "adapters", None) is not None for L in self.layers for part in (L.self_attn, L.mlp)
                   for mod in part._modules.values())

    @torch.no_grad()
    def step(self, ids, pos):
        """Logits of the last position; ids (B, q), pos (q,) int64 positions."""
        if self._adapted():
            raise ValueError("the static decoder runs no adapters (PagedDecoder does): the model's linears have some")
        if ids.shape[1] == 1 and self.fused_ok:
            return self._decode_step(ids, pos)
        return self._prompt_step(ids, pos)

    def _prompt_step(self, ids, pos):
        from transformers.models.qwen3.modeling_qwen3 import apply_rotary_pos_emb
        import torch.nn.functional as F
        m = self.model.model
        B, q = ids.shape
        h = m.embed_tokens(ids)
        cos, sin = m.rotary_emb(h, pos.unsqueeze(0).expand(B, -1))
        mask = self.kpos[None, :] <= pos[:, None]  # (q, max_len): key j visible to query at pos_i iff j <= pos_i
        for i, L in enumerate(self.layers):
            a = L.self_attn
            x = L.input_layernorm(h)
            qo, ko, vo = grouped_forward(x, [a.q_proj, a.k_proj, a.v_proj])
            qs = a.q_norm(qo.view(B, q, self.nh, self.hd)).transpose(1, 2)
            ks = a.k_norm(ko.view(B, q, self.nkv, self.hd)).transpose(1, 2)
            vs = vo.view(B, q, self.nkv, self.hd).transpose(1, 2)
            qs, ks = apply_rotary_pos_emb(qs, ks, cos, sin)
            self.k[i].index_copy_(2, pos, ks.to(self.k[i].dtype))
            self.v[i].index_copy_(2, pos, vs.to(self.v[i].dtype))
            o = F.scaled_dot_product_attention(qs.float(), self.k[i].float(), self.v[i].float(), attn_mask=mask,
                                               enable_gqa=True)
            h = h + a.o_proj(o.transpose(1, 2).reshape(B, q, self.nh * self.hd).to(h.dtype))
            x = L.post_attention_layernorm(h)
            go, uo = grouped_forward(x, [L.mlp.gate_proj, L.mlp.up_proj])
            h = h + L.mlp.down_proj(L.mlp.act_fn(go) * uo)
        return self.model.lm_head(m.norm(h[:, -1:]))[:, -1]

    def _decode_step(self, ids, pos):
        L, lib = self._L, self._lib
        m = self.model.model
        B = ids.shape[0]
        H, nh, hd = self.hidden, self.nh, self.hd
        stream = lib.stream_of(ids)
        vp = lib.ptr
        h = m.embed_tokens(ids).reshape(B, H)
        if h.dtype != torch.bfloat16:
            raise TypeError("the decode step runs bf16 models")
        h = h.contiguous()
        # the residual stream alternates between two buffers: a norm inside a
        # grouped launch reads h + delta while one work-group writes the sum
        h_alt = torch.empty_like(h)
        attn = torch.empty(B, nh * hd, dtype=torch.bfloat16, device=h.device)
        delta = None
        for i, Ly in enumerate(self.layers):
            a = Ly.self_attn
            # residual add + input norm inside the q/k/v launch (one row; on
            # their own launch otherwise)
            qo, ko, vo = self._normed_linears(h, [a.q_proj, a.k_proj, a.v_proj],
                                              {"kind": "rmsnorm", "delta": delta, "h_out": h_alt, "eps": self.eps,
                                               "weight": self._weight(Ly.input_layernorm)})
            h, h_alt = h_alt, h
            norms = (self._weight(a.q_norm), self._weight(a.k_norm)) if hasattr(a, "q_norm") else None
            self._attend(i, qo.contiguous(), ko.contiguous(), vo.contiguous(), norms, pos, attn, stream)
            o = self._linear(attn, a.o_proj).contiguous()
            go, uo = self._normed_linears(h, [Ly.mlp.gate_proj, Ly.mlp.up_proj],
                                          {"kind": "rmsnorm", "delta": o, "h_out": h_alt, "eps": self.eps,
                                           "weight": self._weight(Ly.post_attention_layernorm)})
            h, h_alt = h_alt, h
            go, uo = go.contiguous(), uo.contiguous()
            act = torch.empty_like(go)
            inter = go.shape[-1]
            lib.check(L.qs_dec_silu_mul(vp(go), vp(uo), vp(act), B, inter, inter, inter, inter, stream))
            delta = self._linear(act, Ly.mlp.down_proj).contiguous()
        x = torch.empty_like(h)
        lib.check(L.qs_dec_rmsnorm(vp(h), vp(delta), vp(h), vp(self._weight(m.norm)), vp(x), B, H, H, self.eps, stream))
        return self.model.lm_head(x)

    def _normed_linears(self, h, linears, pre):
        return grouped_forward_pre(h, linears, pre)

    def _linear(self, x, linear):
        return linear(x)

    def _attend(self, i, qo, ko, vo, norms, pos, out, stream):
        """q/k norm, rotary and the cache write inside the attention's launches."""
        L, vp = self._L, self._lib.ptr
        self._lib.check(L.qs_dec_attention_rope(vp(qo), vp(ko), vp(vo), vp(norms[0]), vp(norms[1]), vp(self.cos),
                                                vp(self.sin), vp(pos), vp(self.k[i]), vp(self.v[i]), vp(out),
                                                self.nh * self.hd, vp(self.attn_ws), self.attn_ws.numel(), self.B,
                                                self.nh, self.nkv, self.hd, self.max_len, self.eps, self.scale, stream))


@torch.no_grad()
def greedy_decode_static(model, prompt_ids, new_tokens, use_graph=True):
    """Prefill and greedy decode with StaticDecoder; each decode step replayed
    from one HIP graph unless use_graph=False.  Returns (tokens, prefill s,
    decode s)."""
    B, P = prompt_ids.shape
    dev = prompt_ids.device
    dec = StaticDecoder(model, B, P + new_tokens + 2)
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    tok = dec.step(prompt_ids, torch.arange(P, device=dev)).argmax(-1, keepdim=True)
    torch.cuda.synchronize()
    t1 = time.perf_counter()
    pos = torch.full((1,), P, dtype=torch.long, device=dev)
    toks = [tok.clone()]
    if not use_graph:
        for _ in range(new_tokens - 1):
            tok = dec.step(tok, pos).argmax(-1, keepdim=True)
            pos.add_(1)
            toks.append(tok)
        torch.cuda.synchronize()
        return torch.cat(toks, 1), t1 - t0, time.perf_counter() - t1
    # warm-up (writes position P with the right token, as the first replay will), then capture
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            dec.step(tok, pos)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nxt = dec.step(tok, pos).argmax(-1, keepdim=True)
    torch.cuda.synchronize()
    t2 = time.perf_counter()
    for _ in range(new_tokens - 1):
        graph.replay()
        tok.copy_(nxt)
        pos.add_(1)
        toks.append(nxt.clone())
    torch.cuda.synchronize()
    return torch.cat(toks, 1), t1 - t0, time.perf_counter() - t2


class PagedDecoder(StaticDecoder):
    """StaticDecoder's layers over a paged cache (pages.PagedCache): rows of
    different lengths, prompts that begin while other rows wait, rows that fork
    (beam search) and, with ``window``, streams far longer than what is kept
    visible (the last ``window`` positions and the first ``sinks``; pages that
    fell out are given back).  Everything that a step needs to know of its rows
    lies on the GPU, so a step can be captured once and replayed.

    Layers with q/k norms (Qwen3) have heads of 128; of those without (Llama,
    Qwen2: model types ``llama`` and ``qwen2``) heads of 64, 128 or 256 turn by
    ``rope.append_rotated`` with the config's frequencies, stretched contexts
    included.  Activations are SiLU.  Where linears have adapters (``adapters.attach_adapters``),
    ``which`` (int32 on the GPU, one for every row, -1 for none) says which of
    them a row takes; a captured step follows it, and rows that fork keep it.

    Rows of at most ``max_len`` positions (rounded up to whole pages).  A step
    that runs out of pages or of positions leaves tokens out; it does not wait
    to say so, ``cache.check()`` and the next ``prompt`` raise for it."""

    def __init__(self, model, rows, max_len, page=64, pages=None, window=0, sinks=0):
        from .pages import PagedCache
        columns = -(-max_len // page)
        super().__init__(model, rows, columns * page, cache=False)  # rotary tables to the last page's end
        if not self.silu:
            raise ValueError(f"the paged decode step computes SiLU(gate) * up, the model has {model.config.hidden_act!r}")
        self.normed = all(hasattr(L.self_attn, "q_norm") for L in self.layers)
        if self.normed:
            if not self.fused_ok:
                raise ValueError("the paged decode step takes head_dim 128 and at most 16 query heads per kv head")
        else:
            from .rope import model_frequencies
            cfg = model.config
            if cfg.model_type not in ("llama", "qwen2") or any(hasattr(L.self_attn, "q_norm") for L in self.layers) \
                    or any(t != "full_attention" for t in getattr(cfg, "layer_types", None) or ()):
                raise ValueError(f"the paged decoder takes models of type qwen3, llama and qwen2 whose layers see all of a "
                                 f"row, not {cfg.model_type}")
            if self.hd not in (64, 128, 256) or self.nh % self.nkv or self.nh // self.nkv > 16 or self.hidden % 8:
                raise ValueError(f"the paged decode step takes heads of 64, 128 or 256, at most 16 of them per kv head, got "
                                 f"{self.nh} and {self.nkv} of {self.hd}")
            self.frequencies, self.turn_factor = model_frequencies(cfg, self.dev)
            if 2 * len(self.frequencies) != self.hd:  # their own modules turn whole heads, or fail
                raise ValueError(f"the paged decoder turns whole heads of {cfg.model_type} models, the config has "
                                 f"{2 * len(self.frequencies)} elements of {self.hd} turned")
        self.window, self.sinks = window, sinks
        self.cache = PagedCache(len(self.layers), rows * columns if pages is None else pages, self.nkv, self.hd, rows,
                                columns, page, torch.bfloat16, self.dev)
        self.spans = {"window": window, "sinks": sinks}
        self.which = torch.full((rows,), -1, dtype=torch.int32, device=self.dev)
        self._prompt_which = None  # of a prompt's tokens, while it runs

    def _check_ids(self, ids):
        if ids.device != self.dev or ids.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"ids must be int64 or int32 on {self.dev}, got {ids.dtype} on {ids.device}")

    def _check_beside(self, tokens):
        """Refuses what the layers would refuse of ``which`` and the adapters: before the cache grows, since it keeps what
        it was given room for."""
        from .adapters import check_beside
        dtype = self.model.model.embed_tokens.weight.dtype
        for L in self.layers:
            a, mlp = L.self_attn._modules, L.mlp._modules
            for linears in ((a["q_proj"], a["k_proj"], a["v_proj"]), (a["o_proj"],), (mlp["gate_proj"], mlp["up_proj"]),
                            (mlp["down_proj"],)):
                for linear in linears:
                    if getattr(linear, "adapters", None) is not None:
                        check_beside(linears, self.which, self.B, tokens, dtype, self.dev)
                        break

    def _beside(self, x, linears, outs):
        """The outputs of ``linears`` for x, with the adapters of the tokens' rows."""
        if all(getattr(l, "adapters", None) is None for l in linears):
            return outs
        from .adapters import beside
        flat = [y.reshape(-1, y.shape[-1]) for y in outs]
        which = self.which if self._prompt_which is None else self._prompt_which
        return [f.view(y.shape) for f, y in zip(beside(x.reshape(-1, x.shape[-1]), linears, flat, which), outs)]

    def _normed_linears(self, h, linears, pre):
        if all(getattr(l, "adapters", None) is None for l in linears):
            return grouped_forward_pre(h, linears, pre)
        x = run_preop(h, pre)  # the adapters read the normed rows too
        return self._beside(x, linears, grouped_forward(x, linears))

    def _linear(self, x, linear):
        return self._beside(x, [linear], [linear(x)])[0]

    def _prompt_hidden(self, ids, counts):
        """The last layer's output for all tokens of a prompt call, and the rows' counts."""
        m, cache = self.model.model, self.cache
        T = int(sum(counts))
        if ids.shape != (T,) or len(counts) != self.B:
            raise ValueError(f"ids {tuple(ids.shape)} for {T} tokens in {len(counts)} of {self.B} rows")
        self._check_ids(ids)
        count = torch.tensor(counts, dtype=torch.int32)
        starts = torch.cat([torch.zeros(1, dtype=torch.int32), count.cumsum(0, dtype=torch.int32)]).to(self.dev)
        row = torch.repeat_interleave(torch.arange(self.B), count).to(self.dev)
        self._check_beside(T)
        cache.advance(count.to(self.dev))
        cache.check()
        h = m.embed_tokens(ids)[None]
        if self.normed:
            pos = (cache.lengths + cache.over)[row] - starts[row + 1] + torch.arange(T, device=self.dev)
            cos, sin = m.rotary_emb(h, pos[None])
        self._prompt_which = self.which[row]
        try:
            h = self._prompt_layers(h, starts, (cos, sin) if self.normed else None)
        finally:
            self._prompt_which = None
        if self.window:
            cache.free(window=self.window, sinks=self.sinks)
        return h[0], count

    def _prompt_layers(self, h, starts, turns):
        if self.normed:
            from transformers.models.qwen3.modeling_qwen3 import apply_rotary_pos_emb
        cache, T, bf = self.cache, h.shape[1], torch.bfloat16
        for i, L in enumerate(self.layers):
            a = L.self_attn
            x = L.input_layernorm(h)
            qo, ko, vo = self._beside(x, [a.q_proj, a.k_proj, a.v_proj], grouped_forward(x, [a.q_proj, a.k_proj, a.v_proj]))
            if self.normed:
                q = a.q_norm(qo.view(1, T, self.nh, self.hd)).transpose(1, 2)
                k = a.k_norm(ko.view(1, T, self.nkv, self.hd)).transpose(1, 2)
                q, k = apply_rotary_pos_emb(q, k, *turns)
                q = q[0].transpose(0, 1).to(bf).contiguous()
                cache.append(i, k[0].transpose(0, 1).to(bf).contiguous(), vo.view(T, self.nkv, self.hd).to(bf), starts)
            else:
                q, k, v = (t.view(T, heads, self.hd).to(bf) for t, heads in ((qo, self.nh), (ko, self.nkv), (vo, self.nkv)))
                q = cache.append_rotated(i, q, k, v, self.frequencies, starts, factor=self.turn_factor, out=q)
            o = cache.attend_chunk(i, q, starts, scale=self.scale, **self.spans)
            h = h + self._linear(o.view(1, T, self.nh * self.hd).to(h.dtype), a.o_proj)
            x = L.post_attention_layernorm(h)
            go, uo = self._beside(x, [L.mlp.gate_proj, L.mlp.up_proj], grouped_forward(x, [L.mlp.gate_proj, L.mlp.up_proj]))
            h = h + self._linear(L.mlp.act_fn(go) * uo, L.mlp.down_proj)
        return h

    @torch.no_grad()
    def prompt(self, ids, counts):
        """``counts[r]`` new tokens of row r (0: the row waits), their ids one
        row after the other in ``ids``.  Logits of every row's last token, for
        the rows with tokens."""
        h, count = self._prompt_hidden(ids, counts)
        last = (count.cumsum(0) - 1)[count > 0].to(self.dev)
        return self.model.lm_head(self.model.model.norm(h[last]))

    @torch.no_grad()
    def score(self, ids, counts, top=0, rows=1024):
        """``prompt`` with scores in place of logits (``logprobs.token_logprobs``): entry t is about the token behind
        ids[t] in its row, of which the row's last has none (log probability 0, rank -1; its entropy and alternatives
        are those of the token to come).  The logits of ``rows`` tokens are there at a time."""
        from .logprobs import MAX_TOP, token_logprobs
        most = min(MAX_TOP, self.model.lm_head.weight.shape[0])
        if not 0 <= top <= most or rows < 1:
            raise ValueError(f"{top} alternatives (0 to {most}), the logits of {rows} tokens at a time")
        h, count = self._prompt_hidden(ids, counts)
        behind = torch.full_like(ids, -100)
        behind[:-1] = ids[1:]
        behind[(count.cumsum(0) - 1)[count > 0].to(self.dev)] = -100
        norm, head = self.model.model.norm, self.model.lm_head
        parts = [token_logprobs(head(norm(x)), t.contiguous(), top) for x, t in zip(h.split(rows), behind.split(rows))]
        return tuple(torch.cat(p) for p in zip(*parts))

    @torch.no_grad()
    def step(self, ids, parents=None):
        """One new token for every row, ids (rows,) or (rows, 1): row i goes on
        from row ``parents[i]`` (int32; None: its own), with that row's
        adapters.  Logits (rows, vocab)."""
        if ids.numel() != self.B:
            raise ValueError(f"ids {tuple(ids.shape)} for {self.B} rows")
        self._check_ids(ids)
        if self.model.model.embed_tokens.weight.dtype != torch.bfloat16:
            raise TypeError("the decode step runs bf16 models")
        self._check_beside(self.B)
        self.cache.advance(1, parents)
        if parents is not None and self._adapted():
            named = (parents >= 0) & (parents < self.B)
            self.which.copy_(torch.where(named, self.which[parents.clamp(0, self.B - 1).long()], -1))
        logits = self._decode_step(ids.reshape(-1, 1), None)
        if self.window:
            self.cache.free(window=self.window, sinks=self.sinks)
        return logits

    def _attend(self, i, qo, ko, vo, norms, pos, out, stream):
        from .pages import _pool
        c, vp = self.cache, self._lib.ptr
        heads = (self.B, self.nh, self.hd)
        if norms is None:
            kv = (self.B, self.nkv, self.hd)
            q = c.append_rotated(i, qo.view(heads), ko.view(kv), vo.view(kv), self.frequencies, factor=self.turn_factor,
                                 out=qo.view(heads))
        else:
            q = torch.empty_like(out)
            self._lib.check(self._L.qs_page_append_rope_over(
                vp(qo), vp(ko), vp(vo), vp(norms[0]), vp(norms[1]), vp(self.cos), vp(self.sin), self.cos.shape[0], vp(q),
                self.B, self.nh, self.nkv, self.hd, _pool(c.keys(i), c.values(i), c.table, c.lengths), vp(c.over),
                self.eps, stream))
            q = q.view(heads)
        c.attend_token(i, q, scale=self.scale, out=out.view(heads), **self.spans)


def _each_prompts(which, prompts):
    """The adapters of every prompt, int32 on the host; None: none."""
    if which is None:
        return torch.full((prompts,), -1, dtype=torch.int32)
    which = torch.as_tensor(which)
    if which.shape != (prompts,) or which.is_floating_point() or which.dtype == torch.bool:
        raise ValueError(f"which must be a whole number for each of {prompts} prompts, got {tuple(which.shape)} x {which.dtype}")
    return which.to("cpu", torch.int64).clamp(-1, 2 ** 31 - 1).int()  # numbers beyond name none either way


@torch.no_grad()
def greedy_decode_paged(model, prompts, new_tokens, which=None, top=0, use_graph=True, page=64):
    """Greedy decode of prompts of any lengths (a list of 1-D id tensors), each with the adapters that ``which`` (a
    number for every prompt, -1 for none) names, and the log probabilities of what they take.  Steps are replays of one
    HIP graph unless use_graph=False.  Returns (tokens (prompts, new_tokens), their scores: log probabilities, entropies
    (prompts, new_tokens), the ``top`` best tokens' log probabilities and ids (prompts, new_tokens, top))."""
    from .logprobs import token_logprobs
    if not prompts or any(len(p) < 1 for p in prompts) or new_tokens < 1:
        raise ValueError(f"{new_tokens} new tokens behind prompts of {[len(p) for p in prompts]}: every prompt has a token or more")
    R, dev = len(prompts), prompts[0].device
    which = _each_prompts(which, R)
    dec = PagedDecoder(model, R, max(len(p) for p in prompts) + new_tokens, page)
    dec.which.copy_(which)
    logits = dec.prompt(torch.cat(list(prompts)), [len(p) for p in prompts])
    shapes = (((), torch.int32), ((), torch.float32), ((), torch.float32), ((top,), torch.float32), ((top,), torch.int32))
    out = [torch.zeros(R, new_tokens, *more, dtype=kind, device=dev) for more, kind in shapes]
    last = torch.zeros(R, dtype=torch.int32, device=dev)
    at = torch.zeros(1, dtype=torch.long, device=dev)

    def take(logits):
        _, entropy, _, best, tokens = token_logprobs(logits, last, max(top, 1))
        last.copy_(tokens[:, 0].clamp_min(0))  # a row without a finite logit takes token 0
        for o, new in zip(out, (last, best[:, 0], entropy, best[:, :top], tokens[:, :top])):
            o.index_copy_(1, at, new.unsqueeze(1))
        at.add_(1)

    def step():
        take(dec.step(last.long()))

    take(logits)
    todo, go = new_tokens - 1, step
    if use_graph and todo > 1:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        todo, go = todo - 1, graph.replay
    for _ in range(todo):
        go()
    dec.cache.check()
    return (out[0].long(), *out[1:])


@torch.no_grad()
def perplexity(model, ids, window=2048):
    """The perplexity of a text's ids (n,) under any causal LM, over windows of ``window`` tokens that do not overlap,
    each token given those before it in its window (as scripts/eval_ppl.py:41-65 takes it).  By the model's own forward,
    which runs no adapters: a fine-tune's tokens are scored by ``PagedDecoder.score``."""
    from .logprobs import token_logprobs
    total, count = 0.0, 0
    for part in ids.split(window):
        if len(part) < 2:
            continue
        logits = model(input_ids=part[None], use_cache=False).logits[0, :-1]
        total = total - token_logprobs(logits, part[1:].contiguous())[0].double().sum()
        count += len(part) - 1
    if not count:
        raise ValueError(f"{len(ids)} ids in windows of {window}: no token has one before it")
    return float(torch.exp(total / count))


@torch.no_grad()
def beam_decode(model, prompts, beams, new_tokens, eos=-1, use_graph=True, page=64, which=None):
    """Beam search: the ``beams`` best continuations of each prompt (a list of
    1-D id tensors, of any lengths) by ``new_tokens`` tokens, a beam that took
    ``eos`` going on with it at its score; ``which``: the adapters of each
    prompt (PagedDecoder).  Steps are replays of one HIP graph
    unless use_graph=False.  Returns (tokens (prompts, beams, new_tokens) in
    descending order of scores (prompts, beams), prompt s, decode s)."""
    from .beam import beam_select, reorder_states
    R, dev = len(prompts), prompts[0].device
    which = _each_prompts(which, R)
    longest = max(len(p) for p in prompts)
    columns = -(-(longest + new_tokens) // page)
    # every beam may come to hold all its pages after the prompt's last full one, and a copy of what it goes on from
    pages = sum(len(p) // page + 1 for p in prompts) + R * beams * (-(-new_tokens // page) + 2)
    dec = PagedDecoder(model, R * beams, columns * page, page, pages)
    dec.which.copy_(which.repeat_interleave(beams))
    counts = [0] * (R * beams)
    counts[::beams] = [len(p) for p in prompts]
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    logits = dec.prompt(torch.cat(list(prompts)), counts)
    torch.cuda.synchronize()
    t1 = time.perf_counter()
    # a prompt's row is its first beam, the only one that counts in the first selection
    scores = torch.full((R, beams), float("-inf"), device=dev)
    scores[:, 0] = 0
    scores, parents, last = beam_select(logits.repeat_interleave(beams, 0), scores)
    finished = last == eos
    tokens = torch.zeros(R * beams, new_tokens, dtype=torch.int32, device=dev)
    tokens[:, 0] = last.view(-1)
    at = torch.ones(1, dtype=torch.long, device=dev)

    def step():
        logits = dec.step(last.view(-1).long(), parents.view(-1))
        s, p, t = beam_select(logits, scores, finished=finished, eos=eos)
        old, ended = reorder_states([tokens, finished.view(-1, 1)], p)
        tokens.copy_(old.index_copy(1, at, t.view(-1, 1)))
        finished.copy_(ended.view(R, beams) | (t == eos))
        for keep, new in ((scores, s), (parents, p), (last, t)):
            keep.copy_(new)
        at.add_(1)

    if use_graph and new_tokens > 2:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        torch.cuda.synchronize()
        t1, t0 = time.perf_counter(), t0 + time.perf_counter() - t1  # the capture is no part of either time
        todo, go = new_tokens - 2, graph.replay
    else:
        todo, go = new_tokens - 1, step
    for _ in range(todo):
        go()
    torch.cuda.synchronize()
    t2 = time.perf_counter()
    dec.cache.check()
    return tokens.view(R, beams, new_tokens).long(), scores, t1 - t0, t2 - t1


def linear_bytes(m, n, B):
    """Algorithmic HBM bytes of one quantized-linear call: 2-byte codes per 8
    weights, bf16 activations in and out, 1-bit signs, fp16 scale."""
    return m * n // 8 * 2 + 2 * B * (n + m) + -(-(m + n) // 8) + 2


def linear_gbps(model, batches, reps=20):
    """Per-linear forward time and HBM GB/s (algorithmic bytes) for the
    decoder linears of the first layer, at each batch size: ``reps`` calls of
    the module captured in one HIP graph, replayed and timed with events."""
    layer = get_decoder_layers(model)[0]
    out = []
    dev = next(model.parameters()).device
    for group in get_linear_groups(layer, 0):
        for name, lin in group:
            n, m = lin.in_features, lin.out_features
            for B in batches:
                x = torch.randn(B, n, device=dev).bfloat16()
                with torch.no_grad():
                    lin(x)  # workspace, packed codes
                    torch.cuda.synchronize()
                    s = torch.cuda.Stream(device=dev)
                    s.wait_stream(torch.cuda.current_stream(dev))
                    with torch.cuda.stream(s):
                        lin(x)
                    torch.cuda.current_stream(dev).wait_stream(s)
                    torch.cuda.synchronize()
                    g = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(g):
                        for _ in range(reps):
                            lin(x)
                    g.replay()
                    torch.cuda.synchronize()
                    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
                    e0.record()
                    for _ in range(5):
                        g.replay()
                    e1.record()
                    torch.cuda.synchronize()
                us = e0.elapsed_time(e1) * 1e3 / (5 * reps)
                nb = linear_bytes(m, n, B)
                out.append({"linear": name, "m": m, "n": n, "batch": B, "us": round(us, 2),
                            "GBps": round(nb / (us * 1e-6) / 1e9, 1)})
                del g
    return out


def _graph_time(fn, replays=10):
    """Median ms of one replay of ``fn`` captured in a HIP graph (after a
    warm-up call outside capture and two warm-up replays)."""
    import statistics
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fn()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fn()
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    ev = [torch.cuda.Event(enable_timing=True) for _ in range(replays + 1)]
    ev[0].record()
    for i in range(replays):
        g.replay()
        ev[i + 1].record()
    torch.cuda.synchronize()
    ms = statistics.median(ev[i].elapsed_time(ev[i + 1]) for i in range(replays))
    del g
    return ms


@torch.no_grad()
def linears_step_ms(model, batch):
    """ms of the decoder linears alone for one decode step of ``batch`` rows,
    in StaticDecoder's order and call pattern (q/k/v grouped, o, gate/up
    grouped, down; each layer's input the previous layer's output), replayed
    from a HIP graph."""
    layers = get_decoder_layers(model)
    dev = next(model.parameters()).device
    h = torch.randn(batch, model.config.hidden_size, device=dev).bfloat16()

    def run():
        x = h
        for L in layers:
            a = L.self_attn
            qo, _, _ = grouped_forward(x, [a.q_proj, a.k_proj, a.v_proj])
            o = a.o_proj(qo)
            go, _ = grouped_forward(o, [L.mlp.gate_proj, L.mlp.up_proj])
            x = L.mlp.down_proj(go)
        return x
    return _graph_time(run)


@torch.no_grad()
def linear_gbps_rotated(model, batch):
    """Per decoder linear (q, k, v, o, gate, up, down): us and GB/s
    (algorithmic bytes) of one call, from a HIP graph that calls that linear
    of every decoder layer in turn, so the codes read per replay (for gate /
    up, 64 x 33 MB) far exceed the 256 MB Infinity Cache."""
    layers = get_decoder_layers(model)
    dev = next(model.parameters()).device
    out = []
    for name in ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj"):
        mods = [getattr(L.self_attn if name[0] in "qkvo" else L.mlp, name) for L in layers]
        n, m = mods[0].in_features, mods[0].out_features
        x = torch.randn(batch, n, device=dev).bfloat16()
        # _forward_one: this linear alone (a linked q or gate called under
        # capture would run its whole group)
        ms = _graph_time(lambda: [mod._forward_one(x) for mod in mods])
        us = ms * 1e3 / len(mods)
        out.append({"linear": name, "m": m, "n": n, "batch": batch, "us": round(us, 2),
                    "GBps": round(linear_bytes(m, n, batch) / (us * 1e-6) / 1e9, 1)})
    return out


def measure_decode(layers=64, batches=(1, 8), prompt=512, new=64, device="cuda:0"):
    """The Qwen3-32B-shaped greedy decode of ``new`` tokens after a ``prompt``
    -token random prompt, per batch size: prefill s, decode tok/s and ms per
    step (graph-replayed steps), the decoder linears' ms per step and the
    rest, and per-linear GB/s rotated over all layers."""
    from transformers import Qwen3Config
    cfg = Qwen3Config(**dict(QWEN3_32B, num_hidden_layers=layers))
    dev = torch.device(device)
    t0 = time.perf_counter()
    model = random_quantized_model(cfg, dev)
    torch.cuda.synchronize()
    res = {"model": "Qwen3-32B shape (64 layers, hidden 5120, intermediate 25600, 64 q / 8 kv heads, "
                    "vocab 151936), random init, every decoder linear E8P 2-bit", "layers": layers,
           "code_bytes": sum(m.codes.numel() * 2 for m in model.modules() if isinstance(m, QuantizedLinear)),
           "build_s": round(time.perf_counter() - t0, 1), "prompt": prompt, "new_tokens": new, "runs": []}
    for B in batches:
        g = torch.Generator().manual_seed(B)
        ids = torch.randint(0, cfg.vocab_size, (B, prompt), generator=g).to(dev)
        greedy_decode(model, ids[:, :16], 4)  # warm-up
        toks, pre_s, dec_s = greedy_decode_static(model, ids, new)
        steps = new - 1
        step_ms = 1e3 * dec_s / steps
        lin_ms = linears_step_ms(model, B)
        res["runs"].append({"batch": B, "prefill_s": round(pre_s, 3), "tok_per_s": round(B * steps / dec_s, 2),
                            "ms_per_step": round(step_ms, 3), "linears_ms_per_step": round(lin_ms, 3),
                            "other_ms_per_step": round(step_ms - lin_ms, 3),
                            "linears_GBps": round(res["code_bytes"] / (lin_ms * 1e-3) / 1e9, 1),
                            "per_linear": linear_gbps_rotated(model, B), "first_tokens": toks[0, :8].tolist()})
    del model
    torch.cuda.empty_cache()
    return res


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=64)
    ap.add_argument("--batch", type=int, nargs="+", default=[1, 8])
    ap.add_argument("--prompt", type=int, default=512)
    ap.add_argument("--new", type=int, default=256)
    ap.add_argument("--beams", type=int, default=0, help="also decode each batch by a search with this many beams")
    ap.add_argument("--eager", action="store_true", help="decode steps launched eagerly (no HIP graph)")
    args = ap.parse_args()
    from transformers import Qwen3Config
    cfg = Qwen3Config(**dict(QWEN3_32B, num_hidden_layers=args.layers))
    dev = torch.device("cuda:0")
    t0 = time.perf_counter()
    model = random_quantized_model(cfg, dev)
    torch.cuda.synchronize()
    build_s = time.perf_counter() - t0
    code_bytes = sum(m.codes.numel() * 2 for m in model.modules() if isinstance(m, QuantizedLinear))
    res = {"model": "Qwen3-32B shape (random init, E8P 2-bit decoder linears)", "layers": args.layers,
           "code_bytes": code_bytes, "build_s": round(build_s, 1), "runs": []}
    for B in args.batch:
        g = torch.Generator().manual_seed(B)
        ids = torch.randint(0, cfg.vocab_size, (B, args.prompt), generator=g).to(dev)
        greedy_decode(model, ids[:, :16], 4)  # warm-up
        toks, pre_s, dec_s = greedy_decode_static(model, ids, args.new, use_graph=not args.eager)
        steps = args.new - 1
        res["runs"].append({"batch": B, "graph": not args.eager, "prefill_s": round(pre_s, 3), "decode_s": round(dec_s, 3),
                            "tok_per_s": round(B * steps / dec_s, 2), "ms_per_step": round(1e3 * dec_s / steps, 3),
                            "first_tokens": toks[0, :8].tolist()})
        if args.beams:
            toks, scores, pre_s, dec_s = beam_decode(model, list(ids), args.beams, args.new, use_graph=not args.eager)
            res["runs"][-1]["beams"] = {"beams": args.beams, "prefill_s": round(pre_s, 3), "decode_s": round(dec_s, 3),
                                        "best_scores": [round(x, 3) for x in scores[:, 0].tolist()]}
    res["per_linear"] = linear_gbps(model, args.batch)
    print(json.dumps(res), flush=True)


if __name__ == "__main__":
    main()

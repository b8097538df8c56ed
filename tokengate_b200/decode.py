"""Gated generation: the prefill, then decode over the gated KV cache.

Mirrors the reference's one generation implementation, generate_batch
(tokengate/e2e_gate/decode/gate_decode.py:87-260), with its decode-side
contracts:

  * the cache layout the prefill leaves: layers above the gate hold the
    kept tokens (B, max_n_kept) with rows shorter than max_n_kept padded at
    the end, layers at and below the gate their full padded Phase-1 cache
    (B, max prompt length) — or the kept tokens with prune_below_gate;
    decoded tokens are appended after that prefix (:139-165);
  * the pad-slot mask: prefix slots past each row's valid length are never
    attended (:141-150, :152-164);
  * the folded Phase-2 softmax form (FormDecodeState,
    qwen3_flex_attention.py:978-1116): above the gate, every prefix key keeps
    the additive bias the prefill gave it (for the finalized gate the
    per-head bias times the head-mean scaled-softmax factor of the key's own
    ratio), decoded keys get none, and each decode query is scaled by
    gamma_h * r with r = min(log(max(n_kept + 1 + step, 2)) /
    log(max(pos + 1, 2)), 1) in float32, cast to bf16 (:374-415, :1089-1101);
    phase2_form=False is the plain decode (no bias, no query scale);
  * RoPE at the original positions: the first decode token sits one past
    the last kept position (:137-138);
  * stop when every row's last token is EOS; answers cut at the first EOS.

Each decode step runs the fused layer ops (residual add + RMSNorm, one
[q; k; v] projection, q/k RMSNorm + RoPE, the tg_decode_attn kernel over
the cache, o projection, SwiGLU MLP) and the head.

Beyond the reference, which decodes greedily over a bf16 cache: kv_bits=4
keeps the decode cache in 4 bits (kv4.KV4Cache: 144 bytes per slot and KV
head instead of 512; the prefill's K/V are quantised into it, the step's
k and v as they are appended, and attention runs on the codes), and a
Sampling draws the tokens (tg_sample) instead of the argmax.
"""
import time
from dataclasses import dataclass
from typing import List, Optional, Sequence, Union

import torch
import torch.nn.functional as F

from . import ops
from .kv4 import HEAD_DIM, KV4Cache
from .layers import fused_weights
from .prefill import prefill_batch_for_decode


@dataclass
class GateGenerateResult:
    token_ids: List[List[int]]  # generated ids per row, through the first EOS inclusive
    n_gen: List[int]            # generated tokens per row before the first EOS
    n_kepts: List[int]
    kept_pos: torch.Tensor      # (B, max_n_kept) original positions, on the device
    K_clampeds: List[int]
    prefill_s: float
    decode_s: float
    steps: int                  # decode steps run (batch-wide)
    logprobs: Optional[List[List[float]]] = None  # of token_ids, under the distributions sampled from


@dataclass
class Sampling:
    """How tokens are drawn (ops.sample_tokens): each setting one number, or one per request.

    temperature <= 0 is greedy; top_k None or <= 0, top_p None or >= 1 and min_p None or <= 0 are
    off. generator: a torch.Generator on the model's device for the uniform numbers (None: torch's
    own). One number per request and step is drawn, all of them before the first step."""
    temperature: Union[float, Sequence[float]] = 1.0
    top_k: Union[None, int, Sequence[int]] = None
    top_p: Union[None, float, Sequence[float]] = None
    min_p: Union[None, float, Sequence[float]] = None
    generator: Optional[torch.Generator] = None

    def on(self, B: int, device) -> dict:
        """The (B,) device tensors of the settings, as ops.sample_tokens takes them."""
        out = {}
        for name, dtype in (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32),
                            ("min_p", torch.float32)):
            val = getattr(self, name)
            if val is None:
                if name == "temperature":
                    raise ValueError("temperature must be a number or one per request")
                out[name] = None
                continue
            t = torch.as_tensor(val, dtype=None if dtype is torch.int32 else dtype, device="cpu")
            if dtype is torch.int32 and not bool((t == t.to(dtype)).all()):
                raise ValueError(f"{name} must be whole numbers of 32 bits, got {val}")
            t = t.to(dtype)
            if t.dim() > 1 or (t.dim() == 1 and t.shape[0] != B):
                raise ValueError(f"{name}: one value, or one for each of the {B} requests, got shape {tuple(t.shape)}")
            if t.is_floating_point() and bool(torch.isnan(t).any()):
                raise ValueError(f"{name} must not be NaN")
            out[name] = t.expand(B).contiguous().to(device)
        return out


def _sync(device) -> None:
    if device.type == "cuda":
        torch.cuda.synchronize(device)


def _proj(x: torch.Tensor, w: torch.Tensor, swiglu: bool = False, gemv: bool = True) -> torch.Tensor:
    """A decode-step projection of the (B, 1, K) rows: the tg_gemv kernel
    where it beats cuBLAS on B200 (measured: every projection at B <= 2, the
    layer projections at B <= 4; its CUDA-core FMAs fall behind cuBLAS's
    tensor cores beyond that, first on the 151936-row lm_head), cuBLAS
    otherwise or when gemv is False."""
    B, _, Kd = x.shape
    if gemv and Kd % 256 == 0 and (B <= 2 or (B <= _GEMV_LAYER_MAX_B and w.shape[0] < 32768)):
        return ops.gemv(x.view(B, Kd), w, swiglu=swiglu).view(B, 1, -1)
    y = F.linear(x, w)
    return ops.silu_mul(y) if swiglu else y


# the largest batch whose layer projections (fewer than 32768 output rows)
# run on tg_gemv (measured on B200: at B = 6 and 8 the decode step is
# 8-15 % slower with them there than on cuBLAS)
_GEMV_LAYER_MAX_B = 4


class _DecodeCache:
    """Per-layer K/V with room for the decoded tokens: the prefill's prefix
    copied to the front, decode tokens appended after it."""

    def __init__(self, cache, n_layers: int, extra: int):
        self.k, self.v, self.width = [], [], []
        for i in range(n_layers):
            k, v = cache.layers[i].k_tok, cache.layers[i].v_tok
            B, W, Hkv, D = k.shape
            kb = torch.empty((B, W + extra, Hkv, D), dtype=k.dtype, device=k.device)
            vb = torch.empty_like(kb)
            kb[:, :W].copy_(k)
            vb[:, :W].copy_(v)
            self.k.append(kb)
            self.v.append(vb)
            self.width.append(W)


class _DecodeCacheKV4:
    """The same in 4 bits: the prefill's prefix quantised to the front, decode tokens appended after it. Each layer's
    bf16 K/V are released from `cache` once they are written, so that the peak is the prefill's, not both caches."""

    def __init__(self, cache, n_layers: int, extra: int):
        self.kv, self.width = [], []
        for i in range(n_layers):
            layer = cache.layers[i]
            B, W, Hkv, _ = layer.k_tok.shape
            c = KV4Cache(B, W + extra, Hkv, device=layer.k_tok.device)
            ops.kv4_write(c, layer.k_tok, layer.v_tok)
            layer.k_tok = layer.v_tok = None
            self.kv.append(c)
            self.width.append(W)


def _check_kv4(cfg) -> None:
    """The heads that the 4-bit cache and its attention serve."""
    Hq, Hkv = cfg.num_attention_heads, cfg.num_key_value_heads
    D = getattr(cfg, "head_dim", None) or cfg.hidden_size // Hq
    if D != HEAD_DIM or Hq % Hkv or Hq // Hkv > 8:
        raise ValueError(f"kv_bits=4 serves head_dim {HEAD_DIM} and 1 to 8 query heads per KV head, the model has "
                         f"head_dim {D} and {Hq} query heads on {Hkv} KV heads")


@torch.no_grad()
def generate_batch(model, gate, prompt_ids_list: Sequence, article_starts: Sequence[int],
                   article_ends: Sequence[int], gate_layer: int, max_kept_prefill_tokens,
                   max_new_tokens: int, *, eos_token_id: Optional[int] = None,
                   phase2_form: bool = True, prune_below_gate: bool = False,
                   streamer=None, forced_tokens: Optional[torch.Tensor] = None,
                   logits_out: Optional[list] = None, use_graph: bool = True,
                   use_gemv: bool = True, sampling: Optional[Sampling] = None,
                   kv_bits: int = 16) -> GateGenerateResult:
    """Gated prefill + decode of up to max_new_tokens tokens per row.

    forced_tokens: (B, max_new_tokens - 1) ids fed to the decode steps in
    place of the previous step's argmax (teacher forcing, to score a given
    continuation);
    logits_out: a list that receives each decode step's (B, vocab) fp32 logits;
    use_graph: replay the decode step as one CUDA graph after the first
    (eager) step — the state a step reads (token, position, append slot, key
    count) lives in device buffers the step itself advances; use_gemv: the
    decode projections on the tg_gemv kernel (False: cuBLAS);
    sampling: draw the tokens as it says (None: the argmax of each step) and
    return their log-probabilities;
    kv_bits: 16 for a bf16 decode cache, 4 for a 4-bit one."""
    if max_new_tokens < 1:
        raise ValueError("max_new_tokens must be positive")
    if kv_bits not in (4, 16):
        raise ValueError(f"kv_bits={kv_bits}: 16 (bf16) or 4")
    if kv_bits == 4 and max_new_tokens > 1:
        _check_kv4(model.config)
    device = next(model.parameters()).device
    if sampling is not None:     # refused before the prefill, if at all
        if model.lm_head.weight.shape[0] > ops.SAMPLE_MAX_VOCAB:
            raise ValueError(f"sampling serves vocabularies of up to {ops.SAMPLE_MAX_VOCAB}, the model's has "
                             f"{model.lm_head.weight.shape[0]}")
        draw = sampling.on(len(prompt_ids_list), device)
        u_all = torch.rand((max_new_tokens, len(prompt_ids_list)), dtype=torch.float32, device=device,
                           generator=sampling.generator)
    inner = model.model
    n_layers = len(inner.layers)
    st: dict = {}
    _sync(device)
    t0 = time.perf_counter()
    first, cache, kept_pos, n_kepts, K_cl = prefill_batch_for_decode(
        model, gate, prompt_ids_list, article_starts, article_ends, gate_layer,
        max_kept_prefill_tokens, prune_below_gate=prune_below_gate, fused=True, decode_state=st)
    _sync(device)
    prefill_s = time.perf_counter() - t0
    B = first.shape[0]
    lps = []
    if sampling is not None:
        tok, lp = ops.sample_tokens(st["logits"], u_all[0], **draw)
        first = tok.view(B, 1)
        lps.append(lp)
    if streamer is not None:
        streamer.put(first.detach().cpu())
    gen = [first]
    steps = 0
    t1 = time.perf_counter()
    if max_new_tokens > 1:
        fw = fused_weights(model)
        lens = st["lens"]
        dc = (_DecodeCacheKV4 if kv_bits == 4 else _DecodeCache)(cache, n_layers, max_new_tokens - 1)
        del cache
        n_kept_dev = torch.tensor(n_kepts, dtype=torch.int32, device=device)
        valid_below = n_kept_dev if prune_below_gate else torch.tensor(lens, dtype=torch.int32, device=device)
        last = torch.tensor([n - 1 for n in n_kepts], device=device)
        next_pos = kept_pos[torch.arange(B, device=device), last] + 1            # (B,)
        n_p2 = n_layers - 1 - gate_layer
        bias = st["bias"] if phase2_form else [None] * n_p2
        qs_all = None
        if phase2_form and st["gamma"] is not None:
            # the per-step query scale of every Phase-2 layer, computed as
            # FormDecodeState.step does (float32 on the device)
            s_idx = torch.arange(max_new_tokens - 1, device=device, dtype=torch.float32)[:, None]
            m = (n_kept_dev.float()[None, :] + 1 + s_idx).clamp(min=2.0)               # (steps, B)
            pp = (next_pos.float()[None, :] + s_idx + 1.0).clamp(min=2.0)
            r = (torch.log(m) / torch.log(pp)).clamp(max=1.0)
            gam = st["gamma"].float()                                                   # (L', H)
            qs_all = (gam[None, :, None, :] * r[:, None, :, None]).contiguous()        # (steps, L', B, H)
        lw0 = fw[0]
        nq, nkv, D = lw0.n_q, lw0.n_kv, lw0.head_dim
        # step state on the device, so that one captured step serves every
        # step: the token, its position, each cache's append slot and key count
        cur = first.clone()
        wb, w2 = dc.width[0], dc.width[n_layers - 1]
        extra = max_new_tokens - 1
        # the counters one step advances, one add each: the two caches' append
        # slots and the step index (int64), the two key counts (int32)
        ctr = torch.tensor([wb, w2, 0], dtype=torch.int64, device=device)
        slot_b, slot_2, step_idx = ctr[0:1], ctr[1:2], ctr[2:3]
        nkc = torch.tensor([wb + 1, w2 + 1], dtype=torch.int32, device=device)
        nk_b, nk_2 = nkc[0:1], nkc[1:2]
        # the rotary cos / sin of every decode position, made once by the
        # model's own rotary embedding (elementwise in the position, so equal
        # to making them step by step); a step gathers its row
        step_pos = next_pos.view(B, 1) + torch.arange(extra, device=device).view(1, extra)      # (B, extra)
        like = torch.empty((B, 1, 1), dtype=inner.embed_tokens.weight.dtype, device=device)
        cos_t, sin_t = inner.rotary_emb(like, step_pos)
        rot = torch.stack((cos_t, sin_t), dim=2)                                                 # (B, extra, 2, D)
        qs_cur = torch.empty_like(qs_all[0]) if qs_all is not None else None
        lg_buf = torch.empty((B, model.lm_head.weight.shape[0]), dtype=torch.float32, device=device)
        lp_buf = torch.empty(B, dtype=torch.float32, device=device)

        def step_body():
            h = inner.embed_tokens(cur)                                               # (B, 1, H)
            r = rot.index_select(1, step_idx)                                         # (B, 1, 2, D)
            cos, sin = r[:, :, 0], r[:, :, 1]
            delta = None
            for i in range(n_layers):
                lw = fw[i]
                below = i <= gate_layer
                h, x = ops.add_rmsnorm(h, delta, lw.in_w, lw.eps, h_out=h if delta is not None else None)
                qkv = _proj(x, lw.wqkv, gemv=use_gemv).view(B, 1, nq + 2 * nkv, D)
                q = qkv[:, :, :nq]
                k = qkv[:, :, nq:nq + nkv]
                v = qkv[:, :, nq + nkv:]
                W, li = dc.width[i], i - gate_layer - 1
                slot, nk = (slot_b, nk_b) if below else (slot_2, nk_2)
                valid = valid_below if below else n_kept_dev
                kw = dict(n_keys_dev=nk)
                if not below:
                    kw.update(bias=bias[li], q_scale=qs_cur[li] if qs_cur is not None else None)
                if kv_bits == 4:
                    q = ops.qk_norm_rope_append_kv4(q, k, v, lw.q_norm_w, lw.k_norm_w, cos, sin, lw.qk_eps,
                                                    dc.kv[i], slot)
                    a = ops.decode_attention_kv4(q[:, 0], dc.kv[i], valid, W, W + extra, **kw)
                else:
                    ops.qk_norm_rope_append(q, k, v, lw.q_norm_w, lw.k_norm_w, cos, sin, lw.qk_eps,
                                            dc.k[i], dc.v[i], slot)
                    a = ops.decode_attention(q[:, 0], dc.k[i], dc.v[i], valid, W, W + extra, **kw)
                o = _proj(a.view(B, 1, nq * D), lw.wo, gemv=use_gemv)
                h, x2 = ops.add_rmsnorm(h, o, lw.post_w, lw.eps, h_out=h)
                delta = _proj(_proj(x2, lw.wgu, swiglu=True, gemv=use_gemv), lw.wdown, gemv=use_gemv)
            _, hn = ops.add_rmsnorm(h, delta, inner.norm.weight, float(inner.norm.variance_epsilon))
            lg = _proj(hn, model.lm_head.weight, gemv=use_gemv)[:, -1]
            lg_buf.copy_(lg)
            if sampling is not None:     # the step after step_idx draws with the next row of numbers
                ops.sample_tokens(lg, u_all.index_select(0, step_idx + 1).view(B), token=cur.view(B), logprob=lp_buf,
                                  **draw)
            else:
                cur.copy_(lg.argmax(-1, keepdim=True))
            ctr.add_(1)
            nkc.add_(1)

        graph = None
        eos_seen = torch.zeros(B, dtype=torch.bool, device=device)
        for step in range(extra):
            if eos_token_id is not None:
                eos_seen |= cur[:, 0] == eos_token_id
                if bool(eos_seen.all()):
                    break
            if forced_tokens is not None:
                cur.copy_(forced_tokens[:, step:step + 1].to(device=device, dtype=cur.dtype))
            if qs_cur is not None:
                qs_cur.copy_(qs_all[step])
            if graph is None and use_graph and step > 0:
                # the first step ran eagerly (library handles, kernel attributes);
                # capture the same body once, replay it for the rest
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    step_body()
            if graph is not None:
                graph.replay()
            else:
                step_body()
            if logits_out is not None:
                logits_out.append(lg_buf.clone())
            nxt = cur.clone()
            if streamer is not None:
                streamer.put(nxt.detach().cpu())
            gen.append(nxt)
            if sampling is not None:
                lps.append(lp_buf.clone())
            steps += 1
        del graph
    _sync(device)
    decode_s = time.perf_counter() - t1
    if streamer is not None:
        streamer.end()
    allg = torch.cat(gen, dim=1).cpu().tolist()
    token_ids, n_gen, logprobs = [], [], None
    if lps:
        logprobs = torch.stack(lps, dim=1).cpu().tolist()
    for row in allg:
        if eos_token_id is not None and eos_token_id in row:
            end = row.index(eos_token_id)
            token_ids.append(row[:end + 1])
            n_gen.append(end)
        else:
            token_ids.append(row)
            n_gen.append(len(row))
    if logprobs is not None:
        logprobs = [row[:len(t)] for row, t in zip(logprobs, token_ids)]
    return GateGenerateResult(token_ids, n_gen, list(n_kepts), kept_pos, list(K_cl), prefill_s, decode_s, steps,
                              logprobs)

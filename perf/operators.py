"""The operators of a decode step over a 4-bit KV cache, as cases to be measured.

Four operators, each with a plain form in elementary torch operations and the framework's own call:

  store    K and V rows quantised into the cache and read back
           (ops.kv4_write, ops.kv4_read)
  append   one decode token per row: q/k RMSNorm + RoPE, k and v quantised into the cache's next slot
           (ops.qk_norm_rope_append_kv4; the slot is read back, since 4 bits are compared as values)
  attend   one query token per head against the 4-bit cache, with the gated prefill's key bias, query
           scale and pad slots (ops.decode_attention_kv4)
  sample   the next token from the logits: temperature, top-k, top-p and min-p, from given uniform
           numbers (ops.sample_tokens)

The cache holds a row's 128 values as two groups of 64, each 4-bit codes of a bf16 step `scale` above
a bf16 `low`: value = low + code * scale.
"""
import math

import torch

own = False

_D, _GROUP = 128, 64
_ROW_BYTES = _D // 2 + (_D // _GROUP) * 4        # codes, and a scale and a low per group


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a layer's K/V of a whole 32k prompt (at and below the gate), contiguous
        dict(name="store prompt 32768", op="store", B=1, S=32768, Hkv=8, start=0, fused=False),
        # the kept tokens of a layer above the gate: views of the fused [q | k | v] projection
        dict(name="store kept 2768 views", op="store", B=1, S=2768, Hkv=8, start=0, fused=True),
        # a short second turn, put behind an odd number of cached tokens
        dict(name="store turn 77 at 4099", op="store", B=3, S=77, Hkv=2, start=4099, fused=True),
        # the append of one interactive request's decode step
        dict(name="append B1", op="append", B=1, Hq=16, Hkv=8, slot=2771),
        # the append of a full serving batch
        dict(name="append B64", op="append", B=64, Hq=32, Hkv=8, slot=4095),
        # a layer above the gate: 2768 kept keys with their per-head bias and the scaled query
        dict(name="attend kept 2768", op="attend", B=1, Hq=16, Hkv=8, prefix=2768, keys=2771, bias="head",
             qscale=True, pads="none"),
        # a layer at or below the gate: the whole 32k prompt, no bias
        dict(name="attend prompt 32768", op="attend", B=1, Hq=16, Hkv=8, prefix=32768, keys=32775, bias="none",
             qscale=False, pads="none"),
        # a batch of unlike prompts: pad slots holding rubbish, a row without any key, one bias row for all heads
        dict(name="attend ragged B16 4097", op="attend", B=16, Hq=32, Hkv=8, prefix=4097, keys=4097, bias="row",
             qscale=False, pads="ragged"),
        # the long-context shape: 128k keys, two requests on a GPU
        dict(name="attend 131072 B2", op="attend", B=2, Hq=32, Hkv=8, prefix=131072, keys=131081, bias="none",
             qscale=False, pads="none"),
        # one interactive request, the usual settings
        dict(name="sample B1", op="sample", B=1, V=151936, dtype="bf16", temperature=0.7, top_k=50, top_p=0.9,
             min_p=0.0, spread=2.5, mixed=False),
        # a serving batch whose requests bring settings of their own
        dict(name="sample B64 mixed", op="sample", B=64, V=151936, dtype="fp32", temperature=1.0, top_k=0, top_p=0.95,
             min_p=0.0, spread=2.0, mixed=True),
        # a small odd vocabulary with min-p alone
        dict(name="sample B5 V1001", op="sample", B=5, V=1001, dtype="fp32", temperature=1.3, top_k=0, top_p=1.0,
             min_p=0.05, spread=1.5, mixed=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "append", "attend", "attend", "sample", "sample"])
    if op == "store":
        B = rng.choice([1, 1, 2, 3, 5])
        S = _log_int(rng, 1, 32768 // B)
        return dict(op=op, B=B, S=S, Hkv=rng.choice([1, 2, 4, 8]), start=rng.choice([0, 0, _log_int(rng, 1, 20000)]),
                    fused=rng.random() < 0.5)
    if op == "append":
        Hkv = rng.choice([1, 2, 4, 8])
        return dict(op=op, B=_log_int(rng, 1, 64), Hq=Hkv * rng.choice([1, 2, 4, 8]), Hkv=Hkv, slot=_log_int(rng, 1, 16384) - 1)
    if op == "attend":
        Hkv = rng.choice([1, 2, 4, 8])
        B = rng.choice([1, 1, 2, 3, 7, 16])
        prefix = _log_int(rng, 1, 131072 * 2 // (B * 2))
        return dict(op=op, B=B, Hq=Hkv * rng.choice([1, 2, 4, 8]), Hkv=Hkv, prefix=prefix,
                    keys=prefix + rng.choice([0, 1, _log_int(rng, 1, 300)]), bias=rng.choice(["none", "row", "head"]),
                    qscale=rng.random() < 0.5, pads=rng.choice(["none", "ragged"]))
    return dict(op=op, B=_log_int(rng, 1, 64), V=_log_int(rng, 300, 151936), dtype=rng.choice(["bf16", "fp32"]),
                temperature=round(rng.uniform(0.3, 1.6), 3), top_k=rng.choice([0, 1, 20, 50, 1000]),
                top_p=rng.choice([1.0, 0.95, 0.8, 0.3]), min_p=rng.choice([0.0, 0.0, 0.05, 0.1]),
                spread=round(rng.uniform(0.3, 3.5), 2), mixed=rng.random() < 0.3)


# ------------------------------------------------------------------ inputs
def _rows(g, B, S, H):
    """Rows with the uneven channels of real keys and values: a few are large, most have an offset."""
    gain = torch.exp(0.5 * torch.randn(H, _D, generator=g, device="cuda"))
    mean = 0.5 * torch.randn(H, _D, generator=g, device="cuda")
    return (torch.randn(B, S, H, _D, generator=g, device="cuda") * gain + mean).to(torch.bfloat16)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    c, op = case, case["op"]
    if op == "store":
        k, v = _rows(g, c["B"], c["S"], c["Hkv"]), _rows(g, c["B"], c["S"], c["Hkv"])
        if c["fused"]:      # two query heads per KV head before them
            qkv = torch.cat([torch.zeros(c["B"], c["S"], 2 * c["Hkv"], _D, dtype=k.dtype, device="cuda"), k, v], dim=2)
            k, v = qkv[:, :, 2 * c["Hkv"]:3 * c["Hkv"]], qkv[:, :, 3 * c["Hkv"]:]
        return dict(k=k, v=v)
    if op == "append":
        B, Hq, Hkv = c["B"], c["Hq"], c["Hkv"]
        qkv = torch.cat([_rows(g, B, 1, Hq), _rows(g, B, 1, Hkv), _rows(g, B, 1, Hkv)], dim=2)
        pos = torch.randint(c["slot"], 4 * c["slot"] + 2, (B, 1), generator=g, device="cuda")
        freq = 1e6 ** (-torch.arange(0, _D, 2, device="cuda", dtype=torch.float64) / _D)
        ang = pos.double()[..., None] * freq
        ang = torch.cat([ang, ang], dim=-1)
        return dict(q=qkv[:, :, :Hq], k=qkv[:, :, Hq:Hq + Hkv], v=qkv[:, :, Hq + Hkv:],
                    qw=(1 + 0.2 * rn(_D)).to(torch.bfloat16), kw=(1 + 0.2 * rn(_D)).to(torch.bfloat16),
                    cos=ang.cos().to(torch.bfloat16), sin=ang.sin().to(torch.bfloat16), eps=1e-6,
                    slot=torch.tensor([c["slot"]], dtype=torch.int64, device="cuda"))
    if op == "attend":
        B, Hq, P = c["B"], c["Hq"], c["prefix"]
        k, v = _rows(g, B, c["keys"], c["Hkv"]), _rows(g, B, c["keys"], c["Hkv"])
        n_valid = torch.full((B,), P, dtype=torch.int32, device="cuda")
        if c["pads"] == "ragged":
            n_valid = torch.randint(0, P + 1, (B,), generator=g, device="cuda").to(torch.int32)
            n_valid[0] = P
            n_valid[B // 2] = 0 if B > 2 else P
            pad = torch.arange(c["keys"], device="cuda")[None] >= n_valid[:, None]
            pad[:, P:] = False
            k[pad] = float("nan")
            v[pad] = float("inf")
        bias = None
        if c["bias"] != "none":
            bias = torch.nn.functional.logsigmoid(2 * rn(B, Hq if c["bias"] == "head" else 1, P))
            low = torch.rand(bias.shape, generator=g, device="cuda")
            bias = torch.where(low < 0.02, torch.full_like(bias, -1e9), bias)
            bias = torch.where(low < 0.01, torch.full_like(bias, torch.finfo(torch.float32).min), bias)
        qs = 0.5 + torch.rand(B, Hq, generator=g, device="cuda") if c["qscale"] else None
        return dict(q=rn(B, Hq, _D).to(torch.bfloat16), k=k, v=v, n_valid=n_valid, bias=bias, q_scale=qs)
    B, V = c["B"], c["V"]
    x = c["spread"] * rn(B, V)
    x.scatter_add_(1, torch.randint(0, V, (B, 4), generator=g, device="cuda"), 4 * c["spread"] * torch.rand(B, 4, generator=g, device="cuda"))
    x = x.to(torch.bfloat16 if c["dtype"] == "bf16" else torch.float32)
    full = lambda val, dt: torch.full((B,), val, dtype=dt, device="cuda")  # noqa: E731
    t, k, p, m = (full(c["temperature"], torch.float32), full(c["top_k"], torch.int32), full(c["top_p"], torch.float32),
                  full(c["min_p"], torch.float32))
    if c["mixed"]:          # every fourth request greedy, others with a top-k or a min-p besides
        r = torch.arange(B, device="cuda")
        t = torch.where(r % 4 == 1, torch.zeros_like(t), t * (0.6 + 0.1 * (r % 8)))
        k = torch.where(r % 4 == 2, (r * 7 + 1).to(torch.int32), k)
        m = torch.where(r % 8 == 3, torch.full_like(m, 0.02), m)
    return dict(logits=x, u=torch.rand(B, generator=g, device="cuda"), temperature=t, top_k=k, top_p=p, min_p=m)


def prepare(case, seed):
    """The inputs, and the cache that the program keeps between calls: codes, scales and lows in plain tensors,
    or the framework's cache holding the same rows."""
    s = dict(case=case, **_inputs(case, seed))
    op = case["op"]
    if op == "sample":
        return s
    if own:
        from tokengate_b200 import ops
        from tokengate_b200.kv4 import KV4Cache
        cap = case["start"] + case["S"] if op == "store" else case["slot"] + 1 if op == "append" else case["keys"]
        s["cache"] = KV4Cache(case["B"], cap, case["Hkv"], device="cuda")
        if op == "attend":
            ops.kv4_write(s["cache"], s["k"], s["v"])
    elif op == "attend":
        s["kc"], s["vc"] = _pack(*_quantise(s["k"])), _pack(*_quantise(s["v"]))
    if op == "attend":
        del s["k"], s["v"]
    return s


# ------------------------------------------------------------------ plain forms
def _quantise(x):
    """codes (..., 2, 64) in fp32, scale and low (..., 2, 1) of rows (..., 128). Halves go up: the reciprocal is taken
    2^-22 high, so that its own rounding never takes one down."""
    x = x.float().unflatten(-1, (2, _GROUP))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    half = high * 0.5 - low * 0.5
    scale = (half / torch.full_like(half, 7.5)).to(torch.bfloat16).float()
    scale = torch.where(scale < 2.0 ** -100, torch.zeros_like(scale), scale)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    inverse = 1.0 / torch.where(scale == 0, torch.ones_like(scale), scale) * (1 + 2.0 ** -22)
    codes = torch.floor((x - low) * inverse + 0.5)
    codes = torch.where((scale == 0) | bad, torch.zeros_like(codes), codes)
    return codes, torch.where(bad, torch.full_like(scale, float("nan")), scale), torch.where(bad, torch.zeros_like(low), low)


def _values(codes, scale, low):
    return (low + codes * scale).flatten(-2)


def _pack(codes, scale, low):
    c = codes.flatten(-2).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), scale.to(torch.bfloat16), low.to(torch.bfloat16)


def _unpack(packed, scale, low):
    codes = torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2).float().unflatten(-1, (2, _GROUP))
    return _values(codes, scale.float(), low.float())


def _norm_rope(x, w, cos, sin, eps):
    """In fp32 but for the mean square, whose last bit would otherwise hang on the order of summing, and a code on it."""
    x = x.float()
    y = x * torch.rsqrt(((x * x).double().mean(-1, keepdim=True) + eps).float()) * w.float()
    rot = torch.cat([-y[..., _D // 2:], y[..., :_D // 2]], dim=-1)
    return y * cos.float()[:, :, None] + rot * sin.float()[:, :, None]


def _plain_attend(s):
    c = s["case"]
    B, Hq, Hkv, N = c["B"], c["Hq"], c["Hkv"], c["keys"]
    q = s["q"].float()
    if s["q_scale"] is not None:
        q = (q * s["q_scale"].to(torch.bfloat16).float()[..., None]).to(torch.bfloat16).float()
    j = torch.arange(N, device="cuda")
    seen = (j[None] < s["n_valid"][:, None]) | (j[None] >= c["prefix"])                         # (B, N)
    k = _unpack(*s["kc"]).transpose(1, 2)                                                       # (B, Hkv, N, D)
    x = torch.matmul(q.view(B, Hkv, Hq // Hkv, _D), k.transpose(-1, -2)) * _D ** -0.5           # (B, Hkv, G, N)
    x = x.view(B, Hq, N)
    if s["bias"] is not None:
        x = x + torch.cat([s["bias"], s["bias"].new_zeros(B, s["bias"].shape[1], N - c["prefix"])], dim=-1)
    x = torch.where(seen[:, None], x, torch.full_like(x, float("-inf")))
    top = x.amax(-1, keepdim=True)
    e = torch.where(seen[:, None], torch.exp(x - top), torch.zeros_like(x))
    total = e.sum(-1, keepdim=True)
    p = torch.where(total > 0, e / total, torch.zeros_like(e))
    v = _unpack(*s["vc"])
    v = torch.where(seen[..., None, None], v, torch.zeros_like(v)).transpose(1, 2)
    return torch.matmul(p.view(B, Hkv, Hq // Hkv, N), v).view(B, Hq, _D).to(torch.bfloat16)


def _plain_sample(s):
    """Weights in fp32; their running sums in fp64, so that the token does not hang on the order of summing."""
    raw = s["logits"].float()
    raw = torch.where(torch.isnan(raw), torch.full_like(raw, float("-inf")), raw)
    B, V = raw.shape
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"])
    z = raw / t[:, None].expand(B, V)
    d = z - z.amax(-1, keepdim=True)
    w = torch.exp(d)
    order = torch.sort(raw, dim=-1, descending=True, stable=True).indices
    rank = torch.arange(V, device="cuda")[None]
    n = torch.where(greedy, torch.ones_like(s["top_k"]), torch.where(s["top_k"] <= 0, torch.full_like(s["top_k"], V), s["top_k"]))
    ws = torch.where(rank < n[:, None], w.gather(1, order), torch.zeros_like(w)).double()
    cum = ws.cumsum(-1)
    inside = (cum - ws < s["top_p"].double()[:, None] * cum[:, -1:]) | (s["top_p"] >= 1)[:, None] | (rank == 0)
    keep_sorted = inside & (ws > 0)
    keep = torch.zeros_like(keep_sorted).scatter_(1, order, keep_sorted) & (w >= s["min_p"].clamp(max=1)[:, None])
    kept = torch.where(keep, w, torch.zeros_like(w)).double().cumsum(-1)
    mass = kept[:, -1:]
    token = (kept <= s["u"].double()[:, None] * mass).sum(-1)
    token = torch.minimum(token, (rank * keep).amax(-1))
    return token, d.gather(1, token[:, None])[:, 0] - torch.log(mass[:, 0]).float()


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if own:
        from tokengate_b200 import ops
        if op == "store":
            ops.kv4_write(s["cache"], s["k"], s["v"], start=c["start"])
            return ops.kv4_read(s["cache"], c["start"], c["S"])
        if op == "append":
            q = ops.qk_norm_rope_append_kv4(s["q"], s["k"], s["v"], s["qw"], s["kw"], s["cos"], s["sin"], s["eps"],
                                            s["cache"], s["slot"])
            return (q,) + tuple(ops.kv4_read(s["cache"], c["slot"], 1))
        if op == "attend":
            return ops.decode_attention_kv4(s["q"], s["cache"], s["n_valid"], c["prefix"], c["keys"], bias=s["bias"],
                                            q_scale=s["q_scale"])
        return ops.sample_tokens(s["logits"], s["u"], s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                 min_p=s["min_p"])
    if op == "store":
        return _values(*_quantise(s["k"])).to(torch.bfloat16), _values(*_quantise(s["v"])).to(torch.bfloat16)
    if op == "append":
        q = _norm_rope(s["q"], s["qw"], s["cos"], s["sin"], s["eps"]).to(torch.bfloat16)
        k = _norm_rope(s["k"], s["kw"], s["cos"], s["sin"], s["eps"]).to(torch.bfloat16)
        return q, _values(*_quantise(k)).to(torch.bfloat16), _values(*_quantise(s["v"])).to(torch.bfloat16)
    if op == "attend":
        return _plain_attend(s)
    return _plain_sample(s)


# ------------------------------------------------------------------ work and exact values
def work(case):
    c, op = case, case["op"]
    if op == "store":
        n = 2 * c["B"] * c["S"] * c["Hkv"]
        return {"bytes": n * (2 * _D * 2 + _ROW_BYTES), "flops": 6 * n * _D}
    if op == "append":
        n, q = 2 * c["B"] * c["Hkv"], c["B"] * c["Hq"]
        return {"bytes": n * (2 * _D * 2 + _ROW_BYTES) + q * 4 * _D + c["B"] * 4 * _D, "flops": (n * 12 + q * 8) * _D}
    if op == "attend":     # ragged: half of the prefix is there on average
        keys = c["B"] * (c["keys"] - (c["prefix"] // 2 if c["pads"] == "ragged" and c["B"] > 1 else 0))
        bias = {"none": 0, "row": 1, "head": c["Hq"]}[c["bias"]] * 4
        return {"bytes": keys * (2 * c["Hkv"] * _ROW_BYTES + bias) + 4 * c["B"] * c["Hq"] * _D, "flops": 4 * keys * c["Hq"] * _D}
    return {"bytes": c["B"] * c["V"] * (2 if c["dtype"] == "bf16" else 4) + 32 * c["B"], "flops": 4 * c["B"] * c["V"]}


def _exact_rows(x):
    """The quantiser's definition in 64 bits: the values that the rows' 4 bits stand for."""
    x = x.double().reshape(*x.shape[:-1], _D // _GROUP, _GROUP)
    low = x.min(-1, keepdim=True).values
    step = ((x.max(-1, keepdim=True).values - low) / 15).bfloat16().double()
    step[step < 2.0 ** -100] = 0
    code = ((x - low) / step + 0.5).floor()
    out = torch.where(step > 0, low + code * step, low.expand_as(x))
    out[~x.isfinite().all(-1)] = float("nan")
    return out.reshape(*x.shape[:-2], _D)


def exact(case, seed):
    c, op, s = case, case["op"], _inputs(case, seed)
    if op == "store":
        return _exact_rows(s["k"]), _exact_rows(s["v"])
    if op == "append":
        half = _D // 2

        def turned(x, w):
            x = x.double()
            x = x / (x.pow(2).sum(-1, keepdim=True) / _D + s["eps"]).sqrt() * w.double()
            co, si = s["cos"].double().unsqueeze(2), s["sin"].double().unsqueeze(2)
            a, b = x[..., :half], x[..., half:]
            return torch.cat([a * co[..., :half] - b * si[..., :half], b * co[..., half:] + a * si[..., half:]], -1)

        return turned(s["q"], s["qw"]), _exact_rows(turned(s["k"], s["kw"]).bfloat16()), _exact_rows(s["v"])
    if op == "attend":
        B, Hq, G, P, N = c["B"], c["Hq"], c["Hq"] // c["Hkv"], c["prefix"], c["keys"]
        out = torch.zeros(B, Hq, _D, dtype=torch.float64, device="cuda")
        for b in range(B):
            n = int(s["n_valid"][b])
            at = torch.cat([torch.arange(n, device="cuda"), torch.arange(P, N, device="cuda")])
            if not len(at):
                continue
            kd, vd = _exact_rows(s["k"][b, at]), _exact_rows(s["v"][b, at])
            for h in range(Hq):
                q = s["q"][b, h].double()
                if s["q_scale"] is not None:
                    q = (s["q"][b, h] * s["q_scale"][b, h].bfloat16()).double()
                x = kd[:, h // G] @ q / math.sqrt(_D)
                if s["bias"] is not None:
                    x[:n] += s["bias"][b, h if s["bias"].shape[1] > 1 else 0, :n].double()
                out[b, h] = torch.softmax(x, 0) @ vd[:, h // G]
        return out
    # sample: the log-probability of the token that the definition gives; the token itself is a whole number
    lp = []
    for b in range(c["B"]):
        x = s["logits"][b].double()
        t = float(s["temperature"][b])
        if t <= 0:
            lp.append(0.0)
            continue
        x = x / t
        w = (x - x.max()).exp()
        by = torch.argsort(s["logits"][b].float(), descending=True, stable=True)
        k = int(s["top_k"][b]) or c["V"]
        by = by[:k]
        cum = w[by].cumsum(0)
        if float(s["top_p"][b]) < 1:
            by = by[:int((cum < float(s["top_p"][b]) * cum[-1]).sum()) + 1]
        by = by[w[by] >= float(s["min_p"][b])].sort().values
        cum = w[by].cumsum(0)
        at = min(int((cum <= float(s["u"][b]) * cum[-1]).sum()), len(by) - 1)
        lp.append(float((w[by[at]] / cum[-1]).log()))
    return None, torch.tensor(lp, dtype=torch.float64)

"""The 4-bit KV cache on the B200 against plain 64-bit restatements.

Stored values are compared for equality: the restatement quantises in float64,
where (x - low) / scale + 1/2 is not within rounding of an integer unless it is
one (halves go up on both sides), and rounds low + code * scale to float32 and
then to bfloat16 as the definition says.

Attention tolerance, per element: 2^-8 |out| for the bf16 output (half an ulp
at most), 2^-10 sum_j p_j |v_j - z_j| for p * scale in fp16 (half an ulp of 11
bits, doubled; z_j = low + 8 scale), and 2^-12 sum_j p_j |v_j| for scores and
exponentials in fp32 (|score| < 64 here, so 2^-24 * 64 * a few from the sums
of 128 products, 2^-22 from the exponential).
"""
import math

import numpy as np
import pytest
import torch

from tokengate_b200 import _lib, ops
from tokengate_b200.kv4 import KV4Cache

pytestmark = pytest.mark.gpu


def quantise(x):
    """float64 (values, low + 8 scale) of bf16 rows (..., 128)."""
    g = x.double().cpu().unflatten(-1, (2, 64))
    low, high = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    scale = ((high / 2 - low / 2) / 7.5).float().bfloat16().double()
    scale[scale < 2.0 ** -100] = 0
    code = torch.where(scale > 0, torch.floor((g - low) / scale + 0.5), torch.zeros_like(g))
    val = (low + code * scale).float().bfloat16().double()
    exact = low + code * scale
    bad = ~(torch.isfinite(g).all(-1, keepdim=True) & (high - low < 3.4028235e38)).expand_as(g)
    val[bad] = exact[bad] = float("nan")
    return val.flatten(-2), exact.flatten(-2), (low + 8 * scale).expand_as(g).flatten(-2)


def rows(g, *shape):
    gain = torch.exp(0.5 * torch.randn(shape[-1], generator=g))
    return (torch.randn(*shape, generator=g) * gain + torch.randn(shape[-1], generator=g)).bfloat16()


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


# ------------------------------------------------------------------ store
@pytest.mark.parametrize("B,S,Hkv,start,cap", [
    (1, 1, 1, 0, 1), (1, 1, 8, 31, 33), (2, 16, 2, 0, 16), (1, 17, 4, 7, 64), (3, 77, 2, 99, 200),
    (1, 300, 8, 0, 300), (2, 33, 1, 15, 48), (1, 2768, 8, 3, 2800),
])
def test_write_then_read(cuda, B, S, Hkv, start, cap):
    g = torch.Generator().manual_seed(S + start)
    k, v = rows(g, B, S, Hkv, 128), rows(g, B, S, Hkv, 128)
    c = KV4Cache(B, cap, Hkv, device=cuda)
    c.data.fill_(0xA5)
    before_k, before_v = ops.kv4_read(c)
    ops.kv4_write(c, k.to(cuda), v.to(cuda), start=start)
    gk, gv = ops.kv4_read(c, start, S)
    assert same(gk.double().cpu(), quantise(k)[0])
    assert same(gv.double().cpu(), quantise(v)[0])
    # the slots around it are as they were
    ak, av = ops.kv4_read(c)
    for got, was in ((ak, before_k), (av, before_v)):
        got[:, start:start + S] = 0
        was[:, start:start + S] = 0
        assert same(got.float(), was.float())


def test_views_and_read_into_views(cuda):
    """K/V as views of a fused [q | k | v] projection, read back into (B, H, S, D) memory."""
    g = torch.Generator().manual_seed(5)
    qkv = rows(g, 2, 50, 8, 128).to(cuda)
    k, v = qkv[:, :, 4:6], qkv[:, :, 6:8]
    c = KV4Cache(2, 64, 2, device=cuda)
    ops.kv4_write(c, k, v, start=9)
    ko = torch.zeros(2, 2, 50, 128, dtype=torch.bfloat16, device=cuda)
    vo = torch.zeros_like(ko)
    ops.kv4_read(c, 9, 50, k_out=ko.transpose(1, 2), v_out=vo.transpose(1, 2))
    assert same(ko.transpose(1, 2).double().cpu(), quantise(k)[0])
    assert same(vo.transpose(1, 2).double().cpu(), quantise(v)[0])


def test_hard_rows(cuda):
    """Constant groups, zeros, halves, huge and tiny ranges, infinities and NaN."""
    x = torch.zeros(1, 10, 1, 128, dtype=torch.bfloat16)
    x[0, 0] = 3.140625
    x[0, 1, 0, 0::2] = -0.0
    x[0, 2, 0, :64] = torch.arange(64) * 0.5            # steps of 2.1: many halves of bf16's own
    x[0, 2, 0, 64:] = (torch.arange(64) % 31).float() / 2  # (x - low) / scale in halves exactly: scale 1
    x[0, 3, 0, 0], x[0, 3, 0, 1] = 3.0e38, -3.0e38      # a range past float32's largest: NaN
    x[0, 4, 0, 5], x[0, 4, 0, 70] = 1e-36, 2e-33         # ranges whose step is below 2^-100
    x[0, 5, 0, 7] = float("nan")
    x[0, 6, 0, 100] = float("inf")
    x[0, 7, 0, 3] = float("-inf")
    x[0, 8, 0, :] = torch.randn(128, generator=torch.Generator().manual_seed(1)).bfloat16() * 1e-20
    x[0, 9, 0, 9] = 1.0                                  # one outlier above 63 equals
    c = KV4Cache(1, 10, 1, device=cuda)
    ops.kv4_write(c, x.to(cuda), x.to(cuda))
    gk, gv = ops.kv4_read(c)
    want = quantise(x)[0]
    assert torch.isnan(want[0, 5, 0, :64]).all() and not torch.isnan(want[0, 5, 0, 64:]).any()
    assert same(gk.double().cpu(), want) and same(gv.double().cpu(), want)


def test_codes_next_to_halves(cuda):
    """The definition's own fp32 operations, bit for bit, on values at and beside half steps: halves go up, and so
    does what the reciprocal (2^-22 high) lifts to one."""
    f = np.float32
    tiny = [0.0] + [s * 10.0 ** -e for e in range(2, 9) for s in (1, -1, 3, -3)]
    x = torch.zeros(1, 12, 1, 128, dtype=torch.bfloat16)
    for r in range(12):
        low, step = -0.5 - r, [1.0, 0.75, 2.0, 0.3125][r % 4]
        for h in (0, 64):
            v = [low, low + 15 * step] + [low + (c + 0.5) * step for c in range(15)] + tiny + [t + low + 0.5 * step for t in tiny[:18]]
            x[0, r, 0, h:h + 64] = torch.tensor(v[:64]).clamp(low, low + 15 * step).bfloat16()
    c = KV4Cache(1, 12, 1, device=cuda)
    ops.kv4_write(c, x.to(cuda), x.to(cuda))
    gk, gv = ops.kv4_read(c)
    g = x.float().numpy().reshape(24, 64)
    low, high = g.min(1, keepdims=True), g.max(1, keepdims=True)
    scale = torch.from_numpy(((high * f(0.5) - low * f(0.5)) / f(7.5)).astype(f)).bfloat16().float().numpy()
    inv = ((f(1) / scale) * f(1 + 2.0 ** -22)).astype(f)
    code = np.floor(((g - low).astype(f) * inv).astype(f) + f(0.5)).astype(f)
    assert code.min() == 0 and code.max() == 15
    want = torch.from_numpy((low + code * scale).astype(f)).bfloat16().reshape(1, 12, 1, 128)
    assert torch.equal(gk.cpu(), want) and torch.equal(gv.cpu(), want)


def test_long_cache_offsets(cuda):
    """Slots whose byte offset passes 32 bits: 5.4 GB of cache, written and read near the end."""
    g = torch.Generator().manual_seed(8)
    cap = 4_700_032
    c = KV4Cache(1, cap, 8, device=cuda)
    k, v = rows(g, 1, 40, 8, 128), rows(g, 1, 40, 8, 128)
    ops.kv4_write(c, k.to(cuda), v.to(cuda), start=cap - 41)
    gk, gv = ops.kv4_read(c, cap - 41, 40)
    assert same(gk.double().cpu(), quantise(k)[0]) and same(gv.double().cpu(), quantise(v)[0])
    q = torch.randn(1, 16, 128, generator=g).bfloat16()
    bias = torch.full((1, 1, cap), float("-inf"), device=cuda)
    bias[..., cap - 41:cap - 1] = 0
    nv = torch.tensor([cap - 1], dtype=torch.int32, device=cuda)
    c.data[:, :, :-2].fill_(0)      # what was never written holds zeros here, not NaN
    out = ops.decode_attention_kv4(q.to(cuda), c, nv, cap, cap, bias=bias)
    ref, tol = attend(q, k, v, [40], 40, 40, None, None)
    assert ((out.double().cpu() - ref).abs() <= tol).all()


def test_a_copied_cache_leaves_the_original_alone(cuda):
    import copy
    g = torch.Generator().manual_seed(15)
    k, v = rows(g, 1, 40, 2, 128), rows(g, 1, 40, 2, 128)
    c = KV4Cache(1, 40, 2, device=cuda)
    ops.kv4_write(c, k.to(cuda), v.to(cuda))
    was = c.data.clone()
    d = copy.deepcopy(c)
    ops.kv4_write(d, v.to(cuda), k.to(cuda))
    assert torch.equal(c.data, was)
    assert same(ops.kv4_read(d)[0].double().cpu(), quantise(v)[0]) and same(ops.kv4_read(c)[0].double().cpu(), quantise(k)[0])


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("B,Hq,Hkv,slot,cap", [(1, 16, 8, 0, 1), (1, 4, 1, 40, 64), (3, 8, 8, 31, 32), (5, 16, 2, 99, 100),
                                              (64, 32, 8, 17, 40)])
def test_append(cuda, B, Hq, Hkv, slot, cap):
    g = torch.Generator().manual_seed(B + slot)
    qkv = rows(g, B, 1, Hq + 2 * Hkv, 128).to(cuda)
    q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]
    qw, kw = ((1 + 0.3 * torch.randn(128, generator=g)).bfloat16().to(cuda) for _ in range(2))
    ang = torch.randn(B, 1, 64, generator=g) * 50
    cos, sin = (torch.cat([f(ang)] * 2, -1).bfloat16().to(cuda) for f in (torch.cos, torch.sin))
    c = KV4Cache(B, cap, Hkv, device=cuda)
    c.data.fill_(0x5A)
    was = c.data.clone()
    keep = qkv.clone()
    sl = torch.tensor([slot], dtype=torch.int64, device=cuda)
    out = ops.qk_norm_rope_append_kv4(q, k, v, qw, kw, cos, sin, 1e-6, c, sl)
    assert torch.equal(qkv, keep)

    def turned(x, w):     # float64 of the definition
        x = x.double().cpu()
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.double().cpu()
        rot = torch.cat([-y[..., 64:], y[..., :64]], -1)
        return y * cos.double().cpu()[:, :, None] + rot * sin.double().cpu()[:, :, None]

    # q: the definition within the fp32 chain's error (a few roundings of terms as large as the head's
    # largest value: 2^-20 of it), then one bf16 rounding, which is monotone
    want = turned(q, qw)
    slack = 2 ** -20 * want.abs().amax(-1, keepdim=True)
    got = out.double().cpu()
    assert ((got >= (want - slack).bfloat16().double()) & (got <= (want + slack).bfloat16().double())).all()
    gk, gv = ops.kv4_read(c, slot, 1)
    assert same(gv.double().cpu(), quantise(v)[0])
    # k: within half a step of the turned key, and a bf16 rounding on either side
    wk = turned(k, kw)
    grp = wk.unflatten(-1, (2, 64))
    step = ((grp.amax(-1, keepdim=True) - grp.amin(-1, keepdim=True)) / 15).expand_as(grp).flatten(-2)
    top = grp.abs().amax(-1, keepdim=True).expand_as(grp).flatten(-2)
    assert ((gk.double().cpu() - wk).abs() <= 0.5 * step * (1 + 2 ** -7) + 2 ** -7 * top).all()
    # and exactly the quantised bf16 key: what the bulk write makes of the same rows
    kb = turned(k, kw).float().bfloat16()
    c2 = KV4Cache(B, cap, Hkv, device=cuda)
    ops.kv4_write(c2, kb.to(cuda), v, start=slot)
    near = (ops.kv4_read(c2, slot, 1)[0].double() - gk.double()).abs().cpu() <= 2 ** -6 * top
    assert near.double().mean() > 0.999        # a bf16 rounding may fall the other way and move a code
    # in place, and a slot outside the cache writes nothing
    c.data.copy_(was)
    q2 = q.clone()
    r = ops.qk_norm_rope_append_kv4(q2, k, v, qw, kw, cos, sin, 1e-6, c, torch.tensor([cap], device=cuda), q_out=q2)
    assert r is q2 and torch.equal(q2, out) and torch.equal(c.data, was)


def test_append_of_one_row_takes_any_row_stride(cuda):
    """Strides of dims of one are not used, whatever a view left there; those of more rows must be alike."""
    g = torch.Generator().manual_seed(16)
    q, k, v = rows(g, 1, 1, 4, 128).to(cuda), rows(g, 1, 1, 2, 128).to(cuda), rows(g, 1, 1, 2, 128).to(cuda)
    w = rows(g, 128).to(cuda)
    cos, sin = (torch.randn(1, 1, 128, generator=g).bfloat16().to(cuda) for _ in range(2))
    sl = torch.tensor([3], dtype=torch.int64, device=cuda)
    a, b = KV4Cache(1, 9, 2, device=cuda), KV4Cache(1, 9, 2, device=cuda)
    a.data.zero_()
    b.data.zero_()
    want = ops.qk_norm_rope_append_kv4(q, k, v, w, w, cos, sin, 1e-6, a, sl)
    odd = lambda t: t.as_strided(t.shape, (0, 3) + t.stride()[2:])  # noqa: E731
    got = ops.qk_norm_rope_append_kv4(odd(q), odd(k), v.as_strided(v.shape, (5, 1, 128, 1)), w, w, odd(cos), sin, 1e-6, b, sl)
    assert torch.equal(got, want) and torch.equal(a.data, b.data)
    two = torch.zeros(2, 1, 4, 128, dtype=torch.bfloat16, device=cuda)
    c2 = KV4Cache(2, 9, 2, device=cuda)
    cs = torch.zeros(2, 1, 128, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError, match="strides"):
        ops.qk_norm_rope_append_kv4(two, two[:, :, :2], two[:, :, 2:], w, w, cs, cs[:1].expand(2, -1, -1), 1e-6, c2, sl)


@pytest.mark.parametrize("B,Hkv,slot", [(1, 1, 0), (3, 2, 37), (64, 8, 95)])
def test_append_is_the_bulk_write_of_its_key(cuda, B, Hkv, slot):
    """The slot's bytes are those of a bulk write of the same bf16 key, which the q heads give: the same rows through
    the same arithmetic, handed out."""
    g = torch.Generator().manual_seed(B)
    k, v = rows(g, B, 1, Hkv, 128).to(cuda), rows(g, B, 1, Hkv, 128).to(cuda)
    w = (1 + 0.3 * torch.randn(128, generator=g)).bfloat16().to(cuda)
    ang = torch.randn(B, 1, 64, generator=g) * 50
    cos, sin = (torch.cat([f(ang)] * 2, -1).bfloat16().to(cuda) for f in (torch.cos, torch.sin))
    a, b = KV4Cache(B, 96, Hkv, device=cuda), KV4Cache(B, 96, Hkv, device=cuda)
    a.data.fill_(0x3C)
    b.data.fill_(0x3C)
    key = ops.qk_norm_rope_append_kv4(k, k, v, w, w, cos, sin, 1e-6, a, torch.tensor([slot], dtype=torch.int64, device=cuda))
    ops.kv4_write(b, key, v, start=slot)
    assert torch.equal(a.data, b.data)


# ------------------------------------------------------------------ attention
def attend(q, k, v, n_valid, n_prefix, n_keys, bias, q_scale):
    """float64 (output, tolerance) of the definition over the values that the cache stands for."""
    B, Hq, D = q.shape
    qd = q.double()
    if q_scale is not None:
        qd = (q.float() * q_scale.bfloat16().float()[..., None]).bfloat16().double()
    (_, kd, _), (_, vd, vz) = quantise(k), quantise(v)
    G = Hq // k.shape[2]
    out, tol = torch.zeros(B, Hq, D, dtype=torch.float64), torch.zeros(B, Hq, D, dtype=torch.float64)
    for b in range(B):
        at = [j for j in range(n_keys) if j < n_valid[b] or j >= n_prefix]
        if not at:
            continue
        for h in range(Hq):
            x = kd[b, at, h // G] @ qd[b, h] * D ** -0.5
            if bias is not None:
                bb = torch.zeros(n_keys, dtype=torch.float64)
                bb[:n_prefix] = bias[b, h if bias.shape[1] > 1 else 0, :n_prefix].double()
                x = (x + bb[at]) if bb[at].min() > -1e30 else (x.float() + bb[at].float()).double()
            if x.max() == -math.inf:
                continue
            p = torch.softmax(x, 0)
            vv, zz = vd[b, at, h // G], vz[b, at, h // G]
            out[b, h] = p @ vv
            tol[b, h] = 2 ** -8 * out[b, h].abs() + 2 ** -10 * (p @ (vv - zz).abs()) + 2 ** -12 * (p @ vv.abs()) + 1e-30
    return out, tol


def check_attend(cuda, q, k, v, valid, n_prefix, n_keys, bias=None, qs=None, cap=None, dev_keys=None):
    B, Hkv = q.shape[0], k.shape[2]
    c = KV4Cache(B, cap or n_keys, Hkv, device=cuda)
    c.data.fill_(0xFF)              # slots never written hold NaN steps
    ops.kv4_write(c, k.to(cuda), v.to(cuda))
    nv = torch.tensor(valid, dtype=torch.int32, device=cuda)
    kw = {} if dev_keys is None else dict(n_keys_dev=torch.tensor([n_keys], dtype=torch.int32, device=cuda))
    out = ops.decode_attention_kv4(q.to(cuda), c, nv, n_prefix, dev_keys or n_keys,
                                   bias=None if bias is None else bias.to(cuda),
                                   q_scale=None if qs is None else qs.to(cuda), **kw)
    ref, tol = attend(q, k, v, valid, n_prefix, n_keys, bias, qs)
    err = (out.double().cpu() - ref).abs()
    assert (err <= tol).all(), (err / tol).max()
    return out


@pytest.mark.parametrize("B,Hq,Hkv,n_prefix,n_keys,valid,bias_kind,qs", [
    (1, 16, 8, 2768, 2771, [2700], "head", True),
    (2, 4, 2, 100, 103, [100, 57], "row", False),
    (3, 8, 8, 256, 256, [256, 1, 200], "head", False),
    (1, 16, 2, 300, 520, [300], "row", True),
    (2, 16, 8, 1, 1, [1, 1], None, True),
    (1, 1, 1, 1, 1, [1], "row", False),
    (2, 6, 2, 33, 34, [0, 33], None, False),        # three query heads per KV head
    (3, 7, 1, 64, 64, [64, 0, 5], None, False),     # a row without any key
    (1, 8, 4, 0, 19, [0], None, False),             # decoded keys only
    (2, 32, 8, 5000, 5001, [5000, 31], None, False),
])
def test_attention(cuda, B, Hq, Hkv, n_prefix, n_keys, valid, bias_kind, qs):
    g = torch.Generator().manual_seed(n_keys + B)
    q = torch.randn(B, Hq, 128, generator=g).bfloat16()
    k, v = rows(g, B, n_keys, Hkv, 128), rows(g, B, n_keys, Hkv, 128)
    k /= 2
    for b in range(B):   # pad slots hold rubbish
        k[b, valid[b]:n_prefix] = float("nan")
        v[b, valid[b]:n_prefix] = float("inf")
    bias = None
    if bias_kind:
        bias = torch.randn(B, Hq if bias_kind == "head" else 1, n_prefix, generator=g) * 2
    q_scale = 0.5 + torch.rand(B, Hq, generator=g) if qs else None
    check_attend(cuda, q, k, v, valid, n_prefix, n_keys, bias, q_scale, cap=n_keys + 40)
    check_attend(cuda, q, k, v, valid, n_prefix, n_keys, bias, q_scale, cap=n_keys + 200, dev_keys=n_keys + 150)


@pytest.mark.parametrize("B,Hq,Hkv,n_prefix,n_keys,bias_kind", [
    (40, 2, 1, 70, 75, "row"),          # blocks shared among more rows than a warp holds at once
    (70, 6, 3, 40, 40, None),           # more rows than a wave of blocks
    (33, 4, 4, 260, 260, "head"),
    (2, 40, 5, 700, 705, "row"),        # eight query heads per KV head, an odd number of them
    (5, 14, 2, 3000, 3001, "head"),     # seven
    (1, 3, 1, 20000, 20000, None),
    (20, 16, 8, 500, 501, None),
])
def test_attention_unlike_rows(cuda, B, Hq, Hkv, n_prefix, n_keys, bias_kind):
    """Rows of every length from none to all, so that blocks are shared unevenly."""
    g = torch.Generator().manual_seed(n_keys * B)
    q = torch.randn(B, Hq, 128, generator=g).bfloat16()
    k, v = rows(g, B, n_keys, Hkv, 128) / 2, rows(g, B, n_keys, Hkv, 128)
    valid = [(n_prefix * b * b) // max((B - 1) ** 2, 1) for b in range(B)]
    valid[B // 3] = 0
    for b in range(B):
        k[b, valid[b]:n_prefix] = float("nan")
    bias = None if bias_kind is None else torch.randn(B, Hq if bias_kind == "head" else 1, n_prefix, generator=g)
    check_attend(cuda, q, k, v, valid, n_prefix, n_keys, bias)


@pytest.mark.parametrize("B,Hkv", [(37, 8), (38, 8), (49, 8), (50, 8), (75, 4), (148, 1), (149, 2)])
@pytest.mark.parametrize("n", [33, 500])
def test_attention_of_many_rows(cuda, B, Hkv, n):
    """Batches about as large as the number of blocks that a KV head has, even and unlike rows."""
    g = torch.Generator().manual_seed(B)
    q = torch.randn(B, Hkv, 128, generator=g).bfloat16()
    k, v = rows(g, B, n, Hkv, 128) / 2, rows(g, B, n, Hkv, 128)
    check_attend(cuda, q, k, v, [n] * B, n, n)
    check_attend(cuda, q, k, v, [(7 * b) % (n + 1) for b in range(B)], n, n)


@pytest.mark.parametrize("B", [37, 38, 49, 50])
def test_attention_of_many_long_rows(cuda, B):
    """The same where rows are long enough to take several blocks each; every row holds the same keys."""
    g = torch.Generator().manual_seed(B)
    n = 2100
    q = torch.randn(B, 8, 128, generator=g).bfloat16()
    k, v = rows(g, 1, n, 8, 128) / 2, rows(g, 1, n, 8, 128)
    c = KV4Cache(B, n, 8, device=cuda)
    ops.kv4_write(c, k.to(cuda).expand(B, -1, -1, -1), v.to(cuda).expand(B, -1, -1, -1))
    for valid in ([n] * B, [n * b // (B - 1) for b in range(B)]):
        out = ops.decode_attention_kv4(q.to(cuda), c, torch.tensor(valid, dtype=torch.int32, device=cuda), n, n).cpu()
        for b in range(0, B, 3):
            ref, tol = attend(q[b:b + 1], k, v, [valid[b]], n, n, None, None)
            assert ((out[b:b + 1].double() - ref).abs() <= tol).all(), b


@pytest.mark.parametrize("B,Hq,Hkv", [(1, 4, 4), (3, 16, 2), (40, 8, 8)])
def test_attention_of_one_key(cuda, B, Hq, Hkv):
    """A single key's value comes back as the bf16 rounding of something within p s's rounding (2^-11 of code - 8
    steps) and the cut of the products (2^-14 of a step each, two to a value: 2^-13); other slots masked."""
    g = torch.Generator().manual_seed(Hq)
    q = (3 * torch.randn(B, Hq, 128, generator=g)).bfloat16()
    k, v = rows(g, B, 70, Hkv, 128), rows(g, B, 70, Hkv, 128)
    c = KV4Cache(B, 70, Hkv, device=cuda)
    ops.kv4_write(c, k.to(cuda), v.to(cuda))
    _, exact, zero = quantise(v)
    groups = v.double().unflatten(-1, (2, 64))
    step = ((groups.amax(-1, keepdim=True) - groups.amin(-1, keepdim=True)) / 15).expand_as(groups).flatten(-2) * 1.01
    for j, n_prefix in ((0, 0), (69, 69)):   # the first slot, decoded; the last one behind a masked prompt
        n_valid = torch.zeros(B, dtype=torch.int32, device=cuda)
        out = ops.decode_attention_kv4(q.to(cuda), c, n_valid, n_prefix, j + 1).cpu()
        e, z, s = (t[:, j].repeat_interleave(Hq // Hkv, dim=1) for t in (exact, zero, step))
        slack = 2 ** -11 * (e - z).abs() + 2 ** -13 * s
        assert ((out >= (e - slack).bfloat16()) & (out <= (e + slack).bfloat16())).all()


def test_attention_without_keys_on_the_device(cuda):
    """A device-side count of none (or below): zeros, in both ways of merging."""
    for B, n in ((1, 300), (3, 9000)):
        c = KV4Cache(B, n, 2, device=cuda)
        c.data.fill_(0xFF)
        nv = torch.full((B,), n, dtype=torch.int32, device=cuda)
        for count in (0, -1, -1000):
            nk = torch.tensor([count], dtype=torch.int32, device=cuda)
            out = ops.decode_attention_kv4(torch.ones(B, 4, 128, dtype=torch.bfloat16, device=cuda), c, nv, n, n, n_keys_dev=nk)
            assert (out == 0).all()


def test_attention_masks_of_lowest_value(cuda):
    """-1e9, the type's lowest value and -inf as biases: beside ordinary keys they get no weight, a row
    of the lowest value alone is uniform (as the fp32 sum makes it), a row of -inf alone gives zeros."""
    g = torch.Generator().manual_seed(3)
    q, k, v = torch.randn(1, 8, 128, generator=g).bfloat16(), rows(g, 1, 70, 4, 128), rows(g, 1, 70, 4, 128)
    bias = torch.zeros(1, 8, 70)
    bias[0, 0, ::2] = -1e9
    bias[0, 1, 1:] = torch.finfo(torch.float32).min
    bias[0, 2] = torch.finfo(torch.float32).min
    bias[0, 3] = float("-inf")
    bias[0, 4, :69] = float("-inf")
    bias[0, 5, 40:] = torch.finfo(torch.float32).min
    out = check_attend(cuda, q, k, v, [70], 70, 70, bias)
    assert (out[0, 3] == 0).all()


def test_attention_nan_key_stays_in_its_row(cuda):
    """A NaN in a key that is attended is in its KV head's output; NaN in V only in that group of dims."""
    g = torch.Generator().manual_seed(4)
    q, k, v = torch.randn(2, 8, 128, generator=g).bfloat16(), rows(g, 2, 50, 4, 128), rows(g, 2, 50, 4, 128)
    k[0, 20, 1, 3] = float("nan")
    v[1, 30, 2, 100] = float("nan")
    c = KV4Cache(2, 50, 4, device=cuda)
    ops.kv4_write(c, k.to(cuda), v.to(cuda))
    out = ops.decode_attention_kv4(q.to(cuda), c, torch.tensor([50, 50], dtype=torch.int32, device=cuda), 50, 50)
    bad = torch.zeros(2, 8, 128, dtype=torch.bool)
    bad[0, 2:4] = True
    bad[1, 4:6, 64:] = True
    assert torch.equal(torch.isnan(out).cpu(), bad)


@pytest.mark.parametrize("qm,km,vm", [(1e4, 1e-4, 1.0), (1e-30, 1e28, 1e30), (1.0, 1.0, 1e-30), (3e37, 1e-37, 1e30), (0.0, 1.0, 1.0)])
def test_attention_magnitudes(cuda, qm, km, vm):
    """Queries, keys and values far outside fp16's range."""
    g = torch.Generator().manual_seed(6)
    q = (torch.randn(1, 4, 128, generator=g) * qm).bfloat16()
    k, v = (torch.randn(1, 90, 2, 128, generator=g) * km).bfloat16(), (torch.randn(1, 90, 2, 128, generator=g) * vm / 4).bfloat16()
    v[0, :30] *= 2.0 ** -9      # steps that grow along the keys
    check_attend(cuda, q, k, v, [90], 90, 90)


def test_attention_growing_scores(cuda):
    """Scores that climb by tens along the cache: the running maximum moves at every tile."""
    g = torch.Generator().manual_seed(7)
    q = torch.randn(1, 2, 128, generator=g).bfloat16()
    k, v = rows(g, 1, 700, 1, 128), rows(g, 1, 700, 1, 128)
    bias = torch.linspace(0, 40, 700).repeat(1, 1, 1)
    check_attend(cuda, q, k, v, [700], 700, 700, bias)
    check_attend(cuda, q, k, v, [700], 700, 700, -bias)


@pytest.mark.parametrize("n", [100, 2771, 32768])
def test_what_four_bits_cost(cuda, n):
    """Against attention over the bf16 rows. With errors of a value uniform over its step (variance step^2 / 12), of a
    score s_j = scale * sqrt(sum q^2 step_k^2 / 12), the output's variance is sum_j p_j^2 (step_v^2 / 12 + s_j^2 (v_j -
    out)^2), to first order. The errors' mean square over 2048 outputs is within 1.5^2 of that, and not far below."""
    g = torch.Generator().manual_seed(n)
    Hq, Hkv = 16, 8
    q, k, v = torch.randn(1, Hq, 128, generator=g).bfloat16(), rows(g, 1, n, Hkv, 128), rows(g, 1, n, Hkv, 128)
    c = KV4Cache(1, n, Hkv, device=cuda)
    ops.kv4_write(c, k.to(cuda), v.to(cuda))
    out = ops.decode_attention_kv4(q.to(cuda), c, torch.tensor([n], dtype=torch.int32, device=cuda), n, n)[0].double()
    kd, vd, qd = k[0].double().to(cuda), v[0].double().to(cuda), q[0].double().to(cuda)
    step = lambda x: ((x.unflatten(-1, (2, 64)).amax(-1) - x.unflatten(-1, (2, 64)).amin(-1)) / 15).repeat_interleave(64, -1)  # noqa: E731
    want, var = torch.zeros_like(out), torch.zeros_like(out)
    for h in range(Hq):
        kh, vh = kd[:, h // 2], vd[:, h // 2]
        p = torch.softmax(kh @ qd[h] * 128 ** -0.5, 0)
        want[h] = p @ vh
        s2 = (step(kh) ** 2 / 12) @ qd[h] ** 2 / 128
        var[h] = (p ** 2) @ (step(vh) ** 2 / 12 + s2[:, None] * (vh - want[h]) ** 2)
    got, guess, size = (((out - want) ** 2).mean().sqrt().item(), var.mean().sqrt().item(), (want ** 2).mean().sqrt().item())
    print(f"{n} keys: relative error {got / size:.4f}, expected {guess / size:.4f}")
    assert 0.5 * guess <= got <= 1.5 * guess + 2 ** -9 * size


def test_attention_strides_stream_and_graph(cuda):
    """Strided q, out and bias; a stream of its own; the same call captured and replayed while the cache grows."""
    g = torch.Generator().manual_seed(9)
    big = torch.randn(2, 12, 128, generator=g).bfloat16().to(cuda)
    q = big[:, 2:10]
    k, v = rows(g, 2, 400, 4, 128), rows(g, 2, 400, 4, 128)
    bias = torch.randn(2, 8, 600, generator=g).to(cuda)[:, :, 100:500]
    c = KV4Cache(2, 420, 4, device=cuda)
    ops.kv4_write(c, k.to(cuda), v.to(cuda))
    nv = torch.tensor([390, 300], dtype=torch.int32, device=cuda)
    out = torch.zeros(2, 20, 128, dtype=torch.bfloat16, device=cuda)
    nk = torch.tensor([395], dtype=torch.int32, device=cuda)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.decode_attention_kv4(q, c, nv, 390, 400, bias=bias, out=out[:, 5:13], n_keys_dev=nk)
    torch.cuda.current_stream().wait_stream(s)
    ref, tol = attend(q.cpu(), k, v, [390, 300], 390, 395, bias.cpu(), None)
    assert ((out[:, 5:13].double().cpu() - ref).abs() <= tol).all() and (out[:, :5] == 0).all() and (out[:, 13:] == 0).all()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        cap = ops.decode_attention_kv4(q, c, nv, 390, 400, bias=bias, n_keys_dev=nk)
    for n in (391, 400):
        nk.fill_(n)
        gr.replay()
        ref, tol = attend(q.cpu(), k, v, [390, 300], 390, n, bias.cpu(), None)
        assert ((cap.double().cpu() - ref).abs() <= tol).all()


def test_attention_repeats_bit_for_bit(cuda):
    g = torch.Generator().manual_seed(10)
    q, k, v = torch.randn(2, 16, 128, generator=g).bfloat16().to(cuda), rows(g, 2, 3000, 8, 128), rows(g, 2, 3000, 8, 128)
    c = KV4Cache(2, 3000, 8, device=cuda)
    ops.kv4_write(c, k.to(cuda), v.to(cuda))
    nv = torch.tensor([3000, 2500], dtype=torch.int32, device=cuda)
    a = ops.decode_attention_kv4(q, c, nv, 3000, 3000)
    assert all(torch.equal(a, ops.decode_attention_kv4(q, c, nv, 3000, 3000)) for _ in range(5))


def _masked(cuda, G, value, at, spoil, n=300):
    """A batch of two rows whose keys `at` a bias of `value` masks, with their V rows as `spoil` makes them."""
    g = torch.Generator().manual_seed(G + n)
    q, k, v = torch.randn(2, 2 * G, 128, generator=g).bfloat16(), rows(g, 2, n, 2, 128) / 2, rows(g, 2, n, 2, 128)
    bias = torch.randn(2, 1, n, generator=g)
    bias[..., at] = value
    c = KV4Cache(2, n, 2, device=cuda)
    held = v.clone()
    if isinstance(spoil, float):
        v[:, at] *= spoil
    ops.kv4_write(c, k.to(cuda), v.to(cuda))
    if not isinstance(spoil, float):       # bytes of the two groups' steps and lows (4352: V's parameters in a tile)
        for j in at:
            c.data[:, :, j // 32, 4352 + 8 * (j % 32):4360 + 8 * (j % 32)] = torch.tensor(spoil, dtype=torch.uint8, device=cuda)
    out = ops.decode_attention_kv4(q.to(cuda), c, torch.tensor([n, n], dtype=torch.int32, device=cuda), n, n, bias=bias.to(cuda))
    ref, tol = attend(q, k, held, [n, n], n, n, bias, None)
    err = (out.double().cpu() - ref).abs()
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("G", [2, 4, 8])
@pytest.mark.parametrize("value", [float("-inf"), -1e9, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("at", [[0], [150], [299], list(range(0, 300, 2)), list(range(100)), list(range(64, 300))])
def test_attention_masked_keys_weigh_nothing(cuda, G, value, at):
    """Keys that the bias masks, at either end and between, whatever their V's range: up to bf16's largest, an
    infinite step, and (behind -inf, where nothing is read as a number) NaN."""
    for spoil in (1e10, 1e30, 1e37):
        _masked(cuda, G, value, at, spoil)
    inf, big, nan = [0x80, 0x7F, 0, 0], [0x7F, 0x7F, 0x7F, 0xFF], [0xC0, 0x7F, 0xC0, 0x7F]
    _masked(cuda, G, value, at, inf + inf)
    _masked(cuda, G, value, at, big + inf)
    if value == -math.inf:
        _masked(cuda, G, value, at, nan + big)


@pytest.mark.parametrize("n,B,Hq,Hkv", [(40, 1, 2, 1), (700, 3, 16, 2), (9000, 1, 4, 2)])
def test_attention_rubbish_behind_a_bias(cuda, n, B, Hq, Hkv):
    """Slots that were never written hold random bytes, in K too: a bias of -inf hides them."""
    g = torch.Generator().manual_seed(n)
    q, k, v = torch.randn(B, Hq, 128, generator=g).bfloat16(), rows(g, B, n, Hkv, 128) / 2, rows(g, B, n, Hkv, 128)
    c = KV4Cache(B, n, Hkv, device=cuda)
    c.data.copy_(torch.randint(0, 256, c.data.shape, generator=g).to(torch.uint8))
    lo, hi = n // 3, n // 3 + 20
    ops.kv4_write(c, k[:, lo:hi].to(cuda), v[:, lo:hi].to(cuda), start=lo)
    bias = torch.full((B, 1, n), float("-inf"))
    bias[..., lo:hi] = torch.randn(B, 1, 20, generator=g)
    out = ops.decode_attention_kv4(q.to(cuda), c, torch.full((B,), n, dtype=torch.int32, device=cuda), n, n, bias=bias.to(cuda))
    ref, tol = attend(q, k[:, lo:hi], v[:, lo:hi], [20] * B, 20, 20, bias[..., lo:hi], None)
    assert ((out.double().cpu() - ref).abs() <= tol).all()


def test_long_cache_of_rubbish(cuda):
    """5.4 GB of random bytes behind a bias of -inf, and 40 keys."""
    g = torch.Generator().manual_seed(8)
    cap = 4_700_032
    c = KV4Cache(1, cap, 8, device=cuda)
    c.data.random_(0, 256)
    q, k, v = torch.randn(1, 16, 128, generator=g).bfloat16(), rows(g, 1, 40, 8, 128), rows(g, 1, 40, 8, 128)
    for at in (cap - 41, 1_000_003):
        ops.kv4_write(c, k.to(cuda), v.to(cuda), start=at)
        bias = torch.full((1, 1, cap), float("-inf"), device=cuda)
        bias[..., at:at + 40] = 0
        out = ops.decode_attention_kv4(q.to(cuda), c, torch.tensor([cap], dtype=torch.int32, device=cuda), cap, cap, bias=bias)
        ref, tol = attend(q, k, v, [40], 40, 40, None, None)
        assert ((out.double().cpu() - ref).abs() <= tol).all()


@pytest.mark.parametrize("G", [1, 4, 8])
@pytest.mark.parametrize("apart", [1e4, 1e5, 1e6, 1e7, 1e8, 1e10, 1e20])
def test_attention_groups_of_unlike_steps(cuda, G, apart):
    """The two groups of a row's values far apart, in either order, few and many keys, with and without a bias."""
    g = torch.Generator().manual_seed(G)
    for n in (1, 90, 2100):
        q, k, v = torch.randn(1, 2 * G, 128, generator=g).bfloat16(), rows(g, 1, n, 2, 128), rows(g, 1, n, 2, 128)
        bias = torch.randn(1, 2 * G, n, generator=g)
        for half in (slice(0, 64), slice(64, 128)):
            w = v.clone()
            w[..., half] /= apart
            check_attend(cuda, q, k, w, [n], n, n)
            check_attend(cuda, q, k, w, [n], n, n, bias)


def test_attention_heads_of_unlike_values(cuda):
    """Keys that hold values 1e8 times the others', of weight in one head of a KV head and of none in the rest; and
    values that shrink along the cache while the scores grow."""
    g = torch.Generator().manual_seed(12)
    for G in (2, 4, 8):
        n = 400
        q, k, v = torch.randn(1, 2 * G, 128, generator=g).bfloat16(), rows(g, 1, n, 2, 128) / 2, rows(g, 1, n, 2, 128)
        v[:, 30] *= 1e8
        v[:, 390] *= 1e12
        bias = torch.randn(1, 2 * G, n, generator=g)
        bias[:, 1::2, 30] = bias[:, 1::2, 390] = -90.0
        check_attend(cuda, q, k, v, [n], n, n, bias)
        w = rows(g, 1, n, 2, 128) * torch.logspace(12, 0, n)[None, :, None, None].bfloat16()
        check_attend(cuda, q, k, w, [n], n, n, torch.linspace(-200, 0, n).repeat(1, 1, 1))


@pytest.mark.parametrize("G", [2, 8])
@pytest.mark.parametrize("apart", [1e4, 1e6, 1e8, 1e10])
def test_attention_groups_of_unlike_queries(cuda, G, apart):
    """Large keys meet small queries in one group of dims, in the other the reverse: both count in the scores."""
    g = torch.Generator().manual_seed(G)
    n = 200
    for half in (slice(0, 64), slice(64, 128)):
        q, k, v = torch.randn(1, 2 * G, 128, generator=g).bfloat16(), rows(g, 1, n, 2, 128), rows(g, 1, n, 2, 128)
        q[..., half] /= apart
        k[..., half] *= apart
        check_attend(cuda, q, k, v, [n], n, n)


# ------------------------------------------------------------------ refusals
def test_refusals(cuda):
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=cuda)  # noqa: E731
    c = KV4Cache(1, 10, 2, device=cuda)
    nv = torch.tensor([5], dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError):
        KV4Cache(0, 10, 2, device=cuda)
    with pytest.raises(ValueError, match="CUDA"):
        KV4Cache(1, 10, 2, device="cpu")
    with pytest.raises(TypeError):
        ops.kv4_write(c.data, z(1, 3, 2, 128), z(1, 3, 2, 128))
    for k in (z(1, 3, 3, 128), z(2, 3, 2, 128), z(1, 3, 2, 64), z(1, 3, 2, 128).float(), z(1, 3, 128, 2).transpose(2, 3)):
        with pytest.raises(ValueError):
            ops.kv4_write(c, k, k)
    with pytest.raises(ValueError):
        ops.kv4_write(c, z(1, 3, 2, 128), z(1, 2, 2, 128))
    for start in (-1, 8):
        with pytest.raises(ValueError):
            ops.kv4_write(c, z(1, 3, 2, 128), z(1, 3, 2, 128), start=start)
        with pytest.raises(ValueError):
            ops.kv4_read(c, start, 3)
    odd = torch.zeros(1, 3, 2, 132, dtype=torch.bfloat16, device=cuda)[..., 1:129]
    with pytest.raises(ValueError):                                          # rows off a 16-byte boundary
        ops.kv4_write(c, odd, odd)
    ops.kv4_write(c, z(1, 0, 2, 128), z(1, 0, 2, 128))                       # nothing to write
    assert ops.kv4_read(c, 10, 0)[0].shape == (1, 0, 2, 128)
    with pytest.raises(ValueError):
        ops.decode_attention_kv4(z(1, 4, 128), c, nv, 5, 11)                 # beyond the capacity
    with pytest.raises(ValueError):
        ops.decode_attention_kv4(z(1, 4, 128), c, nv, 6, 5)                  # prefix past n_keys
    with pytest.raises(ValueError):
        ops.decode_attention_kv4(z(2, 4, 128), c, nv, 5, 5)
    with pytest.raises(ValueError):
        ops.decode_attention_kv4(z(1, 4, 128), c, nv.long(), 5, 5)
    with pytest.raises(ValueError):
        ops.decode_attention_kv4(z(1, 3, 128), c, nv, 5, 5)                  # 3 query heads on 2 KV heads
    with pytest.raises(ValueError):
        ops.decode_attention_kv4(z(1, 4, 128), c, nv, 5, 5, bias=torch.zeros(1, 4, 4, device=cuda))
    with pytest.raises(_lib.TokenGateUnsupportedError):
        ops.decode_attention_kv4(z(1, 18, 128), c, nv, 5, 5)                 # 9 per KV head
    sl = torch.tensor([0], dtype=torch.int64, device=cuda)
    a = (z(1, 1, 4, 128), z(1, 1, 2, 128), z(1, 1, 2, 128), z(128), z(128), z(1, 1, 128), z(1, 1, 128), 1e-6, c)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_append_kv4(*a, sl.int())
    with pytest.raises(ValueError):
        ops.qk_norm_rope_append_kv4(a[0], z(1, 1, 4, 128), *a[2:], sl)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_append_kv4(z(1, 2, 4, 128), *a[1:], sl)


def test_a_device_count_of_no_element_is_refused(cuda):
    """An empty tensor has no address, which would read as no count at all."""
    c = KV4Cache(1, 10, 2, device=cuda)
    nv = torch.tensor([5], dtype=torch.int32, device=cuda)
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16, device=cuda)
    for bad in (nv[:0], nv.expand(2)):
        with pytest.raises(ValueError, match="n_keys_dev"):
            ops.decode_attention_kv4(q, c, nv, 5, 5, n_keys_dev=bad)

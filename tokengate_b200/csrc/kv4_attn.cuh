// Decode attention over the 4-bit KV cache (layout: kv4.cuh): the same
// operation as decode_attn.cuh, one query token per (batch row, head),
//   out = softmax_j( softmax_scale * (q' . k_j) + m_j ) V
// with k_j, v_j the values that the codes stand for, low + code * scale.
//
// Per group of 64 dims a value is low + s * code, so
//   q . k         = sum over the row's two groups of  s * (q . code) + low * sum(q)
//   sum_j p_j v_j = sum_j (p_j s_j) code_j + sum_j p_j low_j
// and the tensor cores multiply by the small integers themselves, exact in
// fp16; scales and lows enter in fp32 outside the products. K is the A operand
// (16 keys x 16 dims, m16n8k16) against the heads of one kv head as the 8
// columns; V^T is A (16 dims x 16 keys) against the probabilities. A pair of
// nibbles, masked, IS a pair of fp16 numbers: below 2^11 fp16's bits are linear
// (subnormals and the first binade), so the nibble at bit 0 reads code * 2^-24
// and the one at bit 4 code * 2^-20: five logic instructions unpack eight codes.
// The factors 2^-24 and 2^-20 go into q' (K: each nibble meets its own dim) and
// into the final sums (V: each nibble is a row of the accumulators).
//   q': scaled by a power of two per head and group (largest |q| in [2^12, 2^13))
//       so that bf16 fits fp16; exact down to 2^-22 of the group's largest (the
//       sixteenth that meets the upper nibbles too), 2^-33 of it below.
//   p s: fp16 (11 bits), the one rounding of the products' operands. p is
//       relative to a running maximum that may lag; p s to a power of two of
//       its head and group that keeps the largest p s seen, not the largest s,
//       in the upper half of fp16's range, so that a step counts only with the
//       weight of its key (a masked key's not at all) and no group or head
//       costs another its bits. Maximum and powers move in two branches that
//       the first tiles take and later ones hardly ever. A power shrinks with
//       what was summed when the maximum moves.
//       So that the rounding weighs code - 8 and not code, which is twice as
//       large, sum_j p_j v_j is computed as sum (p s) code - 8 sum (p s) +
//       sum p (low + 8 s), the first two sums of the same rounded p s.
//   The matrix unit aligns a subnormal's product as if it had fp16's smallest
//       exponent, so that each of a step's 16 products is cut at 2^-24 of that:
//       2^-14 of the largest p s (q' s), measured on one key; of several keys
//       2^-12.7 of the dominant one's step was the most seen: as much as the
//       rounding of p s does to a code one step from 8, 2^-16.6 of a group's range.
// Scores, maxima, sums and the accumulators are fp32: finite for keys and values
// up to 2^100.
//
// The cache is read once, at 144 bytes per key: every warp streams its own
// tiles through a ring of two in shared memory (one bulk copy of 4608
// bytes each, no barrier between warps). 2 rows of 131081 keys, 8 kv heads:
// 53.1 us, 302 MB = 5.7 TB/s (87 % of a copy's rate), of which 47 are the loop,
// at DRAM's rate, the rest its start, the merges and the second launch. In the
// L2 cache (one row of 32775: 13.7 us) the loop is bound by instructions, half
// of them the unpacking (issue slots 57 % busy, the ALU pipe 65 %); a short
// cache (one row of 2771: 6.6 us) by latencies one after another: the launch,
// the counts, the first tile, two barriers.
#pragma once

#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "kv4.cuh"

namespace tg {

constexpr unsigned int ERR_KV4 = 1u << 15;  // bit of the device error word
constexpr int kKv4Stages = 2;          // ring tiles per warp
constexpr int kKv4MaxWarps = 16;
constexpr int kKv4MaxCluster = 8;
constexpr int kKv4OStride = 132;       // of a head's sums in shared memory: the four lanes of a row on different banks
constexpr int kKv4Room = 7;            // p s is scaled to [2^7, 2^8) at its largest, 2^15 at most: normal fp16 down to 2^-14
constexpr float kLog2e = 1.4426950408889634f;

struct Kv4AttnParams {
  const __nv_bfloat16* q;
  int64_t q_sb, q_sh;
  const float* q_scale;  // (B, Hq) nullable
  int64_t qs_sb;
  const uint8_t* cache;
  int64_t c_sb, c_sh;    // bytes
  const float* bias;     // (B, Hq|1, n_prefix) nullable, score units
  int64_t bias_sb, bias_sh;
  const int32_t* n_valid;
  int n_prefix, n_keys;
  const int32_t* n_keys_dev;
  __nv_bfloat16* out;
  int64_t o_sb, o_sh;
  float* part;           // nullable: records [Hq][parts + B][kKv4Part] instead of a merge in a cluster
  int parts;             // blocks per kv head that fill the GPU, shared among the batch rows
  int B, G, Hq;
  float scale;
  unsigned int* err;
};
constexpr int kKv4Part = 4 + 128;  // m, l, 2 pad, O[128]

struct alignas(16) Kv4AttnShared {
  __half q[8][128];
  float mul[8][2];                                // per group
  float m[kKv4MaxWarps][8], l[kKv4MaxWarps][8];   // of the warps' columns; m becomes their factors of the merge
  float head_m[8], head_l[8];
  float got_o[8 * 128];                           // [rank][slice]: this block's slice of the blocks' sums
  float got_m[kKv4MaxCluster][8], got_l[kKv4MaxCluster][8];
  uint64_t full[kKv4MaxWarps][kKv4Stages];
};
constexpr int kKv4Ring = (sizeof(Kv4AttnShared) + 127) / 128 * 128;  // byte offset of the warps' rings
constexpr int kv4_attn_smem(int warps) { return kKv4Ring + warps * kKv4Stages * kKv4TileBytes; }

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_16816_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                   uint32_t b0, uint32_t b1) {  // the same from zero
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// The 8 codes of a word as fp16 pairs (nibble j, nibble j + 4): j even * 2^-24, j odd * 2^-20.
__device__ __forceinline__ void kv4_unpack(uint32_t w, uint32_t (&o)[4]) {
  const uint32_t w8 = w >> 8;
  o[0] = w & 0x000F000Fu;
  o[1] = w & 0x00F000F0u;
  o[2] = w8 & 0x000F000Fu;
  o[3] = w8 & 0x00F000F0u;
}
__device__ __forceinline__ float kv4_scale(uint32_t param) { return __uint_as_float(param << 16); }
__device__ __forceinline__ float kv4_low(uint32_t param) { return __uint_as_float(param & 0xFFFF0000u); }

__device__ __forceinline__ float warp_max_rows(float v) {  // over the lanes of equal lane % 4
#pragma unroll
  for (int off = 4; off <= 16; off <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}
__device__ __forceinline__ float warp_sum_rows(float v) {
#pragma unroll
  for (int off = 4; off <= 16; off <<= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// The lane's four values of a head's q, (B, heads, 128) bf16 with any alignment.
__device__ __forceinline__ uint2 kv4_load_q(const __nv_bfloat16* qp, int lane) {
  if ((reinterpret_cast<uintptr_t>(qp) & 7) == 0) return *(reinterpret_cast<const uint2*>(qp) + lane);
  const uint16_t* u = reinterpret_cast<const uint16_t*>(qp) + 4 * lane;
  return make_uint2(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16);
}

// Tiles with attended keys of a row: [0, na) and from tb on, n in all.
struct Kv4Span {
  int na, tb, n;
};
__device__ __forceinline__ Kv4Span kv4_span(int n_valid, int n_prefix, int n_keys) {
  const int tiles = (n_keys + kKv4Keys - 1) / kKv4Keys;
  const int nv = min(max(n_valid, 0), n_prefix);
  Kv4Span r;
  r.na = min((nv + kKv4Keys - 1) / kKv4Keys, tiles);
  r.tb = max(n_prefix / kKv4Keys, r.na);
  r.n = r.na + max(tiles - r.tb, 0);
  return r;
}

// How the `parts` blocks of a kv head are shared among the batch rows: by the
// tiles that each has (rows of unlike length keep every SM as busy), at least
// one to a row that has any. Of the row b for which pick(b, first, count) is
// true, with its blocks [first, first + count): b, first and count to the whole
// warp (b = -1: none). The counts' sum is below parts + B. Every warp computes
// it for itself, 32 rows at a time.
template <typename Pick>
__device__ __forceinline__ void kv4_share(const Kv4AttnParams& p, int n_keys, int lane, Pick pick, int& b, int& first,
                                          int& count) {
  if (p.B == 1) {  // nothing to share, so nothing to wait for
    b = pick(0, 0, p.parts) ? 0 : -1;
    first = 0;
    count = p.parts;
    return;
  }
  auto tiles_of = [&](int r) { return r < p.B ? kv4_span(__ldg(p.n_valid + r), p.n_prefix, n_keys).n : 0; };
  int n = tiles_of(lane);
  float total = (float)__reduce_add_sync(0xffffffffu, (unsigned)n);
  for (int b0 = 32; b0 < p.B; b0 += 32) total += (float)__reduce_add_sync(0xffffffffu, (unsigned)tiles_of(b0 + lane));
  // a share rounded down of all blocks, or rounded up of all but one per row: whichever is more (the same fp32
  // roundings wherever it is computed)
  const float down = __fdiv_rn((float)p.parts, total), up = __fdiv_rn((float)max(p.parts - p.B, 0), total);
  b = -1;
  first = count = 0;
  int run = 0;
  for (int b0 = 0; b0 < p.B && b < 0; b0 += 32) {
    if (b0 > 0) n = tiles_of(b0 + lane);
    const int c = n == 0 ? 0
                         : max(max((int)floorf(__fmul_rn((float)n, down) + 1e-3f), (int)ceilf(__fmul_rn((float)n, up) - 1e-3f)), 1);
    int end = c;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, end, off);
      if (lane >= off) end += a;
    }
    end += run;
    const uint32_t hit = __ballot_sync(0xffffffffu, b0 + lane < p.B && pick(b0 + lane, end - c, c));
    if (hit) {
      const int src = __ffs(hit) - 1;
      b = b0 + src;
      first = __shfl_sync(0xffffffffu, end - c, src);
      count = __shfl_sync(0xffffffffu, c, src);
    }
    run = __shfl_sync(0xffffffffu, end, 31);
  }
}

// Four dims of an output row (any alignment), normalised; no key: zeros.
__device__ __forceinline__ void kv4_store_out(__nv_bfloat16* at, float4 o, float l) {
  const float r = l == 0.f ? 0.f : 1.f / l;
  const uint32_t a = pack_bf16x2(o.x * r, o.y * r), b = pack_bf16x2(o.z * r, o.w * r);
  if ((reinterpret_cast<uintptr_t>(at) & 7) == 0) {
    *reinterpret_cast<uint2*>(at) = make_uint2(a, b);
  } else {
    uint16_t* u = reinterpret_cast<uint16_t*>(at);
    u[0] = (uint16_t)a;
    u[1] = (uint16_t)(a >> 16);
    u[2] = (uint16_t)b;
    u[3] = (uint16_t)(b >> 16);
  }
}

// A warp's running softmax over its tiles. The 8 columns of the products are
// 8 independent softmaxes, lane (g, t) having columns 2 t and 2 t + 1:
//   PAIR (up to 4 query heads per kv head): column 4 s + h is head h over the
//         16-key halves s of the tiles, so no lane works on an empty column
//         and the two are merged at the end (2 rows of 131081 keys, 8 kv
//         heads: 59.6 -> 56.8 us when it came; 444 instructions a tile now,
//         prologues included);
//   else: column h is head h.
// Without a bias the scores are in log2 units; with one they stay in natural
// units, where a bias of the type's lowest value does not overflow.
struct Kv4State {
  uint32_t qf[8][2];    // B fragments of q'
  float2 qs[2], mul[2];  // per column, (group 0, group 1): sum(q'), and what undoes its power of two
  float m[2], l[2];           // running maximum, sum p
  float2 zs[2];               // per column, (group 0, group 1): sum p (low + 8 s) - 8 (p s)
  float acc[8][4];             // sum (p s) code / e, times 2^-24 (rows g) or 2^-20 (rows g + 8)
  float2 einv[2];              // likewise 1 / e: e, the power of two that p s is relative to, is 2^-126 to 2^121
};
__device__ __forceinline__ float kv4_pow2_inverse(float x) {  // of a power of two from 2^-126 to 2^126
  return __uint_as_float(0x7F000000u - __float_as_uint(x));
}

template <bool V>
struct Kv4Bool {
  static constexpr bool value = V;
};

// One tile of 32 keys from shared memory. ALL: every key is attended.
template <bool BIAS, bool PAIR, bool ALL>
__device__ __forceinline__ void kv4_tile(Kv4State& st, const uint8_t* tile, int j0, int n_keys, int nv, int n_prefix,
                                         const float* bias0, const float* bias1, int lane) {
  constexpr int R = PAIR ? 2 : 4;  // key rows of a lane: row0 + 8 r
  const int g = lane >> 2, t = lane & 3;
  const int row0 = PAIR ? 16 * (t >> 1) + g : g;
  uint2 vp[R];
  float sc[R][2], bj[R][2];
  bool row_ok[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int key = j0 + row0 + 8 * r;
    row_ok[r] = ALL || (key < n_keys && (key < nv || key >= n_prefix));
    if (BIAS) {
      const bool has = row_ok[r] && key < n_prefix;
      bj[r][0] = has && bias0 != nullptr ? __ldg(bias0 + key) : 0.f;
      bj[r][1] = has && bias1 != nullptr ? __ldg(bias1 + key) : 0.f;
    }
    vp[r] = *reinterpret_cast<const uint2*>(tile + kKv4Vp + (row0 + 8 * r) * 8);
    if (!row_ok[r]) vp[r] = make_uint2(0u, 0u);  // whatever a masked slot holds
  }
  // ---- q' . code of the two 16-key halves, by group
  float c[2][2][4];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const uint4 x0 = *reinterpret_cast<const uint4*>(tile + (16 * s + g) * 64 + t * 16);
    const uint4 x1 = *reinterpret_cast<const uint4*>(tile + (16 * s + 8 + g) * 64 + t * 16);
    const uint32_t w0[4] = {x0.x, x0.y, x0.z, x0.w}, w1[4] = {x1.x, x1.y, x1.z, x1.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t a[4], d[4];
      kv4_unpack(w0[i], a);
      kv4_unpack(w1[i], d);
      if ((i & 1) == 0)
        mma_f16_16816_zero(c[s][i >> 1], a[0], d[0], a[1], d[1], st.qf[2 * i][0], st.qf[2 * i][1]);
      else
        mma_f16_16816(c[s][i >> 1], a[0], d[0], a[1], d[1], st.qf[2 * i][0], st.qf[2 * i][1]);
      mma_f16_16816(c[s][i >> 1], a[2], d[2], a[3], d[3], st.qf[2 * i + 1][0], st.qf[2 * i + 1][1]);
    }
  }
  // ---- scores
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint2 kp = *reinterpret_cast<const uint2*>(tile + kKv4Kp + (row0 + 8 * r) * 8);
    const float2 sk = __fmul2_rn(make_float2(kv4_scale(kp.x), kv4_scale(kp.y)),
                                 make_float2(16777216.f, 16777216.f));  // 2^24: the codes' units
    const float2 zk = make_float2(kv4_low(kp.x), kv4_low(kp.y));
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int e = 2 * (r & 1) + j;
      const float c0 = PAIR ? (t < 2 ? c[0][0][e] : c[1][0][e]) : c[r >> 1][0][e];
      const float c1 = PAIR ? (t < 2 ? c[0][1][e] : c[1][1][e]) : c[r >> 1][1][e];
      const float2 d = __ffma2_rn(sk, make_float2(c0, c1), __fmul2_rn(zk, st.qs[j]));
      const float v = fmaf(d.x, st.mul[j].x, BIAS ? fmaf(d.y, st.mul[j].y, bj[r][j]) : d.y * st.mul[j].y);
      // -inf in the bias is a mask, whatever the key holds
      sc[r][j] = !row_ok[r] || (BIAS && bj[r][j] == -INFINITY) ? -INFINITY : v;
    }
  }
  // ---- move the running maximum when a score outgrows it: what was summed shrinks by al, of which the powers of two
  // take the exponent (rounded up) and the accumulators the rest
  float top[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    top[j] = fmaxf(sc[0][j], sc[1][j]);
    if (!PAIR) top[j] = fmax3(top[j], sc[R - 2][j], sc[R - 1][j]);
  }
  constexpr float kLag = BIAS ? 4.f : 4.f * kLog2e;
  if (__any_sync(0xffffffffu, top[0] > st.m[0] + kLag || top[1] > st.m[1] + kLag)) {
    // (a warp's first tile rescales nothing: one of the two passes over the accumulators saved where tiles are few)
    const bool summed = __any_sync(0xffffffffu, st.m[0] > -INFINITY || st.m[1] > -INFINITY);
    float f[2][2];
    bool none[2];  // sums that lost all weight are zero, whatever the keys held that a bias has masked
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float mn = fmaxf(st.m[j], warp_max_rows(top[j]));
      const float al = mn == -INFINITY ? 1.f : ex2_approx((st.m[j] - mn) * (BIAS ? kLog2e : 1.f));
      none[j] = BIAS && al == 0.f;
      st.m[j] = mn;
      st.l[j] *= al;
      st.zs[j] = none[j] ? make_float2(0.f, 0.f) : make_float2(st.zs[j].x * al, st.zs[j].y * al);
      const float pow = __uint_as_float((__float_as_uint(al) + 0x007FFFFFu) & 0x7F800000u);
      auto shrink = [&](float& inv) {
        const float e = kv4_pow2_inverse(inv);
        inv = kv4_pow2_inverse(fmaxf(e * pow, 1.17549435e-38f));
        return al == 0.f ? 0.f : al * (e * inv);
      };
      f[0][j] = shrink(st.einv[j].x);
      f[1][j] = shrink(st.einv[j].y);
    }
    if (summed) {
#pragma unroll
      for (int w = 0; w < 8; ++w)
#pragma unroll
        for (int e = 0; e < 4; ++e) st.acc[w][e] = none[e & 1] ? 0.f : st.acc[w][e] * f[w >> 2][e & 1];
    }
  }
  // ---- p and its sums; p s / e, a column's two groups at a time
  float p[R][2], big = 0.f;
  float2 u[R][2];
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float v = sc[r][j];
      const float e = BIAS ? ex2_approx((v - st.m[j]) * kLog2e) : ex2_approx(v - st.m[j]);
      p[r][j] = (BIAS || !ALL) && v == -INFINITY ? 0.f : e;
      st.l[j] += p[r][j];
    }
  }
  {
    float2 sv[R], z[R], odd = make_float2(0.f, 0.f);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      sv[r] = make_float2(kv4_scale(vp[r].x), kv4_scale(vp[r].y));
      z[r] = __ffma2_rn(make_float2(8.f, 8.f), sv[r], make_float2(kv4_low(vp[r].x), kv4_low(vp[r].y)));
      if (BIAS) odd = __ffma2_rn(z[r], make_float2(0.f, 0.f), odd);  // NaN: a step or a low is not finite
    }
    auto sums = [&](auto checked) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const bool none = decltype(checked)::value && p[r][j] == 0.f;  // masked: whatever the key holds
          const float2 pp = make_float2(p[r][j], p[r][j]), nil = make_float2(0.f, 0.f);
          st.zs[j] = __ffma2_rn(pp, none ? nil : z[r], st.zs[j]);
          u[r][j] = __fmul2_rn(__fmul2_rn(pp, none ? nil : sv[r]), st.einv[j]);
          big = fmax3(big, u[r][j].x, u[r][j].y);
        }
    };
    if (BIAS && __any_sync(0xffffffffu, !(odd.x + odd.y == 0.f)))
      sums(Kv4Bool<true>());
    else
      sums(Kv4Bool<false>());
  }
  // ---- move the powers of two when a p s outgrows them
  if (__any_sync(0xffffffffu, big > 32768.f)) {
    float f[2][2];
    float2 ps[R];  // once more, from the tile: fewer registers where it does not happen
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float2 m = make_float2(0.f, 0.f);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint2 pm = *reinterpret_cast<const uint2*>(tile + kKv4Vp + (row0 + 8 * r) * 8);
        const bool none = p[r][j] == 0.f;
        ps[r] = make_float2(none ? 0.f : p[r][j] * kv4_scale(pm.x), none ? 0.f : p[r][j] * kv4_scale(pm.y));
        m = make_float2(fmaxf(m.x, ps[r].x), fmaxf(m.y, ps[r].y));
      }
      // their exponents, both groups' in a word
      uint32_t both = __byte_perm(__float_as_uint(m.x), __float_as_uint(m.y), 0x7632);
#pragma unroll
      for (int off = 4; off <= 16; off <<= 1) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, off));
      auto grow = [&](float& inv, uint32_t exponent) {
        const float e = kv4_pow2_inverse(inv);
        inv = kv4_pow2_inverse(fmaxf(e, __uint_as_float((uint32_t)max((int)(exponent & 255u) - kKv4Room, 1) << 23)));
        return e * inv;
      };
      f[0][j] = grow(st.einv[j].x, both >> 7);
      f[1][j] = grow(st.einv[j].y, both >> 23);
#pragma unroll
      for (int r = 0; r < R; ++r) u[r][j] = __fmul2_rn(ps[r], st.einv[j]);
    }
#pragma unroll
    for (int w = 0; w < 8; ++w)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.acc[w][e] *= f[w >> 2][e & 1];
  }
  // ---- as fp16, and the sums of these; as B fragments (two key rows to a register)
  uint32_t pf[2][R];
  float2 eight[2];  // -8 e
#pragma unroll
  for (int j = 0; j < 2; ++j)
    eight[j] = make_float2(__uint_as_float(0x00800000u - __float_as_uint(st.einv[j].x)),
                           __uint_as_float(0x00800000u - __float_as_uint(st.einv[j].y)));
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const __half2 h0 = __floats2half2_rn(u[r][0].x, u[r][1].x), h1 = __floats2half2_rn(u[r][0].y, u[r][1].y);
    const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
    st.zs[0] = __ffma2_rn(make_float2(f0.x, f1.x), eight[0], st.zs[0]);
    st.zs[1] = __ffma2_rn(make_float2(f0.y, f1.y), eight[1], st.zs[1]);
    pf[0][r] = movmatrix_trans(h2_bits(h0));
    pf[1][r] = movmatrix_trans(h2_bits(h1));
  }
  // ---- P V
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const uint32_t own = (g >> 2) == s ? 0xFFFFFFFFu : 0u;  // PAIR: this half's columns
#pragma unroll
    for (int gr = 0; gr < 2; ++gr) {
      const uint32_t b0 = PAIR ? pf[gr][0] & own : pf[gr][(2 * s) % R], b1 = PAIR ? pf[gr][1] & own : pf[gr][(2 * s + 1) % R];
      const uint4 x = *reinterpret_cast<const uint4*>(tile + kKv4V + s * 1024 + gr * 512 + lane * 16);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a[4];
        kv4_unpack(w[i], a);
        mma_f16_16816(st.acc[4 * gr + i], a[0], a[1], a[2], a[3], b0, b1);
      }
    }
  }
}

// C blocks take one kv head of one row: the tiles that hold attended keys,
// evenly in order to the blocks and in turn to a block's warps. Each warp keeps
// its own running softmax; warps merge in shared memory. The blocks merge in
// one of two ways: as a cluster (grid (C, Hkv, B)), sending each other their
// slices of the output (one barrier, no second launch, no workspace), or, grid
// (parts + B, Hkv), C by kv4_share, through records that kv4_combine_kernel
// merges (so every SM can take part: clusters of 16 leave a quarter of them
// idle).
template <bool BIAS, bool PAIR>
__global__ void __launch_bounds__(32 * kKv4MaxWarps, 1) kv4_attn_kernel(const Kv4AttnParams p) {
  extern __shared__ __align__(128) uint8_t kv4_smem[];
  Kv4AttnShared& sh = *reinterpret_cast<Kv4AttnShared*>(kv4_smem);
  const int W = blockDim.x >> 5;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y;
  int b = blockIdx.z, C = gridDim.x, rank = blockIdx.x;
  constexpr int S = kKv4Stages;
  uint8_t* ring = kv4_smem + kKv4Ring + warp * S * kKv4TileBytes;
  const uint32_t ring_s = smem_u32(ring), full_s = smem_u32(sh.full[warp]);
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kKv4Stages; ++i) mbar_init(full_s + 8 * i, 1);
    fence_mbar_init();
  }
  __syncwarp();
  const bool clustered = p.part == nullptr && C > 1;
  if (clustered) cluster_arrive();
  griddep_wait();
  griddep_launch_dependents();
  const int n_keys = p.n_keys_dev != nullptr ? max(min(__ldg(p.n_keys_dev), p.n_keys), 0) : p.n_keys;
  if (p.part != nullptr) {
    int first;
    kv4_share(p, n_keys, lane, [&](int, int f, int c) { return (int)blockIdx.x >= f && (int)blockIdx.x < f + c; }, b,
              first, C);
    if (b < 0) return;
    rank = blockIdx.x - first;
  }
  // the counts and the heads' q (warp w: heads w, w + W, ..) wait for one another's latency only
  const int nv_raw = __ldg(p.n_valid + b);
  uint2 q_raw = make_uint2(0u, 0u);
  float q_mul = 1.f;
  if (warp < p.G) {
    const int hq = kvh * p.G + warp;
    const __nv_bfloat16* qp = p.q + (int64_t)b * p.q_sb + (int64_t)hq * p.q_sh;
    q_raw = kv4_load_q(qp, lane);
    if (p.q_scale != nullptr) q_mul = p.q_scale[(int64_t)b * p.qs_sb + hq];
  }
  const int nv = min(max(nv_raw, 0), p.n_prefix);
  const uint8_t* base = p.cache + (int64_t)b * p.c_sb + (int64_t)kvh * p.c_sh;
  const Kv4Span span = kv4_span(nv_raw, p.n_prefix, n_keys);
  const int n = span.n;
  // n / C tiles to a block, one more to the first n % C
  const int each = (int)((unsigned)n / (unsigned)C), more = n - each * C;
  const int v0 = rank * each + min(rank, more), v1 = v0 + each + (rank < more);
  const int mine = v1 - v0 > warp ? (v1 - v0 - warp + W - 1) / W : 0;  // this warp's tiles
  auto tile_of = [&](int i) {
    const int v = v0 + warp + i * W;
    return v < span.na ? v : v - span.na + span.tb;
  };
  auto fetch = [&](int i, int s) {
    mbar_arrive_expect_tx(full_s + 8 * s, kKv4TileBytes);
    bulk_load(ring_s + s * kKv4TileBytes, base + (int64_t)tile_of(i) * kKv4TileBytes, kKv4TileBytes, full_s + 8 * s);
  };
  if (lane == 0)
    for (int i = 0; i < min(mine, S); ++i) fetch(i, i);

  // the heads' q', scaled by a power of two
  for (int h = warp; h < (PAIR ? 4 : 8); h += W) {
    if (h != warp && h < p.G) {
      const int hq = kvh * p.G + h;
      q_raw = kv4_load_q(p.q + (int64_t)b * p.q_sb + (int64_t)hq * p.q_sh, lane);
      if (p.q_scale != nullptr) q_mul = p.q_scale[(int64_t)b * p.qs_sb + hq];
    }
    float v[4] = {bf16_lo(q_raw.x), bf16_hi(q_raw.x), bf16_lo(q_raw.y), bf16_hi(q_raw.y)}, mx = 0.f;
    const float qs = round_bf16(q_mul);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (p.q_scale != nullptr) v[e] = round_bf16(v[e] * qs);
      if (h >= p.G) v[e] = 0.f;
      mx = fmaxf(mx, fabsf(v[e]));
    }
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));  // of the group
    // 2^(12 - exponent), inside fp32's normal range on both sides
    const int ex = min(max((int)(__float_as_uint(mx) >> 23) - 127 - 12, -126), 126);
    const float down = __uint_as_float((uint32_t)(127 - ex) << 23);
    if ((lane & 15) == 0) sh.mul[h][lane >> 4] = __uint_as_float((uint32_t)(127 + ex) << 23) * p.scale * (BIAS ? 1.f : kLog2e);
    const __half2 a = __floats2half2_rn(v[0] * down, v[1] * down), c = __floats2half2_rn(v[2] * down, v[3] * down);
    *reinterpret_cast<uint2*>(&sh.q[h][4 * lane]) = make_uint2(h2_bits(a), h2_bits(c));
  }
  __syncthreads();
  Kv4State st;
  // MMA (i, 0): nibbles (0, 4), (1, 5) of word i; (i, 1): (2, 6), (3, 7)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 x = *reinterpret_cast<const uint4*>(&sh.q[PAIR ? g & 3 : g][32 * i + 8 * t]);  // 8 dims
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      uint32_t f = __byte_perm(w[u >> 1], w[2 + (u >> 1)], u & 1 ? 0x7632 : 0x5410);  // dims u, u + 4
      if (u & 1) f = h2_bits(__hmul2(bits_h2(f), __float2half2_rn(0.0625f)));  // its nibbles read 16 times as large
      st.qf[2 * i + (u >> 1)][u & 1] = f;
    }
  }
  const int h0 = PAIR ? 2 * (t & 1) : 2 * t;  // head of column 2 t
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    st.mul[j] = make_float2(sh.mul[h0 + j][0], sh.mul[h0 + j][1]);
    st.m[j] = -INFINITY;
    st.l[j] = 0.f;
    st.zs[j] = make_float2(0.f, 0.f);
    st.einv[j] = make_float2(8.507059173e37f, 8.507059173e37f);  // 2^126
#pragma unroll
    for (int gr = 0; gr < 2; ++gr) {
      const uint4 x = *reinterpret_cast<const uint4*>(&sh.q[h0 + j][64 * gr + 8 * g]);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
      float a = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = __half22float2(bits_h2(w[e]));
        a += f.x + f.y;
      }
      (gr ? st.qs[j].y : st.qs[j].x) = warp_sum_rows(a);
    }
  }
#pragma unroll
  for (int w = 0; w < 8; ++w)
#pragma unroll
    for (int e = 0; e < 4; ++e) st.acc[w][e] = 0.f;
  const float *bias0 = nullptr, *bias1 = nullptr;
  if (BIAS) {
    const float* bp = p.bias + (int64_t)b * p.bias_sb + (int64_t)(kvh * p.G + h0) * p.bias_sh;
    if (h0 < p.G) bias0 = bp;
    if (h0 + 1 < p.G) bias1 = bp + p.bias_sh;
  }

  int i = 0, s = 0, ph = 0;
  for (; i < mine; ++i) {
    // one answer for the warp: lanes that gave up and lanes that did not would wait for one another below
    if (!__all_sync(0xffffffffu, mbar_wait(full_s + 8 * s, ph, p.err, ERR_KV4))) break;
    const int j0 = tile_of(i) * kKv4Keys;
    const uint8_t* tile = ring + s * kKv4TileBytes;
    if (j0 + kKv4Keys <= n_keys && (j0 + kKv4Keys <= nv || j0 >= p.n_prefix))
      kv4_tile<BIAS, PAIR, true>(st, tile, j0, n_keys, nv, p.n_prefix, bias0, bias1, lane);
    else
      kv4_tile<BIAS, PAIR, false>(st, tile, j0, n_keys, nv, p.n_prefix, bias0, bias1, lane);
    __syncwarp();
    if (lane == 0 && i + S < mine) fetch(i + S, s);
    if (++s == S) {
      s = 0;
      ph ^= 1;
    }
  }
  // a copy never came: it and those behind it get their time, each in its own phase, before the ring is used again
  for (int k = 0; k < S && i < mine; ++k, ++i) {
    mbar_wait(full_s + 8 * s, ph, p.err, ERR_KV4);
    if (++s == S) {
      s = 0;
      ph ^= 1;
    }
  }
  __syncwarp();

  // ---- merge the warps: their sums into the rings' memory
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    st.l[j] = warp_sum_rows(st.l[j]);
    st.zs[j] = make_float2(warp_sum_rows(st.zs[j].x), warp_sum_rows(st.zs[j].y));
    if (g == 0) {
      sh.m[warp][2 * t + j] = st.m[j];
      sh.l[warp][2 * t + j] = st.l[j];
    }
  }
  __syncwarp();
  float* so = reinterpret_cast<float*>(ring);  // [8][kKv4OStride] of this warp
#pragma unroll
  for (int w = 0; w < 8; ++w)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float inv = w < 4 ? st.einv[e & 1].x : st.einv[e & 1].y, z = w < 4 ? st.zs[e & 1].x : st.zs[e & 1].y;
      so[(2 * t + (e & 1)) * kKv4OStride + 16 * w + g + 8 * (e >> 1)] =
          fmaf(st.acc[w][e] * (e < 2 ? 16777216.f : 1048576.f), kv4_pow2_inverse(inv), z);
    }
  if (clustered) cluster_wait();  // every block has started
  __syncthreads();
  constexpr float kUnit = BIAS ? kLog2e : 1.f;  // of m
  constexpr int K = PAIR ? 2 : 1;               // columns of a head, 4 apart
  // a warp per head: the maximum over its columns, their factors, the sum of p
  for (int h = warp; h < p.G; h += W) {
    const int w = K == 2 ? lane >> 1 : lane, col = h + (K == 2 ? 4 * (lane & 1) : 0);
    const bool has = w < W;
    const float mw = has ? sh.m[w][col] : -INFINITY, lw = has ? sh.l[w][col] : 0.f;
    float mt = mw;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, off));
    const float f = lw == 0.f ? 0.f : ex2_approx((mw - mt) * kUnit);  // 0: the column saw no key
    float lt = f * lw;                                                // (a NaN sum stays in)
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) lt += __shfl_xor_sync(0xffffffffu, lt, off);
    if (has) sh.m[w][col] = f;
    if (lane == 0) {
      sh.head_m[h] = mt;
      sh.head_l[h] = lt;
    }
  }
  __syncthreads();
  const float* all_o = reinterpret_cast<const float*>(kv4_smem + kKv4Ring);
  const int slice = p.G * 128 / C;  // of a cluster: a multiple of 16
  for (int i4 = threadIdx.x; i4 < p.G * 32; i4 += blockDim.x) {
    const int h = i4 >> 5, d = 4 * (i4 & 31);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < W; ++w) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const float f = sh.m[w][h + 4 * k];
        if (BIAS && f == 0.f) continue;  // no weight: whatever the masked keys held
        const float4 v = *reinterpret_cast<const float4*>(all_o + w * (S * kKv4TileBytes / 4) + (h + 4 * k) * kKv4OStride + d);
        o.x = fmaf(f, v.x, o.x);
        o.y = fmaf(f, v.y, o.y);
        o.z = fmaf(f, v.z, o.z);
        o.w = fmaf(f, v.w, o.w);
      }
    }
    const float mt = sh.head_m[h], lt = sh.head_l[h];
    if (C == 1) {
      kv4_store_out(p.out + (int64_t)b * p.o_sb + (int64_t)(kvh * p.G + h) * p.o_sh + d, o, lt);
    } else if (!clustered) {
      float* rec = p.part + ((int64_t)(kvh * p.G + h) * gridDim.x + blockIdx.x) * kKv4Part;
      *reinterpret_cast<float4*>(rec + 4 + d) = o;
      if (d == 0) *reinterpret_cast<float2*>(rec) = make_float2(mt, lt);
    } else {
      cooperative_groups::cluster_group cl = cooperative_groups::this_cluster();
      *reinterpret_cast<float4*>(cl.map_shared_rank(sh.got_o, 4 * i4 / slice) + rank * slice + 4 * i4 % slice) = o;
      if ((i4 & 31) < C) {
        cl.map_shared_rank(&sh.got_m[rank][h], i4 & 31)[0] = mt;
        cl.map_shared_rank(&sh.got_l[rank][h], i4 & 31)[0] = lt;
      }
    }
  }
  if (!clustered) return;
  __syncwarp();
  cluster_sync_all();
  for (int i = threadIdx.x; i < slice; i += blockDim.x) {
    const int idx = rank * slice + i, h = idx >> 7;
    float mt = sh.got_m[0][h];
    for (int c = 1; c < C; ++c) mt = fmaxf(mt, sh.got_m[c][h]);
    float o = 0.f, lt = 0.f;
    for (int c = 0; c < C; ++c) {
      const float lw = sh.got_l[c][h];
      if (lw != 0.f) {
        const float f = ex2_approx((sh.got_m[c][h] - mt) * kUnit), on = fmaf(f, sh.got_o[c * slice + i], o);
        o = BIAS && f == 0.f ? o : on;
        lt = fmaf(f, lw, lt);
      }
    }
    p.out[(int64_t)b * p.o_sb + (int64_t)(kvh * p.G + h) * p.o_sh + (idx & 127)] =
        __float2bfloat16_rn(lt == 0.f ? 0.f : o / lt);
  }
}

// Merges the blocks' records of one (row, head): 8 warps take every 8th record
// (lane: dims 4 l .. 4 l + 3, 16-byte loads), four at a time with every load
// before any arithmetic, then merge through shared memory.
constexpr int kKv4CombineWarps = 8;
__global__ void __launch_bounds__(32 * kKv4CombineWarps) kv4_combine_kernel(const Kv4AttnParams p) {
  __shared__ float s_m[kKv4CombineWarps], s_l[kKv4CombineWarps];
  __shared__ float s_o[kKv4CombineWarps][128];
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // The counts before the wait: this grid starts when every block of the attention's has passed its own, so what came
  // before that is complete, and the attention writes only records and outputs.
  const int n_keys = p.n_keys_dev != nullptr ? max(min(__ldg(p.n_keys_dev), p.n_keys), 0) : p.n_keys;
  int found, first, C;
  kv4_share(p, n_keys, lane, [&](int r, int, int) { return r == b; }, found, first, C);
  griddep_wait();
  griddep_launch_dependents();
  if (C == 1) return;  // its one block has written the output
  const float* rec = p.part + ((int64_t)h * (p.parts + p.B) + first) * kKv4Part;
  const bool masks = p.bias != nullptr;  // sums without weight may hold anything then
  const float unit = masks ? kLog2e : 1.f;  // of m
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c0 = warp; c0 < C; c0 += 4 * kKv4CombineWarps) {
    float4 v[4];
    float2 ml[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = c0 + k * kKv4CombineWarps;
      ml[k] = make_float2(-INFINITY, 0.f);
      if (c < C) {
        const float* r = rec + (int64_t)c * kKv4Part;
        ml[k] = *reinterpret_cast<const float2*>(r);
        v[k] = *reinterpret_cast<const float4*>(r + 4 + 4 * lane);
      }
    }
    const float mn = fmaxf(fmax3(m, ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
    const float back = l == 0.f ? 0.f : ex2_approx((m - mn) * unit);
    m = mn;
    l *= back;
    o.x *= back;
    o.y *= back;
    o.z *= back;
    o.w *= back;
    if (masks && back == 0.f) o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (ml[k].y != 0.f) {  // 0: the block saw no key (a NaN sum stays in)
        const float f = ex2_approx((ml[k].x - m) * unit);
        l = fmaf(f, ml[k].y, l);
        if (masks && f == 0.f) continue;
        o.x = fmaf(f, v[k].x, o.x);
        o.y = fmaf(f, v[k].y, o.y);
        o.z = fmaf(f, v[k].z, o.z);
        o.w = fmaf(f, v[k].w, o.w);
      }
    }
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  *reinterpret_cast<float4*>(&s_o[warp][4 * lane]) = o;
  __syncthreads();
  if (threadIdx.x < 128) {
    float mt = s_m[0], ot = 0.f, lt = 0.f;
#pragma unroll
    for (int w = 1; w < kKv4CombineWarps; ++w) mt = fmaxf(mt, s_m[w]);
#pragma unroll
    for (int w = 0; w < kKv4CombineWarps; ++w) {
      if (s_l[w] != 0.f) {
        const float f = ex2_approx((s_m[w] - mt) * unit), on = fmaf(f, s_o[w][threadIdx.x], ot);
        ot = masks && f == 0.f ? ot : on;
        lt = fmaf(f, s_l[w], lt);
      }
    }
    p.out[(int64_t)b * p.o_sb + (int64_t)h * p.o_sh + threadIdx.x] = __float2bfloat16_rn(lt == 0.f ? 0.f : ot / lt);
  }
}

}  // namespace tg

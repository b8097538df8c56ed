// Decode attention over the 4-bit KV cache (layout: kv4.cuh): the same
// operation as decode_attn.cuh, one query token per (batch row, head),
//   out = softmax_j( softmax_scale * (q' . k_j) + m_j ) V
// with k_j, v_j the values that the codes stand for, low + code * scale.
//
// Everything rests on writing a value as z + s * (code - 8), z = low + 8 s:
//   q . k = sum over the row's two groups of  s * (q . (code - 8)) + z * sum(q)
//   sum_j p_j v_j = (sum_j (p_j s_j) (code_j - 8)) + sum_j p_j z_j     per group
// so the tensor cores multiply by the small integers code - 8, exact in fp16,
// and the scales and lows enter in fp32 outside the products. K is the A
// operand (16 keys x 16 dims, m16n8k16) against the heads of one kv head as the
// 8 columns; V^T is A (16 dims x 16 keys) against the probabilities. A nibble
// pair becomes two fp16 integers with one LOP3 (or into the mantissa of 1024)
// and one HADD2 / HFMA2.
//   q': scaled by a power of two per head (largest |q| in [256, 512)) so that
//       bf16 fits fp16; exact down to 2^-22 of the largest, 2^-33 of it below.
//   p s: fp16 (11 bits), the one rounding of the products' operands; p is
//       relative to a running maximum that may lag by kKv4Lag, s to a running
//       power of two, so neither leaves fp16's range.
// Scores, maxima, sums and the accumulators are fp32.
#pragma once

#include <cuda_fp16.h>

#include "kv4.cuh"

namespace tg {

constexpr int kKv4Warps = 4;
constexpr int kKv4AttnThreads = 32 * kKv4Warps;
constexpr int kKv4Part = 4 + 128;     // m, l, 2 pad, O[128] per (row, head, split)
constexpr float kKv4Lag = 4.f;        // a score may pass the running maximum by this (natural units)
constexpr float kKv4Head = 4.f;       // p = 2^(4 + ...): small p stay normal in fp16

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
  float* part;           // [B][Hq][n_splits][kKv4Part]
  int Hq, Hkv, G, n_splits, tiles_per_split;
  float scale;
};

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// The 8 codes of a word minus 8, as fp16 pairs (nibble j, nibble j + 4).
__device__ __forceinline__ void kv4_unpack(uint32_t w, uint32_t (&o)[4]) {
  const __half2 c1032 = __float2half2_rn(-1032.f), c72 = __float2half2_rn(-72.f), r16 = __float2half2_rn(0.0625f);
  const uint32_t w8 = w >> 8;
  o[0] = h2_bits(__hadd2(bits_h2((w & 0x000F000Fu) | 0x64006400u), c1032));         // 1024 + n - 1032
  o[1] = h2_bits(__hfma2(bits_h2((w & 0x00F000F0u) | 0x64006400u), r16, c72));      // (1024 + 16 n) / 16 - 72
  o[2] = h2_bits(__hadd2(bits_h2((w8 & 0x000F000Fu) | 0x64006400u), c1032));
  o[3] = h2_bits(__hfma2(bits_h2((w8 & 0x00F000F0u) | 0x64006400u), r16, c72));
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

struct Kv4Tile {
  uint4 k[2][2], v[2][2];
  uint2 kp[4], vp[4];
};

__device__ __forceinline__ void kv4_load_tile(const uint8_t* tile, int lane, Kv4Tile& x) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      x.k[s][r] = ld_nc_v4(reinterpret_cast<const uint4*>(tile + (16 * s + 8 * r + g) * 64 + t * 16));
      x.v[s][r] = ld_nc_v4(reinterpret_cast<const uint4*>(tile + kKv4V + s * 1024 + r * 512 + lane * 16));
      x.kp[2 * s + r] = *reinterpret_cast<const uint2*>(tile + kKv4Kp + (16 * s + 8 * r + g) * 8);
      x.vp[2 * s + r] = *reinterpret_cast<const uint2*>(tile + kKv4Vp + (16 * s + 8 * r + g) * 8);
    }
  }
}

// A CTA takes one kv head of one row and a run of tiles, its warps every
// kKv4Warps-th tile of it; each warp keeps its own running softmax, the CTA
// merges them in shared memory. One split writes the output, more write
// (m, l, O) records that kv4_combine_kernel merges.
__global__ void __launch_bounds__(kKv4AttnThreads) kv4_attn_kernel(const Kv4AttnParams p) {
  __shared__ float sq[8][128];
  __shared__ float s_mul[8];
  __shared__ float s_m[kKv4Warps][8], s_l[kKv4Warps][8];
  __shared__ float s_o[kKv4Warps][8][128];

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  griddep_wait();
  griddep_launch_dependents();
  const int n_keys = p.n_keys_dev != nullptr ? min(__ldg(p.n_keys_dev), p.n_keys) : p.n_keys;
  const int nv = __ldg(p.n_valid + b);
  const uint8_t* base = p.cache + (int64_t)b * p.c_sb + (int64_t)kvh * p.c_sh;

  // the heads' q', scaled by a power of two
  for (int h = warp; h < 8; h += kKv4Warps) {
    float v[4] = {0.f, 0.f, 0.f, 0.f}, mx = 0.f;
    if (h < p.G) {
      const int hq = kvh * p.G + h;
      const __nv_bfloat16* qp = p.q + (int64_t)b * p.q_sb + (int64_t)hq * p.q_sh;
      const float qs = p.q_scale != nullptr ? round_bf16(p.q_scale[(int64_t)b * p.qs_sb + hq]) : 1.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = __bfloat162float(qp[lane + 32 * e]);
        if (p.q_scale != nullptr) v[e] = round_bf16(v[e] * qs);
        mx = fmaxf(mx, fabsf(v[e]));
      }
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    // 2^(8 - exponent), inside fp32's normal range on both sides
    const int ex = min(max((int)(__float_as_uint(mx) >> 23) - 127 - 8, -126), 126);
    const float down = __uint_as_float((uint32_t)(127 - ex) << 23);
    if (lane == 0) s_mul[h] = __uint_as_float((uint32_t)(127 + ex) << 23) * p.scale;
#pragma unroll
    for (int e = 0; e < 4; ++e) sq[h][lane + 32 * e] = __half2float(__float2half_rn(v[e] * down));
  }
  __syncthreads();
  // B fragments: MMA (i, 0): nibbles (0, 4), (1, 5) of word i; (i, 1): (2, 6), (3, 7)
  uint32_t qf[8][2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int d = 32 * i + 8 * t + u;
      qf[2 * i + (u >> 1)][u & 1] = h2_bits(__floats2half2_rn(sq[g][d], sq[g][d + 4]));
    }
  }
  float qsum[2][2], mul[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    mul[j] = s_mul[2 * t + j];
#pragma unroll
    for (int gr = 0; gr < 2; ++gr) {
      float a = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) a += sq[2 * t + j][64 * gr + 8 * g + e];
      qsum[gr][j] = warp_sum_rows(a);
    }
  }

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, zs[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
  float acc[8][4];
#pragma unroll
  for (int w = 0; w < 8; ++w)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[w][e] = 0.f;
  float eref = 1.17549435e-38f, einv = 8.507059173e37f;  // 2^-126, 2^126

  const int t0 = split * p.tiles_per_split;
  const int t1 = min(t0 + p.tiles_per_split, (n_keys + kKv4Keys - 1) / kKv4Keys);
  for (int tile = t0 + warp; tile < t1; tile += kKv4Warps) {
    const int j0 = tile * kKv4Keys;
    if (j0 >= nv && j0 + kKv4Keys <= p.n_prefix) continue;  // pad slots only
    Kv4Tile x;
    kv4_load_tile(base + (int64_t)tile * kKv4TileBytes, lane, x);
    // ---- scores: sc[4 * s + 2 * r + j] of key 16 s + 8 r + g and head 2 t + j
    float sc[8];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      float c[2][4];
#pragma unroll
      for (int gr = 0; gr < 2; ++gr)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[gr][e] = 0.f;
      const uint32_t w0[4] = {x.k[s][0].x, x.k[s][0].y, x.k[s][0].z, x.k[s][0].w};
      const uint32_t w1[4] = {x.k[s][1].x, x.k[s][1].y, x.k[s][1].z, x.k[s][1].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a[4], d[4];
        kv4_unpack(w0[i], a);
        kv4_unpack(w1[i], d);
        mma_f16_16816(c[i >> 1], a[0], d[0], a[1], d[1], qf[2 * i][0], qf[2 * i][1]);
        mma_f16_16816(c[i >> 1], a[2], d[2], a[3], d[3], qf[2 * i + 1][0], qf[2 * i + 1][1]);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint2 kp = x.kp[2 * s + r];
        const float s0 = kv4_scale(kp.x), s1 = kv4_scale(kp.y);
        const float z0 = fmaf(8.f, s0, kv4_low(kp.x)), z1 = fmaf(8.f, s1, kv4_low(kp.y));
        const int key = j0 + 16 * s + 8 * r + g;
        const bool valid = key < n_keys && (key < nv || key >= p.n_prefix);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float v = s0 * c[0][2 * r + j];
          v = fmaf(s1, c[1][2 * r + j], v);
          v = fmaf(z0, qsum[0][j], v);
          v = fmaf(z1, qsum[1][j], v);
          v *= mul[j];
          bool seen = valid;
          if (p.bias != nullptr && key < p.n_prefix && 2 * t + j < p.G && valid) {
            const float bj = __ldg(p.bias + (int64_t)b * p.bias_sb + (int64_t)(kvh * p.G + 2 * t + j) * p.bias_sh + key);
            v += bj;
            seen = bj != -INFINITY;  // a mask, whatever the key holds
          }
          sc[4 * s + 2 * r + j] = seen ? v : -INFINITY;
        }
      }
    }
    // ---- move the running maximum / power of two when a score or a step outgrows them
    float smax = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int key = j0 + 8 * r + g;
      if (key < n_keys && (key < nv || key >= p.n_prefix)) smax = fmaxf(smax, fmaxf(kv4_scale(x.vp[r].x), kv4_scale(x.vp[r].y)));
    }
    float top[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) top[j] = fmaxf(fmaxf(sc[j], sc[2 + j]), fmaxf(sc[4 + j], sc[6 + j]));
    const bool grow = top[0] > m[0] + kKv4Lag || top[1] > m[1] + kKv4Lag || smax * einv > 16.f;
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) smax = fmaxf(smax, __shfl_xor_sync(0xffffffffu, smax, off));
      // a power of two >= smax, at most 2^126
      const uint32_t eb = min((__float_as_uint(smax) >> 23) + 1u, 253u);
      const float enew = fmaxf(eref, __uint_as_float(max(eb, 1u) << 23));
      const float beta = eref / enew;
      eref = enew;
      einv = 1.f / enew;
      float al[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float mn = fmaxf(m[j], warp_max_rows(top[j]));
        al[j] = mn == -INFINITY ? 1.f : ex2_approx((m[j] - mn) * 1.4426950408889634f);
        m[j] = mn;
        l[j] *= al[j];
        zs[0][j] *= al[j];
        zs[1][j] *= al[j];
      }
#pragma unroll
      for (int w = 0; w < 8; ++w)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[w][e] *= al[e & 1] * beta;
    }
    // ---- p, its sums, and P V
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      uint32_t pf[2][2];  // B fragments per group
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint2 vp = x.vp[2 * s + r];
        float pr[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float v = sc[4 * s + 2 * r + j];
          pr[j] = v == -INFINITY ? 0.f : ex2_approx(fmaf(v - m[j], 1.4426950408889634f, kKv4Head));
          l[j] += pr[j];
        }
        const bool any = sc[4 * s + 2 * r] != -INFINITY || sc[4 * s + 2 * r + 1] != -INFINITY;
#pragma unroll
        for (int gr = 0; gr < 2; ++gr) {
          const uint32_t pm = gr ? vp.y : vp.x;
          const float sv = any ? kv4_scale(pm) : 0.f, z = any ? fmaf(8.f, kv4_scale(pm), kv4_low(pm)) : 0.f;
          zs[gr][0] = fmaf(pr[0], z, zs[gr][0]);
          zs[gr][1] = fmaf(pr[1], z, zs[gr][1]);
          const float sn = sv * einv;
          pf[gr][r] = movmatrix_trans(h2_bits(__floats2half2_rn(pr[0] * sn, pr[1] * sn)));
        }
      }
#pragma unroll
      for (int hv = 0; hv < 2; ++hv) {
        const uint32_t w[4] = {x.v[s][hv].x, x.v[s][hv].y, x.v[s][hv].z, x.v[s][hv].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t a[4];
          kv4_unpack(w[i], a);
          mma_f16_16816(acc[4 * hv + i], a[0], a[1], a[2], a[3], pf[hv][0], pf[hv][1]);
        }
      }
    }
  }

  // ---- merge the warps
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    l[j] = warp_sum_rows(l[j]);
    zs[0][j] = warp_sum_rows(zs[0][j]);
    zs[1][j] = warp_sum_rows(zs[1][j]);
    if (g == 0) {
      s_m[warp][2 * t + j] = m[j];
      s_l[warp][2 * t + j] = l[j];
    }
  }
#pragma unroll
  for (int w = 0; w < 8; ++w)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      s_o[warp][2 * t + (e & 1)][16 * w + g + 8 * (e >> 1)] = fmaf(acc[w][e], eref, zs[w >> 2][e & 1]);
  __syncthreads();
  for (int idx = threadIdx.x; idx < p.G * 128; idx += kKv4AttnThreads) {
    const int h = idx >> 7, d = idx & 127;
    float mt = s_m[0][h];
#pragma unroll
    for (int w = 1; w < kKv4Warps; ++w) mt = fmaxf(mt, s_m[w][h]);
    float o = 0.f, lt = 0.f;
#pragma unroll
    for (int w = 0; w < kKv4Warps; ++w) {
      const float lw = s_l[w][h];
      if (lw != 0.f) {  // 0: the warp saw no key (a NaN sum stays in)
        const float f = ex2_approx((s_m[w][h] - mt) * 1.4426950408889634f);
        o = fmaf(f, s_o[w][h][d], o);
        lt = fmaf(f, lw, lt);
      }
    }
    const int hq = kvh * p.G + h;
    if (p.n_splits == 1) {
      p.out[(int64_t)b * p.o_sb + (int64_t)hq * p.o_sh + d] = __float2bfloat16_rn(lt == 0.f ? 0.f : o / lt);
    } else {
      float* rec = p.part + (((int64_t)b * p.Hq + hq) * p.n_splits + split) * kKv4Part;
      rec[4 + d] = o;
      if (d == 0) {
        rec[0] = mt;
        rec[1] = lt;
      }
    }
  }
}

// Merges the splits' (m, l, O) of one (row, head): 128 threads, one dim each.
__global__ void __launch_bounds__(128) kv4_combine_kernel(const Kv4AttnParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
  const float* rec = p.part + ((int64_t)b * p.Hq + h) * p.n_splits * kKv4Part;
  float m = -INFINITY;
  for (int c = 0; c < p.n_splits; ++c) m = fmaxf(m, rec[(int64_t)c * kKv4Part]);
  float o = 0.f, l = 0.f;
  for (int c = 0; c < p.n_splits; ++c) {
    const float* r = rec + (int64_t)c * kKv4Part;
    if (r[1] != 0.f) {  // 0: the split saw no key (a NaN sum stays in)
      const float f = ex2_approx((r[0] - m) * 1.4426950408889634f);
      o = fmaf(f, r[4 + d], o);
      l = fmaf(f, r[1], l);
    }
  }
  p.out[(int64_t)b * p.o_sb + (int64_t)h * p.o_sh + d] = __float2bfloat16_rn(l == 0.f ? 0.f : o / l);
}

}  // namespace tg

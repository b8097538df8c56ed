// The 4-bit KV cache: K and V rows of head_dim 128 held as 4-bit codes with a
// bf16 step and a bf16 low per group of 64 dims, 4.5 bits a value.
//
//   low   = min(x)                                    over the group's 64 bf16 values
//   scale = bf16((max/2 - min/2) / 7.5), 0 below 2^-100 (then every code is 0)
//   code  = floor((x - low) * inv + 1/2) in 0..15,    inv = (1/scale) * (1 + 2^-22)
//   value = bf16(low + code * scale)
// in fp32, one IEEE rounding per operation. The step's reciprocal is taken
// 2^-22 high so that its own rounding never takes an exact half down; low is
// exact (bf16 in, bf16 out). A group that holds a NaN or an infinity, or
// whose range max - min passes fp32's largest, gets a NaN step and reads back
// as NaN.
//
// Layout, made for the attention kernel's MMA fragments (kv4_attn.cuh) and for
// appending without reading: tiles of 32 keys, one contiguous 4608-byte block
// per (batch row, kv head, tile), so a key range is one contiguous stream.
//   [0, 2048)     K codes: 64 bytes per key. Word i of 16-byte piece t holds
//                 dims 32 i + 8 t + (0..7), dim 32 i + 8 t + j at bits 4 j: the
//                 lane (key row, t) of an m16n8k16 A fragment reads its 32 dims
//                 as one 16-byte load.
//   [2048, 4096)  V codes: 1024 bytes per 16 keys, in A-fragment order of V^T:
//                 byte (w / 4) * 512 + (4 g + t) * 16 + (w % 4) * 4 + c holds
//                 dims 16 w + g (low nibble) and 16 w + g + 8 (high nibble) of
//                 key 2 t + (c >> 1) + 8 (c & 1): each byte belongs to one key.
//   [4096, 4352)  K params: per key two words (group 0, 1) = scale | low << 16
//   [4352, 4608)  V params, likewise
#pragma once

#include <cuda_bf16.h>

#include "layer_glue.cuh"
#include "ptx.cuh"

namespace tg {

constexpr int kKv4Keys = 32;              // keys per tile
constexpr int kKv4TileBytes = 4608;
constexpr int kKv4V = 2048;               // byte offsets inside a tile
constexpr int kKv4Kp = 4096;
constexpr int kKv4Vp = 4352;

struct Kv4Group {
  float low, inv;
  uint32_t param;  // scale | low << 16; a NaN scale above a low of 0 for a group that cannot be held
  bool bad;
};

// The group's parameters from its maximum and minus its minimum (NaN where the
// group holds one).
__device__ __forceinline__ Kv4Group kv4_group(float mx, float neg_mn) {
  Kv4Group r;
  const float mn = -neg_mn;
  r.bad = !(__fsub_rn(mx, mn) < INFINITY);  // NaN, an infinity, or a range past fp32's largest
  const float half = __fsub_rn(__fmul_rn(mx, 0.5f), __fmul_rn(mn, 0.5f));
  float scale = round_bf16(__fdiv_rn(half, 7.5f));
  if (scale < 7.888609052210118e-31f) scale = 0.f;  // 2^-100: 1 / scale stays finite, codes stay below 16
  r.inv = (scale == 0.f || r.bad) ? 0.f : __fmul_rn(__frcp_rn(scale), 1.000000238418579f);
  r.low = r.bad ? 0.f : mn;
  r.param = r.bad ? 0x00007FC0u
                  : ((__float_as_uint(scale) >> 16) | (__float_as_uint(mn) & 0xFFFF0000u));
  return r;
}

// 2^23 + code, as bits: 0x4B000000 + code (x finite)
__device__ __forceinline__ uint32_t kv4_code_bits(float x, const Kv4Group& gp) {
  const float u = __fadd_rn(__fmul_rn(__fsub_rn(x, gp.low), gp.inv), 0.5f);
  return __float_as_uint(__fadd_rz(u, 8388608.f));
}
// the same for two values: 2^23 + codes, as bits
__device__ __forceinline__ uint2 kv4_code_bits2(uint32_t pair, float neg_low, float inv) {
  float2 v = make_float2(bf16_lo(pair), bf16_hi(pair));
  v = __fmul2_rn(__fadd2_rn(v, make_float2(neg_low, neg_low)), make_float2(inv, inv));
  v = __fadd2_rz(__fadd2_rn(v, make_float2(0.5f, 0.5f)), make_float2(8388608.f, 8388608.f));
  return make_uint2(__float_as_uint(v.x), __float_as_uint(v.y));
}
// the low bytes of four words, a's lowest
__device__ __forceinline__ uint32_t kv4_low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// byte of a V key inside its 16-key block's words, and its fragment column t
__device__ __forceinline__ int kv4_v_byte(int kb) { return ((kb & 1) << 1) | (kb >> 3); }
__device__ __forceinline__ int kv4_v_t(int kb) { return (kb & 7) >> 1; }

struct Kv4RowsParams {
  const __nv_bfloat16* k;      // write: (B, S, Hkv, 128) source; read: unused
  const __nv_bfloat16* v;
  __nv_bfloat16* k_out;        // read: destination
  __nv_bfloat16* v_out;
  int64_t k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;  // strides of the bf16 side (elements)
  uint8_t* cache;              // (B, Hkv, tiles, 4608)
  int64_t c_sb, c_sh;          // cache strides (bytes)
  int start, count;            // slots [start, start + count)
  int Hkv, blk0;               // 16-key blocks that the slots touch start at block blk0
  unsigned items;              // warps of a batch row: blocks * 2 * Hkv
};

// (max, -min) of 8 bf16 values, as a bf16 pair; NaN propagates
__device__ __forceinline__ __nv_bfloat162 kv4_minmax8(const uint4 x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  __nv_bfloat162 mx = *reinterpret_cast<const __nv_bfloat162*>(&w[0]), mn = mx;
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162*>(&w[i]);
    mx = __hmax2_nan(mx, a);
    mn = __hmin2_nan(mn, a);
  }
  const uint32_t a = *reinterpret_cast<uint32_t*>(&mx), b = *reinterpret_cast<uint32_t*>(&mn) ^ 0x80008000u;
  const uint32_t lo = __byte_perm(a, b, 0x5410), hi = __byte_perm(a, b, 0x7632);  // (max, -min) of the even, the odd
  return __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&lo), *reinterpret_cast<const __nv_bfloat162*>(&hi));
}
__device__ __forceinline__ __nv_bfloat162 shfl_xor_bf162(__nv_bfloat162 v, int off) {
  uint32_t u = *reinterpret_cast<uint32_t*>(&v);
  u = __shfl_xor_sync(0xffffffffu, u, off);
  return *reinterpret_cast<__nv_bfloat162*>(&u);
}

// Bulk write. A warp takes one item = (batch row, 16-key block, half of the
// block's key quads, kv head): lane = 16 tt + c handles dims 8 c .. 8 c + 7 of
// the four keys 2 t, 2 t + 8, 2 t + 1, 2 t + 9 (t = 2 half + tt) of K and of V:
// exactly the keys of its V words, so V is transposed with four lane
// exchanges and no shared memory. Reads are whole 256-byte rows, writes whole
// 32-byte sectors. Consecutive warps take consecutive heads of the same keys
// (adjacent in the source). Rows outside [start, start + count) are neither
// read nor written; a word that mixes both is written byte by byte.
// Bound by instructions as much as by memory (35 us under ncu: issue slots 73 %
// busy, DRAM 49 %), so: the extrema of a lane's 8 rows are reduced and scattered
// in one exchange (lane c % 8 ends up with row c % 8's, 7 shuffles instead of
// 24) and a row's step and reciprocal are computed by that lane alone; codes
// come two at a time (packed fp32) and are gathered by byte permutations. 32768
// keys of 8 heads: 59 us before that (22 instructions a value), 32.1 us now (12;
// 172 MB, 5.4 TB/s = 82 % of a copy's rate), of which extrema and steps are a
// seventh; four blocks an SM (three: 9 % more).
__global__ void __launch_bounds__(256, 4) kv4_write_kernel(const Kv4RowsParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, c = lane & 15;
  const unsigned item = blockIdx.x * 8u + (threadIdx.x >> 5);
  if (item >= p.items) return;
  const unsigned rest = item / (unsigned)p.Hkv;
  const int h = (int)(item - rest * (unsigned)p.Hkv), blk = p.blk0 + (int)(rest >> 1);
  const int t = 2 * (int)(rest & 1u) + (lane >> 4);
  const int64_t b = blockIdx.y;
  // row of key 2 t + {0, 8, 1, 9} in the source
  const int r0 = blk * 16 + 2 * t - p.start;
  const __nv_bfloat16* kb = p.k + b * p.k_sb + (int64_t)h * p.k_sh + (int64_t)r0 * p.k_ss + 8 * c;
  const __nv_bfloat16* vb = p.v + b * p.v_sb + (int64_t)h * p.v_sh + (int64_t)r0 * p.v_ss + 8 * c;
  uint8_t* tile = p.cache + b * p.c_sb + (int64_t)h * p.c_sh + (int64_t)(blk >> 1) * kKv4TileBytes;
  const int row0 = (blk & 1) * 16 + 2 * t;
  uint4 x[8];  // K then V
  bool in[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) in[j] = (unsigned)(r0 + (j >> 1) + 8 * (j & 1)) < (unsigned)p.count;
  const bool whole = in[0] && in[1] && in[2] && in[3];
  auto load = [&](int j) {
    const int dr = (j >> 1) + 8 * (j & 1);
    x[j] = ld_nc_v4(reinterpret_cast<const uint4*>(kb + dr * p.k_ss));
    x[4 + j] = ld_nc_v4(reinterpret_cast<const uint4*>(vb + dr * p.v_ss));
  };
  if (__all_sync(0xffffffffu, whole)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) load(j);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = x[4 + j] = make_uint4(0u, 0u, 0u, 0u);
      if (in[j]) load(j);
    }
  }
  // ---- extrema of the 8 rows: rows split over the lanes as the lanes are merged
  __nv_bfloat162 mm[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) mm[r] = kv4_minmax8(x[r]);
#pragma unroll
  for (int off = 4; off >= 1; off >>= 1) {
    const bool up = (c & off) != 0;
#pragma unroll
    for (int r = 0; r < off; ++r) {
      const __nv_bfloat162 give = up ? mm[r] : mm[r + off], keep = up ? mm[r + off] : mm[r];
      mm[r] = __hmax2_nan(keep, shfl_xor_bf162(give, off));
    }
  }
  const Kv4Group own = kv4_group(__low2float(mm[0]), __high2float(mm[0]));  // of row c % 8
  {
    const int j = c & 3, row = row0 + (j >> 1) + 8 * (j & 1);
    if (j == 0 ? in[0] : j == 1 ? in[1] : j == 2 ? in[2] : in[3])
      *reinterpret_cast<uint32_t*>(tile + ((c & 4) ? kKv4Vp : kKv4Kp) + row * 8 + (c >> 3) * 4) = own.param;
  }
  float neg_low[8], inv[8];
  const float own_neg = -own.low;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    neg_low[r] = __shfl_sync(0xffffffffu, own_neg, (lane & 24) | r);
    inv[r] = __shfl_sync(0xffffffffu, own.inv, (lane & 24) | r);
  }
  if (__any_sync(0xffffffffu, own.bad)) {
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (__shfl_sync(0xffffffffu, own.bad, (lane & 24) | r)) x[r] = make_uint4(0u, 0u, 0u, 0u);  // codes of 0
  }
  // ---- K: the lane's 8 codes are one word of the row
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
    uint32_t two[4];  // a pair's codes in the low byte
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint2 n = kv4_code_bits2(w[e], neg_low[j], inv[j]);
      two[e] = n.x + (n.y << 4);
    }
    const uint32_t word = kv4_low_bytes(two[0], two[1], two[2], two[3]);
    const int row = row0 + (j >> 1) + 8 * (j & 1);
    if (in[j]) *reinterpret_cast<uint32_t*>(tile + row * 64 + (c & 3) * 16 + (c >> 2) * 4) = word;
  }
  // ---- V: byte j of word g = the code of key j at this lane's dim g
  uint32_t acc[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint2 n[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint4 q = x[4 + j];
      n[j] = kv4_code_bits2(e == 0 ? q.x : e == 1 ? q.y : e == 2 ? q.z : q.w, neg_low[4 + j], inv[4 + j]);
    }
    acc[2 * e] = kv4_low_bytes(n[0].x, n[1].x, n[2].x, n[3].x);
    acc[2 * e + 1] = kv4_low_bytes(n[0].y, n[1].y, n[2].y, n[3].y);
  }
  // lanes c (even: low nibbles) and c + 1 (high nibbles) make the 8 words of
  // their 16 dims: the even lane words g = 0..3, the odd one 4..7
  const int odd = c & 1, wd = c >> 1;
  uint8_t* vt = tile + kKv4V + (blk & 1) * 1024 + (wd >> 2) * 512 + t * 16 + (wd & 3) * 4;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const uint32_t give = odd ? acc[g] : acc[4 + g], mine = odd ? acc[4 + g] : acc[g];
    const uint32_t got = __shfl_xor_sync(0xffffffffu, give, 1);
    const uint32_t word = odd ? (mine << 4) | got : mine | (got << 4);
    uint8_t* at = vt + (4 * odd + g) * 64;
    if (whole) {
      *reinterpret_cast<uint32_t*>(at) = word;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (in[j]) at[j] = (uint8_t)(word >> (8 * j));
    }
  }
}

// Read back: the same item and lane mapping, the other way. A nibble becomes a
// float by a byte permutation under the exponent of 2^23 and one packed
// subtraction. Bound by memory: 28.8 us for 32768 keys of 8 heads (91 %).
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4RowsParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, c = lane & 15;
  const unsigned item = blockIdx.x * 8u + (threadIdx.x >> 5);
  if (item >= p.items) return;
  const unsigned rest = item / (unsigned)p.Hkv;
  const int h = (int)(item - rest * (unsigned)p.Hkv), blk = p.blk0 + (int)(rest >> 1);
  const int t = 2 * (int)(rest & 1u) + (lane >> 4);
  const int64_t b = blockIdx.y;
  const uint8_t* tile = p.cache + b * p.c_sb + (int64_t)h * p.c_sh + (int64_t)(blk >> 1) * kKv4TileBytes;
  const int row0 = (blk & 1) * 16 + 2 * t;
  const int odd = c & 1, wd = c >> 1;
  uint32_t kw[4], kp[4], vp[4], vw[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {  // a tile is allocated whole: rows past the range are read, not returned
    const int row = row0 + (j >> 1) + 8 * (j & 1);
    kw[j] = *reinterpret_cast<const uint32_t*>(tile + row * 64 + (c & 3) * 16 + (c >> 2) * 4);
    kp[j] = *reinterpret_cast<const uint32_t*>(tile + kKv4Kp + row * 8 + (c >> 3) * 4);
    vp[j] = *reinterpret_cast<const uint32_t*>(tile + kKv4Vp + row * 8 + (c >> 3) * 4);
    vw[j] = *reinterpret_cast<const uint32_t*>(tile + kKv4V + (blk & 1) * 1024 + (wd >> 2) * 512 +
                                               ((4 * odd + j) * 4 + t) * 16 + (wd & 3) * 4);
  }
  uint32_t acc[8];  // byte j of word g = the code of key j at this lane's dim g
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    // my words are g' = 4 odd + g, the partner's the other four; I keep my nibble of all eight
    const uint32_t got = __shfl_xor_sync(0xffffffffu, vw[g], 1);
    const uint32_t a = odd ? got : vw[g], d = odd ? vw[g] : got;
    acc[g] = (a >> (4 * odd)) & 0x0F0F0F0Fu;
    acc[4 + g] = (d >> (4 * odd)) & 0x0F0F0F0Fu;
  }
  const int r0 = blk * 16 + 2 * t - p.start;
  __nv_bfloat16* kb = p.k_out + b * p.k_sb + (int64_t)h * p.k_sh + (int64_t)r0 * p.k_ss + 8 * c;
  __nv_bfloat16* vb = p.v_out + b * p.v_sb + (int64_t)h * p.v_sh + (int64_t)r0 * p.v_ss + 8 * c;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int dr = (j >> 1) + 8 * (j & 1);
    if ((unsigned)(r0 + dr) >= (unsigned)p.count) continue;
    const float ks = __uint_as_float(kp[j] << 16), kl = __uint_as_float(kp[j] & 0xFFFF0000u);
    const float vs = __uint_as_float(vp[j] << 16), vl = __uint_as_float(vp[j] & 0xFFFF0000u);
    const float2 ks2 = make_float2(ks, ks), kl2 = make_float2(kl, kl), vs2 = make_float2(vs, vs), vl2 = make_float2(vl, vl);
    const uint32_t even = kw[j] & 0x0F0F0F0Fu, high = (kw[j] >> 4) & 0x0F0F0F0Fu;  // dims 2 e, 2 e + 1
    uint32_t ok[4], ov[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // prmt: bytes 0..3 of the codes, 4..7 of 0x4B000000 (7: the exponent, 4: zero)
      float2 v = make_float2(__uint_as_float(__byte_perm(even, 0x4B000000u, 0x7440 + e)),
                             __uint_as_float(__byte_perm(high, 0x4B000000u, 0x7440 + e)));
      v = __ffma2_rn(__fadd2_rn(v, make_float2(-8388608.f, -8388608.f)), ks2, kl2);
      ok[e] = pack_bf16x2(v.x, v.y);
      v = make_float2(__uint_as_float(__byte_perm(acc[2 * e], 0x4B000000u, 0x7440 + j)),
                      __uint_as_float(__byte_perm(acc[2 * e + 1], 0x4B000000u, 0x7440 + j)));
      v = __ffma2_rn(__fadd2_rn(v, make_float2(-8388608.f, -8388608.f)), vs2, vl2);
      ov[e] = pack_bf16x2(v.x, v.y);
    }
    *reinterpret_cast<uint4*>(kb + dr * p.k_ss) = make_uint4(ok[0], ok[1], ok[2], ok[3]);
    *reinterpret_cast<uint4*>(vb + dr * p.v_ss) = make_uint4(ov[0], ov[1], ov[2], ov[3]);
  }
}

struct Kv4AppendParams {
  const __nv_bfloat16* q;  // (rows, n_q, 128), row stride ld_q
  const __nv_bfloat16* k;  // (rows, n_k, 128)
  const __nv_bfloat16* v;
  __nv_bfloat16* q_out;    // (rows, n_q, 128), row stride ld_qo
  int64_t ld_q, ld_k, ld_v, ld_qo;
  const __nv_bfloat16* q_w;
  const __nv_bfloat16* k_w;
  const __nv_bfloat16* cos;  // (rows, 128), row stride ld_cs
  const __nv_bfloat16* sin;
  int64_t ld_cs;
  uint8_t* cache;
  int64_t c_sb, c_sh;
  const int64_t* slot;  // device
  int64_t slots;        // slots the cache holds; a slot outside is not written
  int rows, n_q, n_k;
  float eps;
};

constexpr int kKv4AppendThreads = 128;  // 8 heads per block, one per half-warp

// One decode token per row: q and k heads RMS-normalised and rotated in fp32
// with one rounding to bf16, q to q_out, k and v quantised into slot *slot.
// A half-warp takes one head (of q, k or v): lane l holds dims 4 l .. 4 l + 3
// and their rotate-half partners 64 + 4 l .., which are also the two groups,
// so the rotation needs no exchange and each group is one reduction over the
// 16 lanes. Latency-bound (one token): one head per half-warp and every load
// issued before any arithmetic. The mean square is summed in fp64 (squares of
// bf16 values are exact in it), so a code never hangs on the summation order.
__global__ void __launch_bounds__(kKv4AppendThreads) kv4_append_kernel(const Kv4AppendParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int hl = threadIdx.x & 15;
  const int heads = p.n_q + 2 * p.n_k;
  const int64_t unit = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 4;
  const bool live = unit < (int64_t)p.rows * heads;  // the shuffles below need every lane of the warp
  const int64_t row = live ? unit / heads : 0;
  const int hd = live ? (int)(unit - row * heads) : 0;
  const int kind = hd < p.n_q ? 0 : hd < p.n_q + p.n_k ? 1 : 2;  // q, k, v
  const int hk = hd - p.n_q - (kind == 2 ? p.n_k : 0);
  const __nv_bfloat16* src = kind == 0   ? p.q + row * p.ld_q + (int64_t)hd * 128
                             : kind == 1 ? p.k + row * p.ld_k + (int64_t)hk * 128
                                         : p.v + row * p.ld_v + (int64_t)hk * 128;
  const uint2 xl = reinterpret_cast<const uint2*>(src)[hl], xh = reinterpret_cast<const uint2*>(src)[16 + hl];
  const uint2* wp = reinterpret_cast<const uint2*>(kind == 0 ? p.q_w : p.k_w);
  const uint2* cp = reinterpret_cast<const uint2*>(p.cos + row * p.ld_cs);
  const uint2* sp = reinterpret_cast<const uint2*>(p.sin + row * p.ld_cs);
  const uint2 wl = __ldg(wp + hl), wh = __ldg(wp + 16 + hl);
  const uint2 cl = __ldg(cp + hl), ch = __ldg(cp + 16 + hl), sl = __ldg(sp + hl), sh = __ldg(sp + 16 + hl);
  const int64_t slot = __ldg(p.slot);
  float a[4] = {bf16_lo(xl.x), bf16_hi(xl.x), bf16_lo(xl.y), bf16_hi(xl.y)};
  float d[4] = {bf16_lo(xh.x), bf16_hi(xh.x), bf16_lo(xh.y), bf16_hi(xh.y)};
  double ss = 0.0;
#pragma unroll
  for (int e = 0; e < 4; ++e) ss += (double)(a[e] * a[e]) + (double)(d[e] * d[e]);
#pragma unroll
  for (int off = 8; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
  if (kind < 2) {
    const float rs = rsqrtf((float)(ss * (1.0 / 128.0) + (double)p.eps));
    const float w0[4] = {bf16_lo(wl.x), bf16_hi(wl.x), bf16_lo(wl.y), bf16_hi(wl.y)};
    const float w1[4] = {bf16_lo(wh.x), bf16_hi(wh.x), bf16_lo(wh.y), bf16_hi(wh.y)};
    const float c0[4] = {bf16_lo(cl.x), bf16_hi(cl.x), bf16_lo(cl.y), bf16_hi(cl.y)};
    const float c1[4] = {bf16_lo(ch.x), bf16_hi(ch.x), bf16_lo(ch.y), bf16_hi(ch.y)};
    const float s0[4] = {bf16_lo(sl.x), bf16_hi(sl.x), bf16_lo(sl.y), bf16_hi(sl.y)};
    const float s1[4] = {bf16_lo(sh.x), bf16_hi(sh.x), bf16_lo(sh.y), bf16_hi(sh.y)};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float ya = __fmul_rn(__fmul_rn(a[e], rs), w0[e]), yd = __fmul_rn(__fmul_rn(d[e], rs), w1[e]);
      a[e] = round_bf16(__fadd_rn(__fmul_rn(ya, c0[e]), __fmul_rn(-yd, s0[e])));
      d[e] = round_bf16(__fadd_rn(__fmul_rn(yd, c1[e]), __fmul_rn(ya, s1[e])));
    }
  }
  const uint32_t oa0 = pack_bf16x2(a[0], a[1]), oa1 = pack_bf16x2(a[2], a[3]);
  const uint32_t od0 = pack_bf16x2(d[0], d[1]), od1 = pack_bf16x2(d[2], d[3]);
  if (live && kind == 0) {
    uint2* dst = reinterpret_cast<uint2*>(p.q_out + row * p.ld_qo + (int64_t)hd * 128);
    dst[hl] = make_uint2(oa0, oa1);
    dst[16 + hl] = make_uint2(od0, od1);
  }
  // the two groups' (max, -min); q lanes run along (the shuffles need the warp)
  __nv_bfloat162 ma, md;
  {
    const __nv_bfloat162 u0 = *reinterpret_cast<const __nv_bfloat162*>(&oa0), u1 = *reinterpret_cast<const __nv_bfloat162*>(&oa1);
    const __nv_bfloat162 e0 = *reinterpret_cast<const __nv_bfloat162*>(&od0), e1 = *reinterpret_cast<const __nv_bfloat162*>(&od1);
    const __nv_bfloat162 x0 = __hmax2_nan(u0, u1), n0 = __hmin2_nan(u0, u1), x1 = __hmax2_nan(e0, e1), n1 = __hmin2_nan(e0, e1);
    ma = __halves2bfloat162(__hmax_nan(__low2bfloat16(x0), __high2bfloat16(x0)),
                            __hneg(__hmin_nan(__low2bfloat16(n0), __high2bfloat16(n0))));
    md = __halves2bfloat162(__hmax_nan(__low2bfloat16(x1), __high2bfloat16(x1)),
                            __hneg(__hmin_nan(__low2bfloat16(n1), __high2bfloat16(n1))));
  }
#pragma unroll
  for (int off = 8; off >= 1; off >>= 1) {
    ma = __hmax2_nan(ma, shfl_xor_bf162(ma, off));
    md = __hmax2_nan(md, shfl_xor_bf162(md, off));
  }
  const Kv4Group ga = kv4_group(__low2float(ma), __high2float(ma)), gd = kv4_group(__low2float(md), __high2float(md));
  uint32_t na[4], nd[4];  // codes
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    na[e] = ga.bad ? 0u : kv4_code_bits(a[e], ga) - 0x4B000000u;
    nd[e] = gd.bad ? 0u : kv4_code_bits(d[e], gd) - 0x4B000000u;
  }
  // V: dims 16 w + g and 16 w + g + 8 share a byte: lanes hl and hl ^ 2
  const uint32_t pa = na[0] | na[1] << 8 | na[2] << 16 | na[3] << 24;
  const uint32_t pd = nd[0] | nd[1] << 8 | nd[2] << 16 | nd[3] << 24;
  const uint32_t qa = __shfl_xor_sync(0xffffffffu, pa, 2), qd = __shfl_xor_sync(0xffffffffu, pd, 2);
  if (!live || kind == 0 || slot < 0 || slot >= p.slots) return;
  uint8_t* tile = p.cache + row * p.c_sb + (int64_t)hk * p.c_sh + (slot >> 5) * kKv4TileBytes;
  const int key = (int)(slot & 31);
  if (hl == 0)
    *reinterpret_cast<uint2*>(tile + (kind == 1 ? kKv4Kp : kKv4Vp) + key * 8) = make_uint2(ga.param, gd.param);
  if (kind == 1) {
    // dims 4 hl ..: half hl & 1 of word i = hl / 8 of piece (hl / 2) % 4; the upper group two words on
    uint8_t* at = tile + key * 64 + ((hl >> 1) & 3) * 16 + (hl >> 3) * 4 + (hl & 1) * 2;
    *reinterpret_cast<uint16_t*>(at) = (uint16_t)(na[0] | na[1] << 4 | na[2] << 8 | na[3] << 12);
    *reinterpret_cast<uint16_t*>(at + 8) = (uint16_t)(nd[0] | nd[1] << 4 | nd[2] << 8 | nd[3] << 12);
  } else if ((hl & 2) == 0) {
    const int kb = key & 15;
    uint8_t* at = tile + kKv4V + (key >> 4) * 1024 + kv4_v_t(kb) * 16 + (hl >> 2) * 4 + kv4_v_byte(kb);
    const uint32_t ba = pa | qa << 4, bd = pd | qd << 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      at[((hl & 1) * 4 + e) * 64] = (uint8_t)(ba >> (8 * e));
      at[((hl & 1) * 4 + e) * 64 + 512] = (uint8_t)(bd >> (8 * e));
    }
  }
}

}  // namespace tg

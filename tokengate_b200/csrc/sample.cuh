// Sampling of the next token: temperature, top-k, top-p and min-p from a given
// uniform number per row.
//
//   d_i = x_i / T - x_max / T, w_i = exp(d_i)             (fp32; NaN logits count as -inf)
//   order the row by (x descending, index ascending);
//   keep its first k, then the shortest prefix whose mass reaches p times the
//   mass of those k, then of these every w_i >= min_p (w = 1 is the largest);
//   token = the first index, in index order, at which the running kept mass
//   passes u times the kept mass; logprob = d_token - log(kept mass).
// T <= 0 (or NaN) is greedy. Masses are sums of w * 2^44 in integers, exact, so
// the token depends on no order of summing and every block of a cluster takes
// the same decision (V <= 2^19 keeps them in 64 bits).
//
// A cluster of C blocks takes a row, each an index range of it, whose weights
// it computes once and keeps in shared memory. Bound by latencies (barriers of
// the cluster and of the block, one after another) and by instructions, not by
// memory: the row is read once. 64 fp32 rows of 151936, rules of all kinds: 61
// us, in two rounds of clusters of about 28, of which 4 are the logits' load,
// 5.5 the weights and the histogram, 3 a look's pass, the rest exchanges (issue
// slots 43 % busy where an SM works, 78 instructions a logit). No sort: the k-th
// value (or the value at which the mass reaches p) is found
//   1. by a histogram over 1024 buckets of w, 32 to an octave (linear in w's
//      bits: two instructions, and nearly linear in the logit, so that logits
//      spread over many buckets and shared-memory atomics seldom collide):
//      counts, exact for k; for p the guess that a bucket's logits weigh its
//      middle each. Each block owns a slice of the row's and hands it to the
//      others;
//   2. exactly inside that bucket (or two, where the guess is near an edge):
//      one pass gives the mass above and in it, its smallest and largest logit
//      and the list of its logits (after a wrong guess, the next one from
//      there); where the two differ, every block narrows them down on a copy of
//      all lists, so without a cluster barrier (lists too long for that: by
//      digits, with one each).
// Where no more than 256 logits reach down to the k-th's bucket, they go to one
// block, which orders them by counting and finishes alone (k = 50, p = 0.9: one
// row of 151936 18.3 -> 12.5 us, 64 rows 70 -> 43).
// The threshold is a logit and a number of its ties, which go by index. What is
// kept is then marked in the weights (ties negative), for the walk to the token.
// Blocks write to one another's shared memory and read their own: a remote load
// costs the reader its latency, and sixteen blocks reading one word queue up.
#pragma once

#include <cooperative_groups.h>

#include "ptx.cuh"

namespace tg {

constexpr int kSmpThreads = 512;
constexpr int kSmpWarps = kSmpThreads / 32;
constexpr int kSmpBuckets = 1024;
constexpr int kSmpList = 1024;      // logits of one bucket that a block can list
constexpr int kSmpAllLists = 2048;  // and the cluster
constexpr uint32_t kSmpNoLists = 0xFFFFFFFFu;
constexpr int kSmpCompare = 64;     // listed logits that are compared each with all
constexpr int kSmpFew = 256;        // logits that one block orders by counting
constexpr int kSmpMaxCluster = 16;   // above 8: opt-in
constexpr int kSmpMaxV = 1 << 19;
constexpr double kSmpUnit = 1.0 / 17592186044416.0;  // 2^-44: a mass of 1

struct SampleParams {
  const void* logits;
  int64_t row_stride;  // elements
  int V, chunk;        // indices per block, a multiple of kSmpThreads below 2^16 (the last blocks may hold fewer or none)
  const float* u;
  const float* temperature;
  const int32_t* top_k;   // nullable
  const float* top_p;     // nullable
  const float* min_p;     // nullable
  int64_t* token;
  float* logprob;         // nullable
};

typedef unsigned long long smp_u64;

struct alignas(16) SmpShared {
  uint32_t own[2][kSmpBuckets];   // [0]: this block's histogram; then lists of a bucket's logits, by turns
  uint32_t tot[kSmpBuckets];      // the row's histogram
  union {
    uint32_t all[kSmpAllLists];   // this block's slice of the row's histogram; then the blocks' lists together
    struct {                      // or, in block 0, the few logits down to the k-th's bucket
      smp_u64 few_ord[kSmpFew];   // ordered logit above the index's complement: the order of the row, descending
      smp_u64 few_mass[kSmpFew];
    };
  };
  uint16_t at[kSmpList];          // where in the block's range the listed logits are
  uint32_t dig[2][3][256];        // digit histograms of a refinement, by pass parity: masses in three pieces of 15 bits
  smp_u64 xch[2][kSmpMaxCluster][4];  // what each block of the cluster has sent, by turns
  smp_u64 red[kSmpWarps][4];
  double scan[kSmpWarps];
  smp_u64 pick_above;
  int pick;
  uint32_t n_list, n_few, key_lo, key_hi;
};

__device__ __forceinline__ uint32_t smp_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float smp_unkey(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ float smp_logit(float x) { return x == x ? x + 0.f : -INFINITY; }  // -0 orders as +0
__device__ __forceinline__ float smp_load(const float* p) { return smp_logit(*p); }
__device__ __forceinline__ float smp_load(const __nv_bfloat16* p) { return smp_logit(__bfloat162float(*p)); }

// x / T as x * (1/T) with 1/T held as a sum of two floats (N. Brisebarre and
// J.-M. Muller, "Correctly rounded multiplication by arbitrary precision
// constants", 2008): x * high + RN(x * low) in one fma is within 2^-47 of the
// quotient before its rounding, a division's cost without a division. Outside
// the range of T in which the low part is a normal number and below 1 (so that
// the type's lowest logit times it stays finite, and short of the high part's
// product), and for rows whose maximum is huge or infinite, the division itself.
struct SmpRow {
  float xmax, zmax, t, rh, rl;
  bool plain;  // the usual row: a finite maximum, and quotients as products
  __device__ __forceinline__ void set(float x, float tt) {
    xmax = x;
    t = tt;
    rh = __frcp_rn(t);
    rl = __fdiv_rn(__fmaf_rn(-t, rh, 1.f), t);
    plain = t > 9.5367432e-7f && t < 1.1529215e18f && fabsf(x) < 1e18f;  // 2^-20 < T < 2^60
    zmax = plain ? product(x) : __fdiv_rn(x, t);
  }
  __device__ __forceinline__ float product(float x) const { return __fmaf_rn(x, rh, __fmul_rn(x, rl)); }
};
// exp, held to [0, 1], which the buckets rely on; 0 for NaN
__device__ __forceinline__ float smp_exp(float d) { return __saturatef(expf(d)); }
// The weights of two logits, as smp_exp(smp_d) gives them, of a usual row: two at
// a time up to the exponentials.
__device__ __forceinline__ float2 smp_weights2(float x, float y, const SmpRow& r) {
  float2 d;
  asm("{\n\t.reg .b64 a, h, l, z;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 h, {%4, %4};\n\tmov.b64 l, {%5, %5};\n\tmov.b64 z, {%6, %6};\n\t"
      "mul.rn.f32x2 l, a, l;\n\tfma.rn.f32x2 a, a, h, l;\n\tadd.rn.f32x2 a, a, z;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(x), "f"(y), "f"(r.rh), "f"(r.rl), "f"(-r.zmax));
  return make_float2(smp_exp(d.x), smp_exp(d.y));
}
__device__ __forceinline__ float smp_d(float x, const SmpRow& r) {
  float d;
  if (r.plain) {
    d = __fsub_rn(r.product(x), r.zmax);
  } else {
    d = x == r.xmax ? 0.f : __fsub_rn(__fdiv_rn(x, r.t), r.zmax);
  }
  return d <= 0.f ? d : -INFINITY;  // NaN: a NaN logit, -inf times 0, or quotients that both overflowed
}
// Bucket e holds the weights in (smp_upper(e + 1), smp_upper(e)], the last one all the positive ones below.
__device__ __forceinline__ uint32_t smp_bucket(float w) {
  return min((0x3F800000u - __float_as_uint(w)) >> 18, (uint32_t)kSmpBuckets - 1u);
}
__device__ __forceinline__ float smp_upper(int e) {
  return e >= kSmpBuckets ? 0.f : __uint_as_float(0x3F800000u - ((uint32_t)e << 18));
}
// A mass: w * 2^44 cut to an integer. A thread sums up to 256 of them in a
// double that starts at 256, whose last bit is worth 2^-44: the cut is the
// addition's own, two instructions a weight where integers take six.
__device__ __forceinline__ smp_u64 smp_mass(float w) { return (smp_u64)__float2ull_rz(w * 17592186044416.f); }
struct SmpSum {
  double v = 256.;
  __device__ __forceinline__ void add(float w) { v = __dadd_rz(v, (double)w); }
  __device__ __forceinline__ smp_u64 get() const {
    return (smp_u64)__double_as_longlong(v) & ((1ull << 52) - 1ull);  // v in [256, 512): the mantissa counts
  }
};

// sum over the warp: 24-bit pieces (32 of them stay below 2^32), one reduction instruction each
__device__ __forceinline__ smp_u64 smp_warp_sum(smp_u64 v) {
  const uint32_t a = __reduce_add_sync(0xffffffffu, (uint32_t)v & 0xFFFFFFu);
  const uint32_t b = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 24) & 0xFFFFFFu);
  const uint32_t c = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 48));
  return a + ((smp_u64)b << 24) + ((smp_u64)c << 48);
}
__device__ __forceinline__ smp_u64 smp_warp_scan(smp_u64 v, int lane) {  // inclusive
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const smp_u64 a = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += a;
  }
  return v;
}
__device__ __forceinline__ uint32_t smp_warp_max(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ uint32_t smp_warp_min(uint32_t v) { return __reduce_min_sync(0xffffffffu, v); }

// One row's state in a block.
template <typename T>
struct Smp {
  SmpShared& s;
  const T* x;   // the block's range of the row
  float* sw;    // the range's weights (at first its logits, as fp32)
  int C, rank, n, w0, w1, lane, warp;  // this warp's indices [w0, w1) of the range, contiguous: index order is warp order
  SmpRow row;
  int turn, parity;

  __device__ __forceinline__ void sync() {
    if (C > 1) {
      __syncwarp();  // the cluster barrier wants whole warps
      cluster_sync_all();
    } else {
      __syncthreads();
    }
  }
  // Logits i to i + 3 (i a multiple of 4; -inf past the range)
  __device__ __forceinline__ float4 logits4(int i) const {
    constexpr int kBytes = 4 * sizeof(T);
    if ((reinterpret_cast<uintptr_t>(x) & (kBytes - 1)) == 0 && i + 4 <= n) {
      if constexpr (sizeof(T) == 4) {
        return __ldg(reinterpret_cast<const float4*>(x + i));
      } else {
        const uint2 q = __ldg(reinterpret_cast<const uint2*>(x + i));
        return make_float4(__uint_as_float(q.x << 16), __uint_as_float(q.x & 0xFFFF0000u), __uint_as_float(q.y << 16),
                           __uint_as_float(q.y & 0xFFFF0000u));
      }
    }
    float f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = i + e < n ? smp_load(x + i + e) : -INFINITY;
    return make_float4(f[0], f[1], f[2], f[3]);
  }
  __device__ __forceinline__ float weight_of(float logit) const { return smp_exp(smp_d(logit, row)); }
  // f(i, what is held of indices i to i + 3) over this warp's range, each lane every 32nd four
  template <typename F>
  __device__ __forceinline__ void each4(F f) const {
#pragma unroll 2
    for (int i = w0 + 4 * lane; i < w1; i += 128) f(i, *reinterpret_cast<float4*>(sw + i));
  }
  template <typename V>
  __device__ __forceinline__ V* remote(V* p, int r) const {
    return C > 1 ? cooperative_groups::this_cluster().map_shared_rank(p, r) : p;
  }
  // To every thread: the sums of a and b, the minimum lo, the maximum hi and the sum of cnt (one value per block)
  // over the cluster; before[2]: a and b of the blocks of lower rank. s.red[w][0 .. 1] keeps a and b of warp w.
  __device__ __forceinline__ void reduce(smp_u64& a, smp_u64& b, uint32_t& lo, uint32_t& hi, uint32_t& cnt,
                                         smp_u64* before) {
    a = smp_warp_sum(a);
    b = smp_warp_sum(b);
    lo = smp_warp_min(lo);
    hi = smp_warp_max(hi);
    if (lane == 0) {
      s.red[warp][0] = a;
      s.red[warp][1] = b;
      s.red[warp][2] = lo;
      s.red[warp][3] = hi;
    }
    __syncthreads();
    smp_u64(*o)[4] = s.xch[turn];
    turn ^= 1;
    if (warp == 0) {
      const bool in = lane < kSmpWarps;
      a = smp_warp_sum(in ? s.red[lane][0] : 0ull);
      b = smp_warp_sum(in ? s.red[lane][1] : 0ull);
      lo = smp_warp_min(in ? (uint32_t)s.red[lane][2] : 0xFFFFFFFFu);
      hi = smp_warp_max(in ? (uint32_t)s.red[lane][3] : 0u);
      if (lane < C) {
        smp_u64* to = remote(o[rank], lane);
        to[0] = a;
        to[1] = b;
        to[2] = lo | (smp_u64)hi << 32;
        to[3] = s.n_list;
      }
    }
    sync();
    a = b = 0;
    lo = 0xFFFFFFFFu;
    hi = cnt = 0;
    if (lane < C) {
      a = o[lane][0];
      b = o[lane][1];
      lo = (uint32_t)o[lane][2];
      hi = (uint32_t)(o[lane][2] >> 32);
      cnt = (uint32_t)o[lane][3];
    }
    if (before != nullptr) {
      const smp_u64 sa = smp_warp_scan(a, lane) - a, sb = smp_warp_scan(b, lane) - b;
      before[0] = __shfl_sync(0xffffffffu, sa, rank);
      before[1] = __shfl_sync(0xffffffffu, sb, rank);
    }
    a = smp_warp_sum(a);
    b = smp_warp_sum(b);
    lo = smp_warp_min(lo);
    hi = smp_warp_max(hi);
    const bool over = __any_sync(0xffffffffu, cnt > kSmpList);  // some block's list ran over
    cnt = __reduce_add_sync(0xffffffffu, cnt);
    if (over) cnt = kSmpNoLists;
  }

  // The row's histogram into every block's s.tot: each block's goes to the owners of its slices, and from there to
  // all. In two steps, with a cluster barrier after each.
  __device__ __forceinline__ void merge_to_owner() {
    const int slice = kSmpBuckets / C;
    for (int i = threadIdx.x; i < kSmpBuckets; i += kSmpThreads) {
      const uint32_t v = s.own[0][i];
      if (C == 1) {
        s.tot[i] = v;
      } else if (v != 0u) {
        atomicAdd(remote(s.all, i / slice) + i % slice, v);
      }
    }
  }
  __device__ __forceinline__ void merge_to_all() {
    const int slice = kSmpBuckets / C;
    for (int i = threadIdx.x; i < kSmpBuckets / 4; i += kSmpThreads) {  // 4 buckets to one block
      const int to = i / (slice / 4), j = i % (slice / 4);
      *(reinterpret_cast<uint4*>(remote(s.tot, to) + rank * slice) + j) = *(reinterpret_cast<const uint4*>(s.all) + j);
    }
  }

  // First bucket at which the running count / mass reaches `target` (the last if none does), but of b0 to b1; what is
  // before it, and in it.
  // A bucket's mass is guessed as its count times its middle; the far tail's as next to nothing.
  template <bool BY_MASS>
  __device__ __forceinline__ int crossing(double target, int b0, int b1, double& above, double& inside) {
    constexpr int E = kSmpBuckets / kSmpThreads;
    const int tid = threadIdx.x;
    double v[E], run = 0.;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = E * tid + e;
      const uint32_t cnt = s.tot[i];
      if (BY_MASS) {
        const float mid = i == kSmpBuckets - 1 ? 1e-20f : __uint_as_float(0x3F800000u - ((uint32_t)i << 18) - (1u << 17));
        v[e] = (double)cnt * (double)mid;
        if (i == 0) v[e] += 1. - (double)mid;  // of the first bucket's one is the largest
      } else {
        v[e] = (double)cnt;
      }
      run += v[e];
    }
    const double mine = run;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const double a = __shfl_up_sync(0xffffffffu, run, off);
      if (lane >= off) run += a;
    }
    if (lane == 31) s.scan[warp] = run;
    if (tid == 0) s.pick = kSmpBuckets - 1;
    __syncthreads();
    double part = lane < kSmpWarps ? s.scan[lane] : 0.;  // the warps' sums, scanned by every warp
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const double a = __shfl_up_sync(0xffffffffu, part, off);
      if (lane >= off) part += a;
    }
    const double before_warp = __shfl_sync(0xffffffffu, part, warp > 0 ? warp - 1 : 0);
    double before = run - mine + (warp > 0 ? before_warp : 0.);
    // (a thread just past the crossing may try too: the sums of masses round)
    if (before <= target * (1. + 1e-9) && before + mine >= target) {
      double at = before;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        at += v[e];
        if (at >= target && v[e] > 0.) {
          atomicMin(&s.pick, E * tid + e);
          break;
        }
      }
    }
    __syncthreads();
    const int bk = min(max(s.pick, b0), b1);
    if (bk / E == tid) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (e < bk % E) before += v[e];
        if (e == bk % E) s.scan[1] = v[e];
      }
      s.scan[0] = before;
    }
    __syncthreads();
    above = s.scan[0];
    inside = s.scan[1];
    __syncthreads();
    return bk;
  }

  // Notes in s.at which of w, the weights of indices i to i + 3, are in (w_in, w_over], as long as there is room.
  __device__ __forceinline__ void note(int i, const float (&w)[4], float w_in, float w_over, uint32_t room) {
    bool in[4];
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) m += in[e] = w[e] > w_in && !(w[e] > w_over);
    if (m) {
      uint32_t j = atomicAdd(&s.n_list, m);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (in[e] && j < room) s.at[j] = (uint16_t)(i + e);
        j += in[e];
      }
    }
  }

  // Of the elements in buckets up to `b1` (only those of a logit above `floor_key`, which is below bucket b0 or in b1):
  // the mass above bucket b0, the mass in b0 to b1, the range of the logits there (hi 0: none). Each block lists its
  // logits there (0 for those not above floor_key), `cnt` in all.
  __device__ __forceinline__ void look(int b0, int b1, uint32_t floor_key, smp_u64& above, smp_u64& inside, uint32_t& lo,
                                       uint32_t& hi, uint32_t& cnt) {
    SmpSum over, in;
    const float w_over = smp_upper(b0), w_in = smp_upper(b1 + 1);
    uint32_t* list = s.own[turn];
    lo = 0xFFFFFFFFu;
    hi = 0;
    if (threadIdx.x == 0) s.n_list = 0u;
    __syncthreads();
    each4([&](int i, float4 q) {
      const float w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) over.add(w[e] > w_over ? w[e] : 0.f);
      note(i, w, w_in, w_over, kSmpList);
    });
    __syncthreads();
    const uint32_t m = s.n_list;
    auto take = [&](int i) {
      const uint32_t k = smp_key(smp_load(x + i));
      if (k <= floor_key) return 0u;
      in.add(sw[i]);
      lo = min(lo, k);
      hi = max(hi, k);
      return k;
    };
    if (m <= kSmpList) {
      for (uint32_t j = threadIdx.x; j < m; j += kSmpThreads) list[j] = take(s.at[j]);
    } else {
      for (int i = w0 + lane; i < w1; i += 32) {
        if (sw[i] > w_in && !(sw[i] > w_over)) take(i);
      }
    }
    above = over.get();
    inside = in.get();
    reduce(above, inside, lo, hi, cnt, nullptr);
  }

  // The mass of the listed logits above `key` (lists that did not run over).
  __device__ __forceinline__ void listed_above(uint32_t key, smp_u64& mass) {
    SmpSum sum;
    const uint32_t* list = s.own[turn ^ 1];
    for (uint32_t j = threadIdx.x; j < s.n_list; j += kSmpThreads)
      if (list[j] > key) sum.add(sw[s.at[j]]);
    smp_u64 none = 0;
    uint32_t lo = 0, hi = 0, cnt;
    mass = sum.get();
    reduce(mass, none, lo, hi, cnt, nullptr);
  }

  __device__ __forceinline__ float weight_of_key(uint32_t key) const { return weight_of(smp_unkey(key)); }
  __device__ __forceinline__ smp_u64 mass_of_key(uint32_t key) const { return smp_mass(weight_of_key(key)); }

  // The row's token from the elements in buckets up to `bk`, kSmpFew at most, of which the k largest and the rest of
  // the rules are taken: every block sends its own to block 0, and that one compares each with all.
  __device__ __forceinline__ void few(const SampleParams& p, int b, int i0, int bk, uint32_t top_k, float top_p,
                                      float min_p, float u) {
    const int tid = threadIdx.x;
    if (tid == 0) s.n_list = 0u;
    __syncthreads();
    const float w_in = smp_upper(bk + 1);
    each4([&](int i, float4 q) {
      const float w[4] = {q.x, q.y, q.z, q.w};
      note(i, w, w_in, 1.f, kSmpFew);
    });
    __syncthreads();
    const uint32_t own = s.n_list;
    if (tid == 0) s.pick = (int)atomicAdd(remote(&s.n_few, 0), own);
    __syncthreads();
    for (uint32_t j = tid; j < own; j += kSmpThreads) {
      const int i = s.at[j];
      remote(s.few_ord, 0)[s.pick + j] = (smp_u64)smp_key(smp_load(x + i)) << 32 | ~(uint32_t)(i0 + i);
    }
    sync();
    if (rank != 0) return;
    const int m = (int)s.n_few;
    smp_u64 ord = 0, mass = 0;
    float d = 0.f, w = 0.f;
    if (tid < m) {
      ord = s.few_ord[tid];
      d = smp_d(smp_unkey((uint32_t)(ord >> 32)), row);
      w = smp_exp(d);
      mass = smp_mass(w);
      s.few_mass[tid] = mass;
    }
    const uint32_t at = ~(uint32_t)ord;
    __syncthreads();
    // how many, and what mass, come before in the order (no branches: every load independent of the last)
    uint32_t place = 0;
    smp_u64 ahead = 0;
    if (warp * 32 < m) {
#pragma unroll 8
      for (int j = 0; j < m; ++j) {
        const bool first = s.few_ord[j] > ord;
        place += first;
        ahead += first ? s.few_mass[j] : 0ull;
      }
    }
    bool in = tid < m && place < top_k;
    auto total = [&](smp_u64 v) {  // over the block
      v = smp_warp_sum(v);
      if (lane == 0) s.red[warp][0] = v;
      __syncthreads();
      v = smp_warp_sum(lane < kSmpWarps ? s.red[lane][0] : 0ull);
      __syncthreads();
      return v;
    };
    const smp_u64 of_k = total(in ? mass : 0ull);
    if (top_p < 1.f) in = in && ahead < max((smp_u64)ceil((double)top_p * (double)of_k), 1ull);
    in = in && w >= min_p;
    const smp_u64 kept = total(in ? mass : 0ull);
    if (tid < m) s.few_mass[tid] = in ? mass : 0ull;
    __syncthreads();
    smp_u64 goal = (smp_u64)floor((double)fminf(fmaxf(u, 0.f), 1.f) * (double)kept);
    if (goal >= kept) goal = kept - 1;
    if (warp * 32 < m) {
      smp_u64 before = 0;  // by index
#pragma unroll 8
      for (int j = 0; j < m; ++j) before += (uint32_t)~(uint32_t)s.few_ord[j] < at ? s.few_mass[j] : 0ull;
      if (in && goal >= before && goal < before + mass) {
        p.token[b] = at;
        if (p.logprob != nullptr) p.logprob[b] = d - logf((float)((double)kept * kSmpUnit));
      }
    }
  }

  // Adds a count (of 1) or a mass to bin i of a histogram. Shared memory adds 32 bits natively and 64 only by trying
  // again, which hurts where many elements are of one bin; 15 bits of 2^16 elements fit 32.
  template <bool BY_MASS>
  __device__ __forceinline__ void add_to_bin(uint32_t* dig, uint32_t i, float w) const {
    if (BY_MASS) {
      const smp_u64 m = smp_mass(w);
      atomicAdd(&dig[i], (uint32_t)m & 0x7FFFu);
      atomicAdd(&dig[256 + i], (uint32_t)(m >> 15) & 0x7FFFu);
      atomicAdd(&dig[512 + i], (uint32_t)(m >> 30));
    } else {
      atomicAdd(&dig[i], 1u);
    }
  }

  // A bin's sum of the histogram dig[3][256].
  __device__ __forceinline__ static smp_u64 bin(const uint32_t* dig, int i) {
    return dig[i] + ((smp_u64)dig[256 + i] << 15) + ((smp_u64)dig[512 + i] << 30);
  }

  // Of 256 bins, in order: where the running sum of at(bin) reaches `need`, to s.pick and, less the sum before it,
  // s.pick_above. By warp 0.
  template <bool ASCENDING, typename F>
  __device__ __forceinline__ void pick_bin(F at, smp_u64 need) {
    smp_u64 v[8], sum = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = at(ASCENDING ? lane * 8 + e : 255 - (lane * 8 + e));
      sum += v[e];
    }
    smp_u64 before = smp_warp_scan(sum, lane) - sum;
    if (before < need && need <= before + sum) {
      int e = 0;
#pragma unroll
      for (int q = 0; q < 7; ++q)
        if (e == q && need > before + v[q]) {
          before += v[q];
          ++e;
        }
      s.pick = ASCENDING ? lane * 8 + e : 255 - (lane * 8 + e);
      s.pick_above = before;
    }
  }

  // Exact selection inside buckets b0 to b1, whose admitted logits span [lo, hi] and were listed by the last look()
  // (`cnt` of them): the key and the number of its ties such that the buckets' elements above the key, and those
  // ties, are the fewest whose count (BY_MASS: mass) reaches `need`.
  template <bool BY_MASS>
  __device__ __forceinline__ void refine(int b0, int b1, uint32_t lo, uint32_t hi, uint32_t cnt, smp_u64 need, uint32_t& key,
                                         smp_u64& ties) {
    if (lo == hi) {
      key = lo;
    } else if (cnt < kSmpAllLists) {
      select_listed<BY_MASS>(lo, hi, cnt, need, key);
    } else {
      select_digits<BY_MASS>(b0, b1, lo, hi, cnt != kSmpNoLists, need, key);
    }
    ties = need;
    if (BY_MASS) {
      const smp_u64 w = mass_of_key(key);
      ties = w == 0 ? 1ull : max((need + w - 1) / w, 1ull);
    }
  }

  // On a copy of all blocks' lists, in every block: 256 linear bins of the range of keys narrow it to one bin, until
  // few enough keys are left to compare each with all. `need` becomes what is still needed at the key.
  template <bool BY_MASS>
  __device__ __forceinline__ void select_listed(uint32_t lo, uint32_t hi, uint32_t cnt, smp_u64& need, uint32_t& key) {
    constexpr uint32_t kHalf = kSmpBuckets / 2;
    const uint32_t* cur = s.all;
    {  // the blocks' lists by a warp or more each, at once
      const smp_u64(*sent)[4] = s.xch[turn ^ 1];  // as the last reduce() left it
      const int r = warp % C;
      const smp_u64 ends = smp_warp_scan(lane < C ? sent[lane][3] : 0ull, lane);
      const uint32_t m = (uint32_t)sent[r][3], base = (uint32_t)__shfl_sync(0xffffffffu, ends, r) - m;
      const uint32_t* from = remote(s.own[turn ^ 1], r);
#pragma unroll 4
      for (uint32_t i = warp / C * 32 + lane; i < m; i += kSmpWarps / C * 32) s.all[base + i] = from[i];
    }
    uint32_t* dig = &s.dig[0][0][0];
    smp_u64* masses = reinterpret_cast<smp_u64*>(dig);
    for (int flip = 0;; flip ^= 1) {
      __syncthreads();
      if (lo == hi) {
        key = lo;
        return;
      }
      if (cnt <= kSmpCompare) {
        const uint32_t k = threadIdx.x < cnt ? cur[threadIdx.x] : 0u;
        const bool in = k >= lo && k <= hi;
        if (threadIdx.x < cnt) masses[threadIdx.x] = !in ? 0ull : BY_MASS ? mass_of_key(k) : 1ull;
        __syncthreads();
        if (warp * 32 < (int)cnt) {
          smp_u64 above = 0, equal = 0;
#pragma unroll 8
          for (uint32_t j = 0; j < cnt; ++j) {
            const uint32_t kj = cur[j];
            const smp_u64 m = masses[j];
            above += kj > k ? m : 0ull;
            equal += kj == k ? m : 0ull;
          }
          if (in && above < need && need <= above + equal) {  // (threads of equal keys write the same)
            s.pick = (int)k;
            s.pick_above = above;
          }
        }
        __syncthreads();
        key = (uint32_t)s.pick;
        need -= s.pick_above;
        __syncthreads();
        return;
      }
      const int shift = max(0, 24 - __clz(hi - lo));
      for (int i = threadIdx.x; i < 3 * 256; i += kSmpThreads) dig[i] = 0u;
      if (threadIdx.x == 0) {
        s.n_few = 0u;
        s.key_lo = 0xFFFFFFFFu;
        s.key_hi = 0u;
      }
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < cnt; i += kSmpThreads) {
        const uint32_t k = cur[i];
        if (k >= lo && k <= hi) add_to_bin<BY_MASS>(dig, (hi - k) >> shift, BY_MASS ? weight_of_key(k) : 0.f);
      }
      __syncthreads();
      if (warp == 0) pick_bin<true>([&](int i) { return bin(dig, i); }, need);
      __syncthreads();
      need -= s.pick_above;
      hi -= (uint32_t)s.pick << shift;
      if (hi - lo >= 1u << shift) lo = hi - ((1u << shift) - 1u);  // (the picked bin: something is in it)
      // the bin's keys to a list of their own, if they fit, and their range (of bf16 logits they are often alike)
      uint32_t* kept = s.own[turn] + flip * kHalf;
      uint32_t k0 = 0xFFFFFFFFu, k1 = 0u;
      for (uint32_t i = threadIdx.x; i < cnt; i += kSmpThreads) {
        const uint32_t k = cur[i];
        if (k >= lo && k <= hi) {
          const uint32_t at = atomicAdd(&s.n_few, 1u);
          if (at < kHalf) kept[at] = k;
          k0 = min(k0, k);
          k1 = max(k1, k);
        }
      }
      k0 = smp_warp_min(k0);
      k1 = smp_warp_max(k1);
      if (lane == 0 && k1 != 0u) {
        atomicMin(&s.key_lo, k0);
        atomicMax(&s.key_hi, k1);
      }
      __syncthreads();
      lo = s.key_lo;
      hi = s.key_hi;
      if (s.n_few <= kHalf) {
        cur = kept;
        cnt = s.n_few;
      }
    }
  }

  // Where the lists are too long for one block: 8-bit digits from the highest bit in which lo and hi differ, each
  // block over its own list (or, where a list ran over, over its part of the row: that sees the whole bucket, whose
  // order above a floor that look() was given is the same), with a cluster barrier each.
  template <bool BY_MASS>
  __device__ __forceinline__ void select_digits(int b0, int b1, uint32_t lo, uint32_t hi, bool listed, smp_u64& need,
                                                uint32_t& key) {
    const int top = 31 - __clz(lo ^ hi);
    uint32_t mask = top == 31 ? 0u : ~((2u << top) - 1u), prefix = hi & mask;
    const uint32_t* list = s.own[turn ^ 1];
    for (int shift = max(top - 7, 0);; shift = max(shift - 8, 0)) {
      uint32_t* dig = &s.dig[parity][0][0];
      parity ^= 1;
      for (int i = threadIdx.x; i < 3 * 256; i += kSmpThreads) dig[i] = 0u;
      __syncthreads();
      if (listed) {
        for (uint32_t i = threadIdx.x; i < s.n_list; i += kSmpThreads) {
          const uint32_t k = list[i];
          if (k != 0u && (k & mask) == prefix)
            add_to_bin<BY_MASS>(dig, (k >> shift) & 255u, BY_MASS ? weight_of_key(k) : 0.f);
        }
      } else {
        for (int i = w0 + lane; i < w1; i += 32) {
          const float w = sw[i];
          if (!(w > smp_upper(b1 + 1)) || w > smp_upper(b0)) continue;
          const uint32_t k = smp_key(smp_load(x + i));
          if ((k & mask) == prefix) add_to_bin<BY_MASS>(dig, (k >> shift) & 255u, w);
        }
      }
      sync();
      smp_u64* all = reinterpret_cast<smp_u64*>(s.all);
      if (threadIdx.x < 256) {  // over the cluster's blocks
        smp_u64 v = 0;
#pragma unroll 4
        for (int r = 0; r < C; ++r) v += bin(remote(dig, r), threadIdx.x);
        all[threadIdx.x] = v;
      }
      __syncthreads();
      if (warp == 0) pick_bin<false>([&](int i) { return all[i]; }, need);
      __syncthreads();
      const uint32_t dmask = 255u << shift;
      need -= s.pick_above;
      prefix = (prefix & ~dmask) | ((uint32_t)s.pick << shift);
      mask |= dmask;
      __syncthreads();
      if (shift == 0) break;
    }
    key = prefix;
  }
};

template <typename T>
__global__ void __launch_bounds__(kSmpThreads, 2) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t smp_dyn[];
  SmpShared& s = *reinterpret_cast<SmpShared*>(smp_dyn);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.y;
  const int i0 = min((int)blockIdx.x * p.chunk, p.V), n = min(p.chunk, p.V - i0);
  const int per = p.chunk / kSmpWarps;
  Smp<T> c{s,
                 static_cast<const T*>(p.logits) + (int64_t)b * p.row_stride + i0,
                 reinterpret_cast<float*>(smp_dyn + sizeof(SmpShared)),
                 (int)gridDim.x,
                 (int)blockIdx.x,
                 n,
                 min(warp * per, n),
                 min((warp + 1) * per, n),
                 lane,
                 warp,
                 {},
                 0,
                 0};
  if (c.C > 1) cluster_arrive();
  griddep_wait();
  griddep_launch_dependents();

  for (int i = tid; i < kSmpBuckets; i += kSmpThreads) s.own[0][i] = s.own[1][i] = 0u;
  for (int i = tid; i < kSmpBuckets; i += kSmpThreads) s.all[i] = 0u;
  if (tid == 0) s.n_list = s.n_few = 0u;

  // ---- the largest logit; the range goes to shared memory as fp32 (a NaN as it is: it gets no weight below)
  float top = -INFINITY;
#pragma unroll 8
  for (int i = c.w0 + 4 * lane; i < c.w1; i += 128) {
    const float4 q = c.logits4(i);
    top = fmax3(fmax3(top, q.x, q.y), q.z, q.w);
    *reinterpret_cast<float4*>(c.sw + i) = q;
  }
  float t = p.temperature[b];
  const bool greedy = !(t > 0.f);
  if (greedy) t = 1.f;
  uint32_t top_k = p.top_k != nullptr && p.top_k[b] > 0 ? (uint32_t)p.top_k[b] : 0xFFFFFFFFu;
  if (greedy) top_k = 1u;
  const float top_p = p.top_p != nullptr && p.top_p[b] < 1.f ? fmaxf(p.top_p[b], 0.f) : 1.f;
  const float min_p = p.min_p != nullptr && p.min_p[b] > 0.f ? fminf(p.min_p[b], 1.f) : 0.f;
  const float uu = p.u[b];
  const bool by_k = top_k > 1u && top_k < (uint32_t)p.V, by_p = top_p < 1.f && top_k > 1u;

  uint32_t best = smp_key(smp_logit(top));
  {
    smp_u64 z0 = 0, z1 = 0;
    uint32_t lo = 0, cnt;
    __syncwarp();
    if (c.C > 1) cluster_wait();  // every block has started
    c.reduce(z0, z1, lo, best, cnt, nullptr);
  }
  c.row.set(smp_unkey(best), t);
  uint32_t thr = 0;      // kept: logits above key `thr` (0: below every finite one), and the first `ties` at it,
  smp_u64 ties = 0;      // of weight >= min_p
  smp_u64 my = 0, my_ties = 0, before[2] = {0, 0}, kept = 0;  // this warp's kept mass, without ties; lower blocks'

  if (c.row.xmax == -INFINITY || top_k == 1u) {
    // nothing to choose from, or the lowest index of the largest logit
    uint32_t first = 0xFFFFFFFFu, none = 0, cnt;
    if (top == c.row.xmax) {  // this thread has seen it: among the elements that it loaded
      for (int i = c.w0 + 4 * lane; i < c.w1 && first == 0xFFFFFFFFu; i += 128)
        for (int e = 3; e >= 0; --e)
          if (i + e < n && smp_load(c.x + i + e) == c.row.xmax) first = i0 + i + e;
    }
    c.reduce(my, my_ties, first, none, cnt, nullptr);
    if (c.rank == 0 && tid == 0) {
      p.token[b] = first;
      if (p.logprob != nullptr) p.logprob[b] = c.row.xmax == -INFINITY ? __uint_as_float(0x7FC00000u) : 0.f;
    }
    return;
  }

  // ---- weights, their mass, and the histograms
  const bool cut = by_k || by_p;
  {
    SmpSum sum;
    uint32_t far = 0;
    const float w_min = cut ? 0.f : min_p;
    auto take = [&](const float4 q) {
      const float w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) sum.add(w[e] >= w_min ? w[e] : 0.f);
      if (cut) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t k = smp_bucket(w[e]);
          if (k < kSmpBuckets - 1) {
            atomicAdd(&s.own[0][k], 1u);
          } else {
            far += w[e] > 0.f;  // the far tail shares the last bucket: counted apart
          }
        }
      }
    };
    if (c.row.plain) {  // logits become weights
      c.each4([&](int, float4& q) {
        const float2 a = smp_weights2(q.x, q.y, c.row), b = smp_weights2(q.z, q.w, c.row);
        q = make_float4(a.x, a.y, b.x, b.y);
      });
    } else {
      // The padding up to a four's end goes to zero with the range's last index, by the warp that holds that one: the
      // warps after it have no range (and would turn it a second time, while others read it).
      if (c.w0 < c.w1) {
#pragma unroll 1
        for (int i = c.w0 + lane; i < ((c.w1 + 3) & ~3); i += 32) c.sw[i] = c.weight_of(c.sw[i]);
      }
      __syncwarp();
    }
    c.each4([&](int, float4 q) { take(q); });
    my = sum.get();
    if (cut) {
      far = __reduce_add_sync(0xffffffffu, far);
      if (lane == 0 && far) atomicAdd(&s.own[0][kSmpBuckets - 1], far);
    }
  }
  bool listed = min_p == 0.f;
  float w_listed = 0.f;  // the lower end of the buckets that the last look() listed
  if (cut) {
    smp_u64 total = my, above = 0, inside = 0;
    uint32_t lo = 0, hi = 0, cnt;
    double above_n, in_n;
    __syncthreads();
    c.merge_to_owner();
    if (c.C > 1) {
      c.sync();
      c.merge_to_all();
    }
    c.reduce(total, inside, lo, hi, cnt, nullptr);
    if (by_k) {
      const int bk = c.template crossing<false>((double)top_k, 0, kSmpBuckets - 1, above_n, in_n);
      if ((uint32_t)above_n + s.tot[bk] <= kSmpFew) {  // (the same in every block)
        c.few(p, b, i0, bk, top_k, top_p, min_p, uu);
        return;
      }
      c.look(bk, bk, 0u, above, inside, lo, hi, cnt);
      w_listed = smp_upper(bk + 1);
      total = above + inside;
      if (hi != 0u) {
        const smp_u64 need = (smp_u64)top_k - (smp_u64)above_n;
        if (need >= s.tot[bk]) {  // the whole bucket, or fewer logits than k
          thr = lo - 1u;
        } else {
          c.template refine<false>(bk, bk, lo, hi, cnt, need, thr, ties);
          if (by_p) {
            inside = 0;
            if (lo != hi) {
              if (cnt != kSmpNoLists) c.listed_above(thr, inside); else c.look(bk, bk, thr, above, inside, lo, hi, cnt);
            }
            total = above + inside + ties * c.mass_of_key(thr);
          }
        }
      }
    }
    if (by_p) {
      const double goal = (double)top_p * (double)total;
      const smp_u64 need = max((smp_u64)ceil(goal), 1ull);
      const int bt = thr != 0u ? (int)smp_bucket(c.weight_of_key(thr)) : kSmpBuckets - 1;
      // exact: guess from what a look has found, until the mass above buckets b0 to b1 is short of `need` and the mass
      // with them is not. Two buckets where the guess is near the edge of one and the lists stay short.
      int first = 0, last = bt, b0, b1;
      double at = goal * kSmpUnit;
      for (;;) {
        b0 = b1 = c.template crossing<true>(at, first, last, above_n, in_n);
        const double unsure = 3e-4 * at;
        if (at - above_n < unsure) {
          if (b0 > first && s.tot[b0 - 1] + s.tot[b0] < kSmpAllLists) --b0;
        } else if (above_n + in_n - at < unsure) {
          if (b1 < last && s.tot[b1] + s.tot[b1 + 1] < kSmpAllLists) ++b1;
        }
        c.look(b0, b1, b1 == bt ? thr : 0u, above, inside, lo, hi, cnt);
        if (above >= need && b0 > first) {
          last = b0 - 1;
        } else if (above + inside < need && b1 < last) {
          first = b1 + 1;
        } else {
          break;
        }
        at = fmax(above_n + ((double)need - (double)above) * kSmpUnit, 1e-30);
      }
      w_listed = smp_upper(b1 + 1);
      if (above + inside < need) {
        // everything above the top-k threshold is in, and some of its ties
        const smp_u64 w = thr != 0u ? c.mass_of_key(thr) : 0ull, left = need - (above + inside);
        if (w != 0) ties = min(ties, (left + w - 1) / w);
        listed = false;  // the last look() left the ties out
      } else {
        c.template refine<true>(b0, b1, lo, hi, cnt, need - above, thr, ties);
      }
    }
  }

  // ---- the kept mass by warp and block
  const float w_thr = thr != 0u ? c.weight_of_key(thr) : 0.f;
  const int bt = thr != 0u ? (int)smp_bucket(w_thr) : kSmpBuckets;
  // what is kept: weights above w_lo, and as negative ones the ties
  float w_lo = 0.f;
  if (!cut) {
    if (min_p > 0.f) w_lo = __uint_as_float(__float_as_uint(min_p) - 1u);
  } else if (listed && s.n_list <= kSmpList) {
    // what the last look() found: s.red[w][0] is the mass that warp w has above the buckets it listed
    w_lo = w_listed;
    if (lane == 0) s.red[warp][1] = 0ull;
    __syncthreads();
    const uint32_t* list = s.own[c.turn ^ 1];
    for (uint32_t j = tid; j < s.n_list; j += kSmpThreads) {
      const int i = s.at[j];
      const float w = c.sw[i];
      if (list[j] > thr) {
        atomicAdd(&s.red[i / per][0], smp_mass(w));
      } else if (list[j] == thr && ties != 0) {
        atomicAdd(&s.red[i / per][1], 1ull);
        c.sw[i] = -w;
      } else {
        c.sw[i] = 0.f;
      }
    }
    __syncthreads();
    my = lane == 0 ? s.red[warp][0] : 0ull;
    my_ties = lane == 0 ? s.red[warp][1] : 0ull;
    __syncwarp();
  } else {
    const float w_over = smp_upper(bt), w_in = smp_upper(bt + 1);
    SmpSum sum;
    uint32_t nt = 0;
    c.each4([&](int i, float4& q) {
      float w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        bool in = w[e] >= min_p && w[e] > w_in, tie = false;
        if (in && !(w[e] > w_over)) {
          const uint32_t k = smp_key(smp_load(c.x + i + e));
          in = k > thr;
          tie = k == thr && ties != 0;
        }
        if (in) sum.add(w[e]);
        nt += tie;
        w[e] = in ? w[e] : tie ? -w[e] : 0.f;
      }
      q = make_float4(w[0], w[1], w[2], w[3]);
    });
    my = sum.get();
    my_ties = nt;
  }
  smp_u64 all_ties = my_ties;
  kept = my;
  {
    uint32_t lo = 0, hi = 0, cnt;
    c.reduce(kept, all_ties, lo, hi, cnt, before);
  }
  // s.red[w][0 .. 1] still holds the block's warps' masses and ties
  const smp_u64 w_tie = smp_mass(w_thr);
  auto with_ties = [&](smp_u64 m, smp_u64 nt) { return m + min(nt, ties) * w_tie; };
  kept = with_ties(kept, all_ties);
  // first index with running mass > u * kept; u of 1 or more takes the last kept token
  smp_u64 goal = (smp_u64)floor((double)fminf(fmaxf(uu, 0.f), 1.f) * (double)kept);
  if (goal >= kept) goal = kept - 1;
  {
    const smp_u64 wm = lane < kSmpWarps ? s.red[lane][0] : 0ull, wt = lane < kSmpWarps ? s.red[lane][1] : 0ull;
    const smp_u64 em = before[0] + smp_warp_scan(wm, lane), et = before[1] + smp_warp_scan(wt, lane);
    const smp_u64 m0 = __shfl_sync(0xffffffffu, em - wm, warp), t0 = __shfl_sync(0xffffffffu, et - wt, warp);
    const smp_u64 m1 = __shfl_sync(0xffffffffu, em, warp), t1 = __shfl_sync(0xffffffffu, et, warp);
    if (goal >= with_ties(m0, t0) && goal < with_ties(m1, t1)) {
      // this warp holds the token: steps of 512 indices to the one that passes the goal, of 128, and its lanes' four
      smp_u64 fm = m0, ft = t0;
      auto step = [&](int i, SmpSum& sum, uint32_t& nt) {
        if (i >= c.w1) return;
        const float4 q = *reinterpret_cast<const float4*>(c.sw + i);
        const float w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sum.add(w[e] > w_lo ? w[e] : 0.f);
          nt += w[e] < 0.f;
        }
      };
      int base = c.w0;
      for (; base < c.w1; base += 512) {
        SmpSum sum;
        uint32_t nt = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) step(base + 128 * e + 4 * lane, sum, nt);
        const smp_u64 bm = fm + smp_warp_sum(sum.get()), bt = ft + __reduce_add_sync(0xffffffffu, nt);
        if (with_ties(bm, bt) > goal) break;
        fm = bm;
        ft = bt;
      }
      for (; base < c.w1; base += 128) {
        SmpSum sum;
        uint32_t nt = 0;
        const int i = base + 4 * lane;
        step(i, sum, nt);
        const smp_u64 im = fm + smp_warp_scan(sum.get(), lane), it = ft + smp_warp_scan(nt, lane);
        const uint32_t hit = __ballot_sync(0xffffffffu, with_ties(im, it) > goal);
        if (hit) {
          if (lane == __ffs(hit) - 1) {
            smp_u64 m = im - sum.get(), t = it - nt;
            for (int e = 0; e < 4; ++e) {
              const float w = c.sw[i + e];
              if (w > w_lo) m += smp_mass(w);
              t += w < 0.f;
              if (with_ties(m, t) > goal) {
                p.token[b] = i0 + i + e;
                if (p.logprob != nullptr)
                  p.logprob[b] = smp_d(smp_load(c.x + i + e), c.row) - logf((float)((double)kept * kSmpUnit));
                break;
              }
            }
          }
          break;
        }
        fm = __shfl_sync(0xffffffffu, im, 31);
        ft = __shfl_sync(0xffffffffu, it, 31);
      }
    }
  }
}

}  // namespace tg

// Sampling of the next token: temperature, top-k, top-p and min-p from a given
// uniform number per row.
//
//   d_i = x_i / T - x_max / T, w_i = exp(d_i)             (fp32; NaN logits count as -inf)
//   order the row by (x descending, index ascending);
//   keep its first k, then the shortest prefix whose mass reaches p times the
//   mass of those k, then of these every w_i >= min_p (w = 1 is the largest);
//   token = the first index, in index order, at which the running kept mass
//   passes u times the kept mass; logprob = d_token - log(kept mass).
// T <= 0 (or NaN) is greedy. Masses are sums of rint(w * 2^44) in 64-bit
// integers: exact, so the token depends on no order of summing and every
// block of a cluster takes the same decision (V <= 2^19 keeps them in range).
//
// A cluster of C blocks takes a row, each an index range of it, copied to its
// shared memory where it fits. No sort: the k-th value (or the value at which
// the mass reaches p) is found
//   1. by a histogram over 2048 linear buckets of d, 1/64 wide (linear in the
//      logit, so that logits spread over many buckets and shared-memory atomics
//      seldom collide), counts for k and exp(d + bucket / 64) in fixed point
//      for p, the latter only as a guess;
//   2. exactly inside that bucket: the bucket's mass above and inside, and its
//      smallest and largest key, in one pass (a wrong guess moves by a bucket);
//      then 8-bit digits of the ordered key from the highest bit in which the
//      two differ (none for bf16 logits, whose buckets hold one value).
// The threshold is a key and a number of its ties, which go by index.
#pragma once

#include <cooperative_groups.h>

#include "ptx.cuh"

namespace tg {

constexpr int kSmpThreads = 1024;
constexpr int kSmpWarps = kSmpThreads / 32;
constexpr int kSmpBuckets = 2048;
constexpr int kSmpMaxCluster = 8;
constexpr int kSmpMaxV = 1 << 19;
constexpr float kSmpMassOne = 17592186044416.f;  // 2^44

struct SampleParams {
  const void* logits;
  int64_t row_stride;  // elements
  int V, chunk;        // indices per block, a multiple of 128 (the last blocks may hold fewer or none)
  int in_smem;         // the block's range is copied to shared memory
  const float* u;
  const float* temperature;
  const int32_t* top_k;   // nullable
  const float* top_p;     // nullable
  const float* min_p;     // nullable
  int64_t* token;
  float* logprob;         // nullable
};

struct SmpShared {
  uint32_t cnt[kSmpBuckets];   // this block's histogram, then its slice's totals
  uint32_t mass[kSmpBuckets];
  uint32_t tot_cnt[kSmpBuckets];  // the row's histogram, written by every block of the cluster
  float tot_mass[kSmpBuckets];
  unsigned long long dig[2][256];  // digit histograms of a refinement, by pass parity
  unsigned long long xch[8];       // what the other blocks read of this one
  unsigned long long red[kSmpWarps][4];
  float redf[kSmpWarps];
  double scan[kSmpWarps];
  int pick;
  unsigned long long pick_above;
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

__device__ __forceinline__ float smp_d(float x, float xmax, float zmax, float t) {
  if (x == xmax) return 0.f;
  const float d = __fsub_rn(__fdiv_rn(x, t), zmax);
  return d <= 0.f ? d : -INFINITY;  // NaN: both quotients overflowed
}
__device__ __forceinline__ unsigned long long smp_mass(float w) { return (unsigned long long)rintf(w * kSmpMassOne); }
__device__ __forceinline__ int smp_bucket(float d) { return min((int)(-d * 64.f), kSmpBuckets - 1); }

template <typename V>
__device__ __forceinline__ V smp_warp_sum(V v) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
__device__ __forceinline__ uint32_t smp_warp_max(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ uint32_t smp_warp_min(uint32_t v) { return __reduce_min_sync(0xffffffffu, v); }

// The row-wide facts every thread carries.
struct SmpRow {
  float xmax, zmax, t;
};

// The block's elements through `f(local index, logit)`.
template <typename T, typename F>
__device__ __forceinline__ void smp_each(const T* x, int n, F f) {
  for (int i = threadIdx.x; i < n; i += kSmpThreads) f(i, smp_load(x + i));
}

// Exact selection inside bucket `bk`: finds the key T and the number r of its
// ties to take so that the elements of the bucket above T, and r at T, are the
// fewest whose count (BY_MASS: mass) reaches `need`. Returns also the mass and
// the count above T inside the bucket.
template <bool BY_MASS, typename T>
__device__ void smp_refine(SmpShared& s, cooperative_groups::cluster_group cl, int C, const T* x, int n,
                           const SmpRow& row, int bk, uint32_t lo_key, uint32_t hi_key, unsigned long long need,
                           int& parity, uint32_t& key_out, unsigned long long& ties_out) {
  // every key of the bucket lies in [lo_key, hi_key]
  uint32_t prefix = 0, mask = 0;
  if (lo_key == hi_key) {
    prefix = lo_key;
  } else {
    const int top = 31 - __clz(lo_key ^ hi_key);
    mask = top == 31 ? 0u : ~((2u << top) - 1u);
    prefix = hi_key & mask;
    for (int shift = max(top - 7, 0);; shift = max(shift - 8, 0)) {
      unsigned long long* dig = s.dig[parity];
      for (int i = threadIdx.x; i < 256; i += kSmpThreads) dig[i] = 0ull;
      __syncthreads();
      smp_each(x, n, [&](int, float v) {
        const uint32_t k = smp_key(v);
        if ((k & mask) != prefix || v == -INFINITY) return;
        const float d = smp_d(v, row.xmax, row.zmax, row.t);
        if (smp_bucket(d) != bk) return;
        atomicAdd(&dig[(k >> shift) & 255u], BY_MASS ? smp_mass(expf(d)) : 1ull);
      });
      if (C > 1) cl.sync(); else __syncthreads();
      // the cluster's digit totals in dig order, from the highest digit down, by warp 0 of every block
      if (threadIdx.x < 32) {
        unsigned long long v[8], sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int dgt = 255 - (threadIdx.x * 8 + e);
          v[e] = 0;
          for (int c = 0; c < C; ++c) v[e] += C > 1 ? cl.map_shared_rank(dig, c)[dgt] : dig[dgt];
          sum += v[e];
        }
        unsigned long long before = sum;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const unsigned long long a = __shfl_up_sync(0xffffffffu, before, off);
          if ((int)threadIdx.x >= off) before += a;
        }
        before -= sum;
        if (before < need && need <= before + sum) {
          int e = 0;
          while (need > before + v[e]) before += v[e++];
          s.pick = 255 - (threadIdx.x * 8 + e);
          s.pick_above = before;
        }
      }
      __syncthreads();
      const uint32_t dmask = shift + 8 >= 32 ? ~0u << shift : (255u << shift);
      need -= s.pick_above;
      prefix = (prefix & ~dmask) | ((uint32_t)s.pick << shift);
      mask |= dmask;
      parity ^= 1;
      __syncthreads();
      if (shift == 0) break;
    }
  }
  key_out = prefix;
  if (BY_MASS) {
    const unsigned long long w = smp_mass(expf(smp_d(smp_unkey(prefix), row.xmax, row.zmax, row.t)));
    ties_out = w == 0 ? 1ull : (need + w - 1) / w;
    if (ties_out == 0) ties_out = 1;
  } else {
    ties_out = need;
  }
}

template <typename T>
__global__ void __launch_bounds__(kSmpThreads, 1) sample_kernel(const SampleParams p) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint8_t smp_dyn[];
  SmpShared& s = *reinterpret_cast<SmpShared*>(smp_dyn);
  T* held = reinterpret_cast<T*>(smp_dyn + sizeof(SmpShared));
  cg::cluster_group cl = cg::this_cluster();
  const int C = gridDim.x, rank = blockIdx.x, b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int i0 = min(rank * p.chunk, p.V), n = min(p.chunk, p.V - i0);
  const T* x = static_cast<const T*>(p.logits) + (int64_t)b * p.row_stride + i0;
  auto sync_all = [&]() {
    if (C > 1) cl.sync(); else __syncthreads();
  };
  griddep_wait();
  griddep_launch_dependents();

  float t = p.temperature[b];
  const bool greedy = !(t > 0.f);
  if (greedy) t = 1.f;
  uint32_t top_k = p.top_k != nullptr && p.top_k[b] > 0 ? (uint32_t)p.top_k[b] : 0xFFFFFFFFu;
  if (greedy) top_k = 1u;
  const float top_p = p.top_p != nullptr && p.top_p[b] < 1.f ? fmaxf(p.top_p[b], 0.f) : 1.f;
  const float min_p = p.min_p != nullptr && p.min_p[b] > 0.f ? fminf(p.min_p[b], 1.f) : 0.f;

  // ---- the largest logit
  uint32_t best = 0;
  for (int i = tid; i < n; i += kSmpThreads) {
    const T v = x[i];
    if (p.in_smem) held[i] = v;
    best = max(best, smp_key(smp_load(&v)));
  }
  if (p.in_smem) x = held;
  best = smp_warp_max(best);
  if (lane == 0) s.red[warp][0] = best;
  __syncthreads();
  if (warp == 0) {
    best = smp_warp_max((uint32_t)s.red[lane][0]);
    if (lane == 0) s.xch[0] = best;
  }
  sync_all();
  for (int c = 0; c < C; ++c) best = max(c ? best : 0u, (uint32_t)(C > 1 ? *cl.map_shared_rank(&s.xch[0], c) : s.xch[0]));
  SmpRow row;
  row.xmax = smp_unkey(best);
  row.t = t;
  row.zmax = __fdiv_rn(row.xmax, t);
  if (row.xmax == -INFINITY) {  // nothing to choose from (the same in every block of the cluster)
    if (rank == 0 && tid == 0) {
      p.token[b] = 0;
      if (p.logprob != nullptr) p.logprob[b] = __uint_as_float(0x7FC00000u);
    }
    sync_all();
    return;
  }

  // ---- the threshold: keys above `thr`, and the first `ties` at it
  uint32_t thr = 0;  // key 0 is below every finite logit's
  unsigned long long ties = 0;
  const bool by_k = top_k > 1u && top_k < (uint32_t)p.V, by_p = top_p < 1.f && top_k > 1u;
  if (top_k == 1u) {  // greedy, or a prefix of one: the lowest index of the largest value
    thr = best;
    ties = 1;
  }
  if (by_k || by_p) {
    for (int i = tid; i < kSmpBuckets; i += kSmpThreads) s.cnt[i] = s.mass[i] = 0u;
    __syncthreads();
    unsigned long long all = 0;  // exact mass, per thread
    uint32_t far_n = 0;          // the last bucket gathers the far tail: counted apart
    smp_each(x, n, [&](int, float v) {
      if (v == -INFINITY) return;
      const float d = smp_d(v, row.xmax, row.zmax, row.t);
      const int bk = smp_bucket(d);
      if (by_p) all += smp_mass(expf(d));
      if (bk == kSmpBuckets - 1) {
        ++far_n;
        return;
      }
      atomicAdd(&s.cnt[bk], 1u);
      if (by_p) atomicAdd(&s.mass[bk], (uint32_t)rintf(expf(fmaf((float)bk, 1.f / 64.f, d)) * 4096.f));
    });
    far_n = __reduce_add_sync(0xffffffffu, far_n);
    if (lane == 0 && far_n) atomicAdd(&s.cnt[kSmpBuckets - 1], far_n);
    all = smp_warp_sum(all);
    if (lane == 0) s.red[warp][0] = all;
    __syncthreads();
    if (warp == 0) {
      all = smp_warp_sum(s.red[lane][0]);
      if (lane == 0) s.xch[1] = all;
    }
    sync_all();
    // totals: each block sums its slice of the buckets and hands it to all
    const int slice = kSmpBuckets / C;
    for (int i = rank * slice + tid; i < (rank + 1) * slice; i += kSmpThreads) {
      uint32_t a = 0;
      float m = 0.f;
      for (int c = 0; c < C; ++c) {
        a += C > 1 ? cl.map_shared_rank(s.cnt, c)[i] : s.cnt[i];
        m += (float)(C > 1 ? cl.map_shared_rank(s.mass, c)[i] : s.mass[i]);
      }
      m *= expf((float)i * (-1.f / 64.f)) * (1.f / 4096.f);
      for (int c = 0; c < C; ++c) {
        (C > 1 ? cl.map_shared_rank(s.tot_cnt, c) : s.tot_cnt)[i] = a;
        (C > 1 ? cl.map_shared_rank(s.tot_mass, c) : s.tot_mass)[i] = m;
      }
    }
    unsigned long long total = 0;
    for (int c = 0; c < C; ++c) total += C > 1 ? *cl.map_shared_rank(&s.xch[1], c) : s.xch[1];
    sync_all();
    int parity = 0;

    // first bucket at which the running count / mass reaches `target`
    auto crossing = [&](bool by_mass, double target, double& above) {
      const double a0 = by_mass ? (double)s.tot_mass[2 * tid] : (double)s.tot_cnt[2 * tid];
      const double a1 = by_mass ? (double)s.tot_mass[2 * tid + 1] : (double)s.tot_cnt[2 * tid + 1];
      double run = a0 + a1;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const double a = __shfl_up_sync(0xffffffffu, run, off);
        if (lane >= off) run += a;
      }
      if (lane == 31) s.scan[warp] = run;
      if (tid == 0) s.pick = kSmpBuckets - 1;
      __syncthreads();
      double before = run - a0 - a1;
      for (int w = 0; w < warp; ++w) before += s.scan[w];
      if (before + a0 >= target && a0 > 0.) atomicMin(&s.pick, 2 * tid);
      else if (before + a0 + a1 >= target && a1 > 0.) atomicMin(&s.pick, 2 * tid + 1);
      __syncthreads();
      const int bk = s.pick;
      if (2 * tid == bk || 2 * tid + 1 == bk) s.scan[0] = bk == 2 * tid ? before : before + a0;
      __syncthreads();
      above = s.scan[0];
      __syncthreads();
      return bk;
    };
    // of the elements that the threshold so far admits: mass above bucket bk, mass in it, its keys' range
    auto look = [&](int bk, bool limited, uint32_t tk, unsigned long long& above, unsigned long long& inside,
                    uint32_t& lo, uint32_t& hi) {
      unsigned long long a = 0, m = 0;
      uint32_t kl = 0xFFFFFFFFu, kh = 0;
      smp_each(x, n, [&](int, float v) {
        if (v == -INFINITY) return;
        const uint32_t k = smp_key(v);
        if (limited && k <= tk) return;
        const float d = smp_d(v, row.xmax, row.zmax, row.t);
        const int e = smp_bucket(d);
        if (e > bk) return;
        const unsigned long long w = smp_mass(expf(d));
        if (e < bk) {
          a += w;
        } else {
          m += w;
          kl = min(kl, k);
          kh = max(kh, k);
        }
      });
      a = smp_warp_sum(a);
      m = smp_warp_sum(m);
      kl = smp_warp_min(kl);
      kh = smp_warp_max(kh);
      if (lane == 0) {
        s.red[warp][0] = a;
        s.red[warp][1] = m;
        s.red[warp][2] = kl;
        s.red[warp][3] = kh;
      }
      __syncthreads();
      // xch[2..5] are rewritten by a later look only after another cluster barrier (parity)
      unsigned long long* xo = &s.xch[2];
      if (warp == 0) {
        a = smp_warp_sum(s.red[lane][0]);
        m = smp_warp_sum(s.red[lane][1]);
        kl = smp_warp_min((uint32_t)s.red[lane][2]);
        kh = smp_warp_max((uint32_t)s.red[lane][3]);
        if (lane == 0) {
          xo[0] = a;
          xo[1] = m;
          xo[2] = kl;
          xo[3] = kh;
        }
      }
      sync_all();
      above = inside = 0;
      lo = 0xFFFFFFFFu;
      hi = 0;
      for (int c = 0; c < C; ++c) {
        const unsigned long long* o = C > 1 ? cl.map_shared_rank(xo, c) : xo;
        above += o[0];
        inside += o[1];
        lo = min(lo, (uint32_t)o[2]);
        hi = max(hi, (uint32_t)o[3]);
      }
      sync_all();  // before anyone writes xch again
    };

    unsigned long long kept = total;  // mass of the top-k set
    double above_n;
    if (by_k) {
      const int bk = crossing(false, (double)top_k, above_n);
      unsigned long long above, inside;
      uint32_t lo, hi;
      look(bk, false, 0u, above, inside, lo, hi);
      if (hi != 0u) {
        const uint32_t in_bucket = s.tot_cnt[bk];
        const unsigned long long need = (unsigned long long)top_k - (unsigned long long)above_n;
        if (need >= in_bucket) {  // the whole bucket (or fewer finite logits than k)
          thr = lo - 1u;
          ties = 0;
          kept = above + inside;
        } else {
          smp_refine<false>(s, cl, C, x, n, row, bk, lo, hi, need, parity, thr, ties);
          if (by_p) {
            unsigned long long a2, m2;
            uint32_t l2, h2;
            look(bk, true, thr, a2, m2, l2, h2);
            kept = a2 + m2 + ties * smp_mass(expf(smp_d(smp_unkey(thr), row.xmax, row.zmax, row.t)));
          }
        }
      }
    }
    if (by_p) {
      const double goal = (double)top_p * (double)kept;
      unsigned long long need = (unsigned long long)ceil(goal);
      if (need < 1) need = 1;
      int bp = crossing(true, goal * (1.0 / (double)kSmpMassOne), above_n);
      // exact: move the guess until the mass above bucket bp is short of `need` and the mass with it is not
      unsigned long long above = 0, inside = 0;
      uint32_t lo, hi;
      bool beyond = false;  // the boundary lies among the top-k threshold's own ties
      for (;;) {
        look(bp, by_k && thr != 0u, thr, above, inside, lo, hi);
        if (above >= need && bp > 0) {
          do --bp; while (bp > 0 && s.tot_cnt[bp] == 0u);
        } else if (above + inside < need && bp < kSmpBuckets - 1) {
          int nb = bp + 1;
          while (nb < kSmpBuckets && s.tot_cnt[nb] == 0u) ++nb;
          if (nb == kSmpBuckets) {
            beyond = true;
            break;
          }
          bp = nb;
        } else {
          beyond = above + inside < need;
          break;
        }
      }
      if (beyond) {
        // everything above the top-k threshold is in; some of its ties are still needed
        if (by_k && thr != 0u && ties > 0) {
          const unsigned long long w = smp_mass(expf(smp_d(smp_unkey(thr), row.xmax, row.zmax, row.t)));
          const unsigned long long left = need - (above + inside);
          const unsigned long long r = w == 0 ? ties : (left + w - 1) / w;
          ties = r < ties ? r : ties;
        }
      } else {
        // the digit passes see the whole bucket; above the top-k threshold the order is the same
        smp_refine<true>(s, cl, C, x, n, row, bp, lo, hi, need - above, parity, thr, ties);
      }
    }
  }

  // ---- the kept mass, by 128-index pieces, then the token
  auto admitted = [&](float v, float& d, float& w) {  // 0: no, 1: above the threshold, 2: a tie
    if (v == -INFINITY) return 0;
    const uint32_t k = smp_key(v);
    if (k < thr || (k == thr && ties == 0)) return 0;
    d = smp_d(v, row.xmax, row.zmax, row.t);
    w = expf(d);
    if (!(w >= min_p)) return 0;
    return k > thr ? 1 : 2;
  };
  unsigned long long mass = 0;
  uint32_t n_tie = 0;
  smp_each(x, n, [&](int, float v) {
    float d, w;
    const int a = admitted(v, d, w);
    if (a == 1) mass += smp_mass(w);
    if (a == 2) ++n_tie;
  });
  mass = smp_warp_sum(mass);
  n_tie = __reduce_add_sync(0xffffffffu, n_tie);
  if (lane == 0) {
    s.red[warp][0] = mass;
    s.red[warp][1] = n_tie;
  }
  __syncthreads();
  if (warp == 0) {
    mass = smp_warp_sum(s.red[lane][0]);
    const unsigned long long nt = smp_warp_sum(s.red[lane][1]);
    if (lane == 0) {
      s.xch[6] = mass;
      s.xch[7] = nt;
    }
  }
  sync_all();
  const unsigned long long w_tie =
      thr != 0u ? smp_mass(expf(smp_d(smp_unkey(thr), row.xmax, row.zmax, row.t))) : 0ull;
  unsigned long long kept = 0, before = 0, tie_before = 0, own = 0, tie_run = 0;
  for (int c = 0; c < C; ++c) {
    const unsigned long long* o = C > 1 ? cl.map_shared_rank(&s.xch[6], c) : &s.xch[6];
    const unsigned long long tk = o[1] < ties - tie_run ? o[1] : ties - tie_run;
    const unsigned long long here = o[0] + tk * w_tie;
    if (c == rank) {
      before = kept;
      tie_before = tie_run;
      own = here;
    }
    kept += here;
    tie_run += tk;
  }
  // first index with running mass > u * kept; u >= 1 (or its rounding) takes the last kept token
  const float uu = p.u[b];
  const double goal_f = (double)fminf(fmaxf(uu, 0.f), 1.f) * (double)kept;
  unsigned long long goal = (unsigned long long)floor(goal_f);
  if (goal >= kept) goal = kept - 1;
  if (kept > 0 && goal >= before && goal < before + own && warp == 0) {
    // warp 0 walks its block's range; `run` is the kept mass before the piece
    unsigned long long run = before, tr = tie_before;
    for (int base = 0; base < n; base += 32) {
      const int i = base + lane;
      float d = 0.f, w = 0.f;
      const int a = i < n ? admitted(smp_load(x + i), d, w) : 0;
      const uint32_t tm = __ballot_sync(0xffffffffu, a == 2);
      const unsigned long long tie_rank = tr + __popc(tm & ((1u << lane) - 1u));
      unsigned long long mine = a == 1 || (a == 2 && tie_rank < ties) ? smp_mass(w) : 0ull;
      unsigned long long inc = mine;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += y;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, run + inc > goal);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          p.token[b] = i0 + i;
          if (p.logprob != nullptr) p.logprob[b] = d - logf((float)((double)kept * (1.0 / (double)kSmpMassOne)));
        }
        break;
      }
      run += __shfl_sync(0xffffffffu, inc, 31);
      tr += __popc(tm);
    }
  }
  sync_all();  // no block leaves while another may read its shared memory
}

}  // namespace tg

// One token per row of logits: temperature, min-p, top-k, top-p, then an
// inverse-CDF draw with a given uniform number.
//
// Definition. The entries above -inf (NaN counts as masked) of a row, ordered
// by falling logit, then rising column; e_i = 2^((x_i - max) log2(e) / T).
// Every filter keeps a prefix of that order:
//   min-p  the entries with e_i >= min_p
//   top-k  the first k of them
//   top-p  the shortest prefix that holds top_p of their mass
// and the draw is the first kept column, in column order, whose running mass
// exceeds u * (kept mass). A prefix is a key threshold plus a number of ties:
// an entry is kept if its key is above the threshold's, or equal and among
// the first n_tie equal ones by column. Both cuts that depend on masses are
// decisions of the form "sum < target": a relative error e of the masses
// flips a row's token with a probability of up to (entries) * e, 2^17 * 2^-24
// in fp32, so masses are computed and summed in fp64, in a fixed order.
//
// A row is read by a cluster of 1..8 CTAs; warp w of the cluster owns the
// w-th contiguous segment of the row. Passes over the row:
//   1  its largest logit (and every thread's own);
//   2  where a filter keeps few entries (top-k up to 1024, min-p, or a top-p
//      cut near the top), the candidates above a threshold that is known to
//      hold the cut are collected (at most 2048), sorted in shared memory by
//      one CTA, cut, and drawn from there. The threshold of a top-k is an
//      order statistic of the threads' maxima; that of a top-p comes from the
//      masses of 16 bands of logits (each thread sums bands of its own in
//      shared memory: no atomics, a fixed order);
//   3  otherwise (deep cuts) the band that holds the cut is split again until
//      its entries fit the list; the kept mass is summed per segment, and the
//      segment of the draw is scanned.
// Rows that resist (thousands of equal logits at a cut, top-k beyond 1024)
// descend through 16 bands of keys per pass, exact for every input.
#pragma once

#include <cooperative_groups.h>

#include "fh_fused.cuh"

namespace fh {

constexpr int kSmpThreads = 512;
constexpr int kSmpWarps = kSmpThreads / 32;
constexpr int kSmpBands = 16;
constexpr int kSmpMaxCluster = 8;
constexpr int kSmpList = 2048;   // candidates one CTA sorts
constexpr int kSmpMaxK = 1024;   // largest top-k that goes through the list
constexpr int kSmpCache = 8;     // vectors of a row that a thread keeps (CACHED)

struct SampleArgs {
  const void *logits;
  int n;
  long long stride;  // elements between rows
  // per row, or null: the scalar
  const float *temperature;
  const int32_t *top_k;
  const float *top_p;
  const float *min_p;
  float temperature0, top_p0, min_p0;
  int32_t top_k0;
  const double *uniforms;
  const int32_t *ids;  // column -> id, or null
  long long ids_stride;
  int64_t *out;
  float *prob;  // or null
};

struct __align__(16) SmpShared {
  union {
    struct {
      double mass[kSmpBands][kSmpThreads];
      uint32_t cnt[kSmpBands][kSmpThreads];
    } band;
    struct {
      unsigned long long item[kSmpList];   // key << 32 | ~column
      unsigned long long order[kSmpList];  // ~column << 32 | position in item
      double w[kSmpList];
    } list;
  };
  // values exchanged between the CTAs of a cluster, double-buffered so that
  // one cluster barrier per exchange is enough
  double x_mass[2][kSmpBands];
  unsigned long long x_cnt[2][kSmpBands];
  double sum_mass[kSmpBands];
  unsigned long long sum_cnt[kSmpBands];
  double seg_d[kSmpMaxCluster * kSmpWarps];
  int seg_i[kSmpMaxCluster * kSmpWarps];
  double warp_d[kSmpWarps];
  int warp_i[kSmpWarps];
  float warp_f[kSmpWarps];
  double scan_d[kSmpWarps];
  int scan_i[33];
  int count;  // list entries
  int best, last;
  unsigned long long cut_key;
  long long cut_ties;
};

// Order of the logits: monotone in x, with -0 equal to +0.
__device__ __forceinline__ uint32_t smp_key(float x) { return mono(x + 0.0f); }

template <typename E>
struct SmpElem;
template <>
struct SmpElem<float> {
  static constexpr int kVec = 4;
  __device__ __forceinline__ static float to_float(float v) { return v; }
  __device__ __forceinline__ static float none() { return -INFINITY; }
  __device__ __forceinline__ static void unpack(const uint4 &v, float *f) {
    f[0] = __uint_as_float(v.x);
    f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z);
    f[3] = __uint_as_float(v.w);
  }
};
template <>
struct SmpElem<__nv_bfloat16> {
  static constexpr int kVec = 8;
  __device__ __forceinline__ static float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
  __device__ __forceinline__ static __nv_bfloat16 none() { return __float2bfloat16(-INFINITY); }
  __device__ __forceinline__ static void unpack(const uint4 &v, float *f) {
    Vec<__nv_bfloat16>::to_float(v, f);
  }
};
template <>
struct SmpElem<__half> {
  static constexpr int kVec = 8;
  __device__ __forceinline__ static float to_float(__half v) { return __half2float(v); }
  __device__ __forceinline__ static __half none() { return __float2half(-INFINITY); }
  __device__ __forceinline__ static void unpack(const uint4 &v, float *f) {
    Vec<__half>::to_float(v, f);
  }
};

// A row as 16-byte vectors of its aligned address range: vector v holds the
// columns v * kVec - mis .. + kVec - 1; columns outside the row read as -inf
// (only the first and last vector have such, and are read one by one).
template <typename E>
struct SmpRow {
  static constexpr int kVec = SmpElem<E>::kVec;
  const E *p;
  int n, mis, nv;
  __device__ __forceinline__ SmpRow(const E *row, int n_)
      : p(row), n(n_), mis((int)((reinterpret_cast<uintptr_t>(row) / sizeof(E)) % kVec)) {
    nv = n > 0 ? (n + mis + kVec - 1) / kVec : 0;
  }
  __device__ __forceinline__ int column(int v) const { return v * kVec - mis; }
  __device__ __forceinline__ uint4 raw(int v) const {
    const int c0 = column(v);
    if (c0 >= 0 && c0 + kVec <= n) return __ldg(reinterpret_cast<const uint4 *>(p + c0));
    union {
      uint4 u;
      E e[kVec];
    } x;
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      x.e[i] = c0 + i >= 0 && c0 + i < n ? p[c0 + i] : SmpElem<E>::none();
    return x.u;
  }
  // NaN is masked like -inf
  __device__ __forceinline__ static void unpack(const uint4 &u, float *f) {
    SmpElem<E>::unpack(u, f);
#pragma unroll
    for (int i = 0; i < kVec; ++i) f[i] = f[i] == f[i] ? f[i] : -INFINITY;
  }
};

// 2^t for -100 < t <= 0 (a relative error below 2e-14): t = n + f with n the
// nearest integer, 2^f by a polynomial of degree 9 through the Chebyshev nodes
// of [-1/2, 1/2], n added to the exponent.
__device__ __forceinline__ double smp_exp2(double t) {
  const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is n
  const double r = t + magic;
  const int n = __double2loint(r);
  const double f = t - (r - magic);
  double p = 1.02059053204931027e-07;
  p = fma(p, f, 1.32596452439290570e-06);
  p = fma(p, f, 1.52526729253468732e-05);
  p = fma(p, f, 1.54034337512549968e-04);
  p = fma(p, f, 1.33335582007937186e-03);
  p = fma(p, f, 9.61812919393430395e-03);
  p = fma(p, f, 5.55041086646516774e-02);
  p = fma(p, f, 2.40226506956403407e-01);
  p = fma(p, f, 6.93147180559946174e-01);
  p = fma(p, f, 1.00000000000001354e+00);
  return __hiloint2double(__double2hiint(p) + (n << 20), __double2loint(p));
}

// Mass of a logit relative to the row's largest, 2^((x - m) c). `depth` is
// (m - x) c in fp32: a monotone measure of how far down a logit is, which also
// drops masses below 2^-72, less than the rounding of their sum.
struct SmpMass {
  double md, c;
  float m, cf;
  __device__ __forceinline__ SmpMass(float m_, float T)
      : md((double)m_), c(1.4426950408889634 / (double)T), m(m_),
        cf(fminf((float)(2.0 * c), 3.402823466e38f)) {}
  // halved first: m - x may pass the largest fp32
  __device__ __forceinline__ float depth(float x) const { return fmaf(-0.5f, x, 0.5f * m) * cf; }
  __device__ __forceinline__ double at_depth(float x, float d) const {
    return d < 72.f ? smp_exp2(((double)x - md) * c) : 0.0;
  }
  __device__ __forceinline__ double operator()(float x) const {
    return at_depth(x, depth(x));
  }
};

// A prefix of the order: keys above `key`, and the first `ties` equal ones.
struct SmpCut {
  uint32_t key;
  long long ties;
};

template <typename E, bool CACHED>
struct SmpCtx {
  SmpRow<E> row;
  SmpShared &S;
  int rank, size;  // CTA in its cluster
  int v0, v1;      // this warp's segment
  int phase;       // exchanges so far
  int tid, warp, lane;
  uint4 *cache;    // this thread's share of the row in shared memory (CACHED)

  // The first pass: f(vector, kVec values) over this warp's segment, a lane
  // every 32 vectors; a CACHED row stays in shared memory.
  template <typename F>
  __device__ __forceinline__ void first(F f) {
    constexpr int kVec = SmpRow<E>::kVec;
    if constexpr (CACHED) {
#pragma unroll
      for (int i = 0; i < kSmpCache; ++i) {
        const int v = v0 + lane + 32 * i;
        if (v < v1) cache[kSmpThreads * i] = row.raw(v);
      }
      each(f);
    } else {
      int v = v0 + lane;
      for (; v + 96 < v1; v += 128) {
        uint4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = row.raw(v + 32 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x[kVec];
          row.unpack(u[i], x);
          f(v + 32 * i, x);
        }
      }
      for (; v < v1; v += 32) {
        float x[kVec];
        row.unpack(row.raw(v), x);
        f(v, x);
      }
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) {
    if constexpr (CACHED) {
      constexpr int kVec = SmpRow<E>::kVec;
#pragma unroll 1
      for (int i = 0, v = v0 + lane; v < v1; ++i, v += 32) {
        float x[kVec];
        row.unpack(cache[kSmpThreads * i], x);
        f(v, x);
      }
    } else {
      first(f);
    }
  }
};

// Sums x_*[phase & 1][0..n) over the cluster's CTAs, in rank order, into
// sum_*. Contains a cluster barrier and a block barrier.
template <typename Ctx>
__device__ __forceinline__ void smp_exchange(Ctx &C, int n) {
  namespace cg = cooperative_groups;
  cg::cluster_group cl = cg::this_cluster();
  const int b = C.phase & 1;
  ++C.phase;
  cl.sync();
  if (C.tid < n) {
    double d = 0.0;
    unsigned long long k = 0ull;
    for (int r = 0; r < C.size; ++r) {
      const SmpShared *R = cl.map_shared_rank(&C.S, r);
      d += R->x_mass[b][C.tid];
      k += R->x_cnt[b][C.tid];
    }
    C.S.sum_mass[C.tid] = d;
    C.S.sum_cnt[C.tid] = k;
  }
  __syncthreads();
}

// Exclusive prefix sum of one double per thread, in a fixed order.
__device__ __forceinline__ double smp_scan(SmpShared &S, double v, double *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double t = __shfl_up_sync(0xFFFFFFFFu, x, o);
    if (lane >= o) x += t;
  }
  __syncthreads();
  if (lane == 31) S.scan_d[warp] = x;
  __syncthreads();
  double before = 0.0, all = 0.0;
#pragma unroll
  for (int i = 0; i < kSmpWarps; ++i) {
    if (i == warp) before = all;
    all += S.scan_d[i];
  }
  *total = all;
  return before + (x - v);
}

// Sums the threads' bands: warp b band b, lane by lane, then over the cluster.
template <bool MASS, bool CNT, typename Ctx>
__device__ __forceinline__ void smp_band_sums(Ctx &C) {
  SmpShared &S = C.S;
  __syncthreads();
  double d = 0.0;
  unsigned long long k = 0ull;
  for (int i = C.lane; i < kSmpThreads; i += 32) {
    if (MASS) d += S.band.mass[C.warp][i];
    if (CNT) k += S.band.cnt[C.warp][i];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (MASS) d += __shfl_xor_sync(0xFFFFFFFFu, d, o);
    if (CNT) k += __shfl_xor_sync(0xFFFFFFFFu, k, o);
  }
  if (C.lane == 0) {
    S.x_mass[C.phase & 1][C.warp] = d;
    S.x_cnt[C.phase & 1][C.warp] = k;
  }
  smp_exchange(C, kSmpBands);
}

// Counts (and masses) of the entries in 16 bands of keys, [lo + (i << shift),
// ...) up to hi, into sum_cnt (sum_mass).
template <bool MASS, typename Ctx>
__device__ __forceinline__ void smp_key_bands(Ctx &C, const SmpMass &w, uint32_t lo, uint32_t hi,
                                              int shift) {
  SmpShared &S = C.S;
#pragma unroll
  for (int i = 0; i < kSmpBands; ++i) {
    if (MASS) S.band.mass[i][C.tid] = 0.0;
    S.band.cnt[i][C.tid] = 0u;
  }
  C.each([&](int, const float *f) {
#pragma unroll
    for (int i = 0; i < decltype(C.row)::kVec; ++i) {
      const uint32_t k = smp_key(f[i]);
      if (k >= lo && k <= hi) {
        const int b = (int)((k - lo) >> shift);
        S.band.cnt[b][C.tid] += 1u;
        if (MASS) S.band.mass[b][C.tid] += w(f[i]);
      }
    }
  });
  smp_band_sums<MASS, true>(C);
}

__device__ __forceinline__ int smp_shift(uint32_t lo, uint32_t hi) {
  const uint32_t span = hi - lo;
  const int bits = 32 - __clz(span);
  return bits > 4 ? bits - 4 : 0;
}

// First k entries: the key of the k-th largest and how many of its ties.
// Returns false (cut unchanged) when there are fewer than k keys in [lo, hi].
template <typename Ctx>
__device__ __forceinline__ bool smp_top_k(Ctx &C, const SmpMass &w, uint32_t lo, uint32_t hi,
                                          long long k, SmpCut &cut) {
  unsigned long long above = 0ull;
  for (int pass = 0; pass < 9; ++pass) {
    const int shift = smp_shift(lo, hi);
    smp_key_bands<false>(C, w, lo, hi, shift);
    int b = kSmpBands - 1;
    for (; b >= 0; --b) {
      if (above + C.S.sum_cnt[b] >= (unsigned long long)k) break;
      above += C.S.sum_cnt[b];
    }
    __syncthreads();
    if (b < 0) return false;
    const uint32_t nlo = lo + ((uint32_t)b << shift);
    if (shift == 0) {
      cut.key = nlo;
      cut.ties = k - (long long)above;
      return true;
    }
    hi = nlo + min(hi - nlo, (1u << shift) - 1u);
    lo = nlo;
  }
  return false;
}

// How many of `have` equal entries bring `need` of their mass (at least one;
// all of them where their mass is zero).
__device__ __forceinline__ long long smp_ties(double need, long long have) {
  const double n = ceil(need);
  return n >= (double)have || n != n ? have : n < 1.0 ? 1 : (long long)n;
}

// Shortest prefix of the base prefix with mass >= p * (its mass).
template <typename Ctx>
__device__ __forceinline__ void smp_top_p(Ctx &C, const SmpMass &w, const SmpCut &base,
                                          uint32_t key_max, double p, SmpCut &cut) {
  // the base's ties enter as one more band below its other keys
  const double tie_w = base.ties > 0 ? w(unmono(base.key)) : 0.0;
  double above = 0.0, target = 0.0;
  uint32_t lo = base.key + 1u, hi = key_max;
  if (lo > hi) {  // only ties of one key
    cut.key = base.key;
    cut.ties = smp_ties(p * (double)base.ties, base.ties);
    return;
  }
  for (int pass = 0; pass < 9; ++pass) {
    const int shift = smp_shift(lo, hi);
    smp_key_bands<true>(C, w, lo, hi, shift);
    const double *mass = C.S.sum_mass;
    const unsigned long long *cnt = C.S.sum_cnt;
    if (pass == 0) {
      double z = 0.0;
      for (int b = kSmpBands - 1; b >= 0; --b) z += mass[b];
      target = p * (z + (double)base.ties * tie_w);
    }
    int b = kSmpBands - 1, lowest = -1;
    double before = above;  // mass above the lowest non-empty band
    for (; b >= 0; --b) {
      if (cnt[b] == 0ull) continue;
      lowest = b;
      before = above;
      if (above + mass[b] >= target) break;
      above += mass[b];
    }
    if (b < 0 && pass == 0 && base.ties > 0) {  // down into the base's ties
      cut.key = base.key;
      cut.ties = smp_ties((target - above) / tie_w, base.ties);
      return;
    }
    if (b < 0) {  // rounding: the target is the whole band's mass
      b = lowest;
      above = before;
    }
    const long long have = (long long)cnt[b];
    __syncthreads();
    const uint32_t nlo = lo + ((uint32_t)b << shift);
    if (shift == 0) {
      cut.key = nlo;
      cut.ties = smp_ties((target - above) / w(unmono(nlo)), have);
      return;
    }
    hi = nlo + min(hi - nlo, (1u << shift) - 1u);
    lo = nlo;
  }
}

// Smallest key whose mass is at least min_p (at most the largest entry's).
__device__ __forceinline__ uint32_t smp_min_key(const SmpMass &w, float m, float min_p) {
  const uint32_t top = smp_key(m);
  const double t = log2((double)min_p);
  auto enough = [&](uint32_t k) { return ((double)unmono(k) - w.md) * w.c >= t; };
  // bisect the keys; the border's rounded value is nearly always within a step
  uint32_t lo = smp_key(-INFINITY), hi = top;  // lo: too little, hi: enough
  const uint32_t g = smp_key((float)fmin((double)m, w.md + t / w.c));
  if (g > lo + 2u && !enough(g - 2u)) lo = g - 2u;
  if (g + 2u < hi && enough(g + 2u)) hi = g + 2u;
  while (hi - lo > 1u) {
    const uint32_t mid = lo + (hi - lo) / 2u;
    if (enough(mid))
      hi = mid;
    else
      lo = mid;
  }
  return hi;
}

// The three nested band levels of a top-p descent, in units of depth (a
// factor 2 of mass): 2, 1/8 and 1/128 wide, the last of a level open-ended.
// Each is a monotone step function of the logit, so that a band is a run of
// the order whatever the rounding.
struct SmpBand {
  int level;      // levels already chosen
  int j0, j1, j2; // the chosen bands
  __device__ __forceinline__ static int clamp(float x) {
    return (int)fmaxf(0.f, fminf(x, (float)(kSmpBands - 1)));
  }
  __device__ __forceinline__ static int band0(float d) { return clamp(d * 0.5f); }
  __device__ __forceinline__ int band1(float d) const { return clamp((d - 2.f * j0) * 8.f); }
  __device__ __forceinline__ int band2(float d) const {
    return clamp((d - 2.f * j0 - 0.125f * j1) * 128.f);
  }
  // -1: before the chosen band, +1: behind it, 0: in it
  __device__ __forceinline__ int side(float d) const {
    int s = band0(d) - j0;
    if (s == 0 && level > 1) s = band1(d) - j1;
    if (s == 0 && level > 2) s = band2(d) - j2;
    return s;
  }
  __device__ __forceinline__ int next(float d) const {
    return level == 0 ? band0(d) : level == 1 ? band1(d) : band2(d);
  }
};

// Entries with in(x) into this CTA's list; returns the cluster's total, and
// gathers the lists in rank 0's when they fit. Contains cluster barriers.
template <typename Ctx, typename In>
__device__ __forceinline__ int smp_collect(Ctx &C, In in) {
  namespace cg = cooperative_groups;
  cg::cluster_group cl = cg::this_cluster();
  SmpShared &S = C.S;
  __syncthreads();
  if (C.tid == 0) S.count = 0;
  __syncthreads();
  C.each([&](int v, const float *f) {
    constexpr int kVec = decltype(C.row)::kVec;
    uint32_t hit = 0u;
#pragma unroll
    for (int i = 0; i < kVec; ++i) hit |= in(f[i]) ? 1u << i : 0u;
    if (hit) {
      int at = atomicAdd(&S.count, __popc(hit));
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        if ((hit >> i) & 1u) {
          if (at < kSmpList)
            S.list.item[at] = ((unsigned long long)smp_key(f[i]) << 32) |
                              (0xFFFFFFFFu - (uint32_t)(C.row.column(v) + i));
          ++at;
        }
    }
  });
  __syncthreads();
  if (C.tid == 0) S.x_cnt[C.phase & 1][0] = (unsigned long long)S.count;
  smp_exchange(C, 1);
  const unsigned long long total = S.sum_cnt[0];
  if (total > (unsigned long long)kSmpList) return kSmpList + 1;
  if (C.size > 1) {
    if (C.rank == 0) {
      int base = S.count;
      for (int r = 1; r < C.size; ++r) {
        const SmpShared *R = cl.map_shared_rank(&S, r);
        const int cnt = R->count;
        for (int i = C.tid; i < cnt; i += kSmpThreads) S.list.item[base + i] = R->list.item[i];
        base += cnt;
      }
    }
    cl.sync();  // the others' lists may go
  }
  __syncthreads();
  return (int)total;
}

// Descending bitonic sort of n2 (a power of two) words by the whole CTA.
__device__ __forceinline__ void smp_sort(unsigned long long *a, int n2) {
  for (int size = 2; size <= n2; size <<= 1) {
    for (int step = size >> 1; step > 0; step >>= 1) {
      __syncthreads();
      for (int t = threadIdx.x; t < n2 / 2; t += kSmpThreads) {
        const int i = 2 * t - (t & (step - 1)), j = i + step;
        const unsigned long long x = a[i], y = a[j];
        if ((x < y) == ((i & size) == 0)) {
          a[i] = y;
          a[j] = x;
        }
      }
    }
  }
  __syncthreads();
}

__device__ __forceinline__ int smp_pow2(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

// Sorts the list and leaves its masses in list.w. Returns this thread's
// exclusive prefix of the masses of items kPer * tid .. + kPer - 1.
constexpr int kSmpPer = kSmpList / kSmpThreads;
template <typename Ctx>
__device__ __forceinline__ double smp_sort_list(Ctx &C, const SmpMass &w, int n, double *wt,
                                                double *total) {
  SmpShared &S = C.S;
  const int n2 = smp_pow2(n);
  for (int i = n + C.tid; i < n2; i += kSmpThreads) S.list.item[i] = 0ull;
  smp_sort(S.list.item, n2);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kSmpPer; ++i) {
    const int at = C.tid * kSmpPer + i;
    wt[i] = at < n ? w(unmono((uint32_t)(S.list.item[at] >> 32))) : 0.0;
    if (at < n) S.list.w[at] = wt[i];
    sum += wt[i];
  }
  return smp_scan(S, sum, total);
}

template <typename E>
__device__ __forceinline__ void smp_emit(const SampleArgs &a, int r, int col, double prob) {
  a.out[r] = a.ids ? (int64_t)a.ids[(long long)r * a.ids_stride + col] : (int64_t)col;
  if (a.prob) a.prob[r] = (float)prob;
}

// The draw from the first `keep` items of the sorted list (rank 0's CTA).
template <typename E, typename Ctx>
__device__ __forceinline__ void smp_draw_list(Ctx &C, const SampleArgs &a, int r, int keep,
                                              double u) {
  SmpShared &S = C.S;
  if (keep == 1) {
    if (C.tid == 0) smp_emit<E>(a, r, (int)(0xFFFFFFFFu - (uint32_t)S.list.item[0]), 1.0);
    return;
  }
  const int n2 = smp_pow2(keep);
  for (int i = C.tid; i < n2; i += kSmpThreads)
    S.list.order[i] = i < keep ? (S.list.item[i] << 32) | (uint32_t)i : 0ull;
  if (C.tid == 0) {
    S.best = 0x7FFFFFFF;
    S.last = -1;
  }
  smp_sort(S.list.order, n2);  // rising columns
  double wt[kSmpPer], sum = 0.0, total;
#pragma unroll
  for (int i = 0; i < kSmpPer; ++i) {
    const int at = C.tid * kSmpPer + i;
    wt[i] = at < keep ? S.list.w[(uint32_t)S.list.order[at]] : 0.0;
    sum += wt[i];
  }
  double run = smp_scan(S, sum, &total);
  const double target = u * total;
#pragma unroll
  for (int i = 0; i < kSmpPer; ++i) {
    const int at = C.tid * kSmpPer + i;
    run += wt[i];
    if (wt[i] > 0.0) {
      if (run > target) atomicMin(&S.best, at);
      atomicMax(&S.last, at);
    }
  }
  __syncthreads();
  if (C.tid == 0) {
    // past the end by rounding: the last entry with a mass
    const unsigned long long o = S.list.order[S.best != 0x7FFFFFFF ? S.best : S.last];
    smp_emit<E>(a, r, (int)(0xFFFFFFFFu - (uint32_t)(o >> 32)), S.list.w[(uint32_t)o] / total);
  }
}

// The draw from the prefix `cut` of the whole row.
template <typename E, typename Ctx>
__device__ __forceinline__ void smp_draw_row(Ctx &C, const SampleArgs &a, const SmpMass &w,
                                             const SmpCut &cut, double tie_w, int r, double u) {
  namespace cg = cooperative_groups;
  cg::cluster_group cl = cg::this_cluster();
  constexpr int kVec = SmpRow<E>::kVec;
  SmpShared &S = C.S;
  const int tid = C.tid, warp = C.warp, lane = C.lane, size = C.size;
  const float xc = unmono(cut.key);
  double sum = 0.0;
  int ties = 0;
  C.each([&](int, const float *f) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      if (f[i] > xc) sum += w(f[i]);
      ties += f[i] == xc;
    }
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    ties += __shfl_xor_sync(0xFFFFFFFFu, ties, o);
  }
  if (lane == 0) {
    S.warp_d[warp] = sum;
    S.warp_i[warp] = ties;
  }
  if (tid == 0) {
    S.best = 0x7FFFFFFF;
    S.last = -1;
  }
  cl.sync();
  // every CTA finds the segment of the draw: thread i has segment i
  const int segs = size * kSmpWarps;
  double mass = 0.0;
  int seg_ties = 0;
  if (tid < segs) {
    const SmpShared *R = cl.map_shared_rank(&S, tid / kSmpWarps);
    mass = R->warp_d[tid % kSmpWarps];
    seg_ties = R->warp_i[tid % kSmpWarps];
  }
  int all_ties;
  const int ties_before = block_exclusive_scan(seg_ties, S.scan_i, &all_ties);
  const long long left = cut.ties - ties_before;
  if (left > 0) mass += (double)min(left, (long long)seg_ties) * tie_w;
  double total;
  const double before = smp_scan(S, mass, &total);
  const double target = u * total;
  if (mass > 0.0) {
    if (before + mass > target) atomicMin(&S.best, tid);
    atomicMax(&S.last, tid);
  }
  __syncthreads();
  const int seg = S.best != 0x7FFFFFFF ? S.best : S.last;
  if (tid == seg) {
    S.seg_d[0] = before;
    S.cut_ties = left;
  }
  __syncthreads();
  const double seg_before = S.seg_d[0];
  const long long seg_left = S.cut_ties;
  if (tid == 0) {
    S.best = 0x7FFFFFFF;
    S.last = -1;
  }
  __syncthreads();
  if (seg / kSmpWarps == C.rank) {
    const int sv0 = (int)((long long)C.row.nv * seg / segs);
    const int sv1 = (int)((long long)C.row.nv * (seg + 1) / segs);
    const int per = (sv1 - sv0 + kSmpThreads - 1) / kSmpThreads;
    const int a0 = min(sv1, sv0 + tid * per), a1 = min(sv1, a0 + per);
    int t = 0;
    if (cut.ties > 0) {
      for (int v = a0; v < a1; ++v) {
        float f[kVec];
        C.row.unpack(C.row.raw(v), f);
#pragma unroll
        for (int i = 0; i < kVec; ++i) t += f[i] == xc;
      }
    }
    int t_total;
    const int t_before = block_exclusive_scan(t, S.scan_i, &t_total);
    double d = 0.0;
    long long lft = seg_left - t_before;
    for (int v = a0; v < a1; ++v) {
      float f[kVec];
      C.row.unpack(C.row.raw(v), f);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        if (f[i] > xc)
          d += w(f[i]);
        else if (f[i] == xc && lft-- > 0)
          d += tie_w;
      }
    }
    double seg_total;
    double run = seg_before + smp_scan(S, d, &seg_total);
    lft = seg_left - t_before;
    int best = 0x7FFFFFFF, last = -1;
    for (int v = a0; v < a1; ++v) {
      float f[kVec];
      C.row.unpack(C.row.raw(v), f);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        double x = 0.0;
        if (f[i] > xc)
          x = w(f[i]);
        else if (f[i] == xc && lft-- > 0)
          x = tie_w;
        run += x;
        if (x > 0.0) {
          last = C.row.column(v) + i;
          if (run > target) best = min(best, last);
        }
      }
    }
    if (best != 0x7FFFFFFF) atomicMin(&S.best, best);
    if (last >= 0) atomicMax(&S.last, last);
    __syncthreads();
    if (tid == 0) {
      // past the end by rounding: the last kept column
      const int col = S.best != 0x7FFFFFFF ? S.best : S.last;
      const float x = SmpElem<E>::to_float(C.row.p[col]);
      smp_emit<E>(a, r, col, (x > xc ? w(x) : tie_w) / total);
    }
  }
}

// CACHED: every lane's share of the row is at most kSmpCache vectors, kept in
// shared memory.
template <typename E, bool CACHED>
__global__ void __launch_bounds__(kSmpThreads, CACHED ? 1 : 2) k_sample(SampleArgs a) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) unsigned char smp_raw[];
  SmpShared &S = *reinterpret_cast<SmpShared *>(smp_raw);
  cg::cluster_group cl = cg::this_cluster();
  constexpr int kVec = SmpRow<E>::kVec;
  const int size = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int r = blockIdx.x / size;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  SmpCtx<E, CACHED> C{SmpRow<E>(reinterpret_cast<const E *>(a.logits) + (long long)r * a.stride, a.n),
                      S, rank, size, 0, 0, 0, tid, warp, lane,
                      reinterpret_cast<uint4 *>(smp_raw + sizeof(SmpShared)) + tid};
  {
    const int gw = rank * kSmpWarps + warp, warps = size * kSmpWarps;
    C.v0 = (int)((long long)C.row.nv * gw / warps);
    C.v1 = (int)((long long)C.row.nv * (gw + 1) / warps);
  }
  float T = a.temperature ? a.temperature[r] : a.temperature0;
  const long long k = a.top_k ? a.top_k[r] : a.top_k0;
  const float p = a.top_p ? a.top_p[r] : a.top_p0;
  const float mp = a.min_p ? a.min_p[r] : a.min_p0;
  double u = a.uniforms[r];
  u = u > 0.0 ? u : 0.0;
  const bool greedy = !(T > 0.f);
  if (greedy) T = 1.f;

  // the thread's and the row's largest logit
  float mt = -INFINITY;
  C.first([&](int, const float *f) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) mt = fmaxf(mt, f[i]);
  });
  float m = mt;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  if (lane == 0) S.warp_f[warp] = m;
  cl.sync();
  m = -INFINITY;
  for (int i = lane; i < size * kSmpWarps; i += 32)
    m = fmaxf(m, cl.map_shared_rank(&S, i / kSmpWarps)->warp_f[i % kSmpWarps]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));

  const uint32_t key_none = smp_key(-INFINITY);
  if (m == -INFINITY) {  // nothing left in this row
    if (rank == 0 && tid == 0) {
      a.out[r] = -1;
      if (a.prob) a.prob[r] = 0.f;
    }
    cl.sync();
    return;
  }
  const SmpMass w(m, T);
  const uint32_t key_max = smp_key(m);
  const bool use_k = k > 0 && k < a.n, use_p = p < 1.f;
  SmpCut cut{key_none, 0};
  double tie_w = 1.0;
  bool drawn = false;
  if (greedy || k == 1 || p <= 0.f) {
    cut.key = key_max;
    cut.ties = 1;
  } else if (m == INFINITY) {
    // the +inf entries are equal and have all the mass: every filter counts
    int cnt = 0;
    C.each([&](int, const float *f) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) cnt += f[i] == INFINITY;
    });
    const int all = __reduce_add_sync(0xFFFFFFFFu, cnt);
    if (lane == 0) S.x_cnt[C.phase & 1][warp] = (unsigned long long)all;
    smp_exchange(C, kSmpBands);
    cut.key = key_max;
    for (int i = 0; i < kSmpWarps; ++i) cut.ties += (long long)S.sum_cnt[i];
    if (use_k) cut.ties = min(cut.ties, k);
    if (use_p) cut.ties = smp_ties((double)p * (double)cut.ties, cut.ties);
  } else {
    if (mp > 0.f) cut.key = smp_min_key(w, m, fminf(mp, 1.f)) - 1u;
    bool done = !use_k && !use_p && !(mp > 0.f);
    if (!done && ((use_k && k <= kSmpMaxK) || (!use_k && mp > 0.f))) {
      // candidates above a threshold that keeps the first k
      uint32_t thr = cut.key + 1u;
      if (use_k) {
        // about `want` entries of a row in random order lie above the
        // threads' rank-th largest maximum: a thread's maximum is above it
        // with probability 1 - exp(-want / threads)
        const float want = fminf(3.f * (float)k + 256.f, 1500.f);
        const int rank_t = max(1, (int)(kSmpThreads *
                                        (1.f - expf(-want / (float)(kSmpThreads * size)))));
        const uint32_t kt = smp_key(mt);
        uint32_t pre = 0u;
        for (int bit = 31; bit >= 12; --bit) {
          const uint32_t c = pre | (1u << bit);
          if (__syncthreads_count(kt >= c) >= rank_t) pre = c;
        }
        if (size > 1) {
          if (tid == 0) S.x_cnt[C.phase & 1][0] = pre;
          const int b = C.phase & 1;
          ++C.phase;
          cl.sync();
          for (int q = 0; q < size; ++q)
            pre = max(pre, (uint32_t)cl.map_shared_rank(&S, q)->x_cnt[b][0]);
        }
        thr = max(thr, pre);
      }
      const float xt = unmono(thr);
      const int got = smp_collect(C, [&](float x) { return x >= xt; });
      if (got <= kSmpList && (thr == cut.key + 1u || got >= k)) {
        if (rank == 0) {
          double wt[kSmpPer], z;
          double run = smp_sort_list(C, w, got, wt, &z);
          int keep = use_k ? (int)min(k, (long long)got) : got;
          if (use_p) {
            // mass of the first `keep`, then the prefix that reaches the target
            double part = 0.0;
#pragma unroll
            for (int i = 0; i < kSmpPer; ++i) part += tid * kSmpPer + i < keep ? wt[i] : 0.0;
            smp_scan(S, part, &z);
            const double target = (double)p * z;
            int in = 0;
#pragma unroll
            for (int i = 0; i < kSmpPer; ++i) {
              in += tid * kSmpPer + i < keep && run < target;
              run += wt[i];
            }
            int before, all;
            before = block_exclusive_scan(in, S.scan_i, &all);
            (void)before;
            keep = max(1, all);
          }
          smp_draw_list<E>(C, a, r, keep, u);
        }
        drawn = done = true;
      } else if (!use_k && !use_p) {
        done = true;  // min-p alone keeps a long prefix: its threshold is the cut
      }
    }
    if (!done && !use_k && use_p) {
      // top-p over the entries above cut.key: bands of logits
      const float xb = unmono(cut.key);
      SmpBand band{0, 0, 0, 0};
      double above = 0.0, target = 0.0;
      float width = 2.f, top = 0.f;  // of the bands of this level; depth of the first
      for (; band.level < 3 && !done;) {
#pragma unroll
        for (int i = 0; i < kSmpBands; ++i) S.band.mass[i][tid] = 0.0;
        C.each([&](int, const float *f) {
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            const float d = w.depth(f[i]);
            if (f[i] > xb && (band.level == 0 || band.side(d) == 0))
              S.band.mass[band.next(d)][tid] += w.at_depth(f[i], d);
          }
        });
        smp_band_sums<true, false>(C);
        if (band.level == 0) {
          double z = 0.0;
          for (int i = 0; i < kSmpBands; ++i) z += S.sum_mass[i];
          target = (double)p * z;
        }
        int j = 0;
        double head = 0.0;  // smallest number of entries that explains the masses before band j
        for (; j < kSmpBands - 1; ++j) {
          const double lo_cnt = S.sum_mass[j] * (double)exp2f(top + width * j);
          if (above + S.sum_mass[j] >= target) {
            // entries of the band at least: its mass / its largest mass
            if (band.level == 0 && head + lo_cnt <= kSmpList) head = -1.0;
            else head = lo_cnt;
            break;
          }
          head += lo_cnt;
          above += S.sum_mass[j];
        }
        __syncthreads();
        if (band.level == 0) band.j0 = j;
        else if (band.level == 1) band.j1 = j;
        else band.j2 = j;
        ++band.level;
        top += width * j;
        width *= 0.0625f;
        if (head < 0.0) {
          // the whole prefix down to the band may fit the list
          const int got = smp_collect(C, [&](float x) { return x > xb && band.side(w.depth(x)) <= 0; });
          if (got <= kSmpList) {
            if (rank == 0) {
              double wt[kSmpPer], z;
              double run = smp_sort_list(C, w, got, wt, &z);
              int in = 0;
#pragma unroll
              for (int i = 0; i < kSmpPer; ++i) {
                in += tid * kSmpPer + i < got && run < target;
                run += wt[i];
              }
              int all;
              (void)block_exclusive_scan(in, S.scan_i, &all);
              smp_draw_list<E>(C, a, r, max(1, all), u);
            }
            drawn = done = true;
            break;
          }
        }
        if (head > (double)kSmpList) continue;
        const int got = smp_collect(C, [&](float x) { return x > xb && band.side(w.depth(x)) == 0; });
        if (got == 0 || got > kSmpList) continue;
        // the cut lies among these: the key and the ties of its last entry
        if (rank == 0) {
          double wt[kSmpPer], z;
          double run = above + smp_sort_list(C, w, got, wt, &z);
          int in = 0;
#pragma unroll
          for (int i = 0; i < kSmpPer; ++i) {
            in += tid * kSmpPer + i < got && run < target;
            run += wt[i];
          }
          int all;
          (void)block_exclusive_scan(in, S.scan_i, &all);
          const int keep = max(1, all);
          const uint32_t key = (uint32_t)(S.list.item[keep - 1] >> 32);
          int same = 0;
#pragma unroll
          for (int i = 0; i < kSmpPer; ++i) {
            const int at = tid * kSmpPer + i;
            same += at < keep && (uint32_t)(S.list.item[at] >> 32) == key;
          }
          (void)block_exclusive_scan(same, S.scan_i, &all);
          if (tid == 0) {
            S.cut_key = key;
            S.cut_ties = all;
          }
        }
        cl.sync();
        const SmpShared *R = cl.map_shared_rank(&S, 0);
        cut.key = (uint32_t)R->cut_key;
        cut.ties = R->cut_ties;
        cl.sync();  // read before rank 0 writes its cut_ties again
        done = true;
      }
    }
    if (!done) {  // key by key
      if (use_k) smp_top_k(C, w, cut.key + 1u, key_max, k, cut);
      if (use_p) {
        const SmpCut base = cut;
        smp_top_p(C, w, base, key_max, (double)p, cut);
      }
    }
    if (cut.ties > 0) tie_w = w(unmono(cut.key));
  }
  if (!drawn) smp_draw_row<E>(C, a, w, cut, tie_w, r, u);
  cl.sync();
}

}  // namespace fh

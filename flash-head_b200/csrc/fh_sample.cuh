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
//   1  its largest logit. Without a filter, the masses too. A row that is not kept
//      in shared memory also yields its candidates, the entries above a
//      threshold that a sample of the row gives, and under a top-p its mass in
//      fp32, whose error is bounded;
//   2  the candidates (at most 2048, in column order) are joined, sorted in
//      shared memory by one CTA, cut, and drawn from there. A mass known to a
//      factor is enough unless the cut differs between its two ends;
//   3  a top-p whose cut lies deeper: fp32 masses of 46 bands of logits say where
//      it lies (each thread sums bands of its own in shared memory: no atomics,
//      a fixed order), then one pass collects the entries of the band as
//      candidates and sums the exact masses above it. The segment of the draw is
//      scanned.
// Rows that resist (thousands of equal logits at a cut, top-k beyond 1024)
// descend through 16 bands of keys per pass, exact for every input.
//
// Bound: an unfiltered row costs a pass in fp64, not its bytes: an exponential
// is 14 fp64 instructions, about 9 clocks of an SM per 32 entries, 33 us for 256
// rows of 128256 entries against 10 us of reading. Filtered rows are bound by
// latency: a chain of passes, exchanges, a sort and scans, which the rows of
// other clusters cover in part. Measured, bf16 rows of 128256 unless said
// otherwise: one row with top-k and top-p 16.4 us; 64 rows of mixed filters 55
// us; 256 rows without a filter 70 us (0.9 TB/s), with top-k 50 52 us (1.3
// TB/s); 256 fp32 rows of 151936 with top-p 197 us, 114 us where the cut lies
// among the first candidates.
#pragma once

#include <cooperative_groups.h>

#include "fh_fused.cuh"

namespace fh {

constexpr int kSmpThreads = 256;
// CTAs per SM, of 64 registers a thread (rows in shared memory: half as many).
// Two of 128 registers are better for fp64 chains alone (256 unfiltered rows: 63
// us against 70), four for everything with candidates (256 rows with top-k 50 and
// top-p: 98 us against 74; 256 fp32 rows with top-p: 233 against 197).
constexpr int kSmpResident = 4;
constexpr int kSmpWarps = kSmpThreads / 32;
constexpr int kSmpBands = 16;
constexpr int kSmpWin = 48;  // bands of a window, the parts above and below it among them
constexpr int kSmpMaxCluster = 8;
constexpr int kSmpChunk = 2048;  // vectors of the segment of the draw looked at together
constexpr int kSmpList = 2048;   // candidates one CTA sorts
constexpr int kSmpPart = 512;    // candidates of one warp
constexpr int kSmpMaxK = 1024;   // largest top-k that goes through the list
// Vectors of a row that a thread keeps at most (CACHED): what two CTAs of an SM have
// room for.
constexpr int kSmpCache = 14;

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
  int cache;    // vectors that a thread keeps (CACHED)
};

struct __align__(16) SmpShared {
  union {
    struct {
      double mass[kSmpBands][kSmpThreads];
      uint32_t cnt[kSmpBands][kSmpThreads];
    } band;
    float win[kSmpWin][kSmpThreads];
    struct {
      // the warps' candidates, key << 32 | column, by column; later the sorted
      // keys of the whole list
      unsigned long long part[kSmpWarps][kSmpPart];
      uint32_t key[kSmpList], col[kSmpList];  // the whole list, by column
    } list;
    struct {
      double mass[kSmpChunk];
      int ties[kSmpChunk];
    } vec;  // kept mass and ties of the vectors of a piece of the row
  };
  // values exchanged between the CTAs of a cluster, double-buffered so that
  // one cluster barrier per exchange is enough
  double x_mass[2][kSmpWin];
  unsigned long long x_cnt[2][kSmpBands];
  double sum_mass[kSmpWin];
  unsigned long long sum_cnt[kSmpBands];
  // per warp: kept mass of its segment in units of 2^warp_k, and ties; of the
  // first pass: largest logit, whether the mass has to be summed again
  double warp_d[kSmpWarps];
  double warp_k[kSmpWarps];
  int warp_i[kSmpWarps];
  float warp_f[kSmpWarps];
  int warp_bad[kSmpWarps];
  double seg_before;
  long long seg_left;
  double scan_d[kSmpWarps];
  int scan_i[33];
  int part_n[kSmpWarps];  // candidates a warp found
  uint32_t warp_key[kSmpWarps];
  int verdict;
  int best, last;
  unsigned long long cut_key;
  long long cut_ties;
};

// Order of the logits: monotone in x, with -0 equal to +0. A NaN has no key (what
// comes out for one is some number's).
__device__ __forceinline__ uint32_t smp_key(float x) { return mono(x + 0.0f); }

// A key as a threshold that logits are compared with. No logit has the key of
// -0, but +0 > -0 does not hold: the next lower number stands for it.
__device__ __forceinline__ float smp_float(uint32_t key) {
  return unmono(key == 0x7FFFFFFFu ? 0x7FFFFFFEu : key);
}

template <typename E>
struct SmpElem;
template <>
struct SmpElem<float> {
  static constexpr int kVec = 4;
  __device__ __forceinline__ static float to_float(float v) { return v; }
  static constexpr uint32_t kNone = 0xFF800000u;  // -inf in every element of a word
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
  static constexpr uint32_t kNone = 0xFF80FF80u;
  __device__ __forceinline__ static __nv_bfloat16 none() { return __float2bfloat16(-INFINITY); }
  __device__ __forceinline__ static void unpack(const uint4 &v, float *f) {
    Vec<__nv_bfloat16>::to_float(v, f);
  }
};
template <>
struct SmpElem<__half> {
  static constexpr int kVec = 8;
  __device__ __forceinline__ static float to_float(__half v) { return __half2float(v); }
  static constexpr uint32_t kNone = 0xFC00FC00u;
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
  __device__ __forceinline__ float at(int c) const { return SmpElem<E>::to_float(p[c]); }
  __device__ __forceinline__ int column(int v) const { return v * kVec - mis; }
  __device__ __forceinline__ uint4 raw(int v) const {
    const int c0 = column(v);
    if (c0 >= 0 && c0 + kVec <= n) return __ldg(reinterpret_cast<const uint4 *>(p + c0));
    return edge(p, c0, n);
  }
  __device__ __noinline__ static uint4 edge(const E *p, int c0, int n) {
    union {
      uint4 u;
      E e[kVec];
    } x;
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      x.e[i] = c0 + i >= 0 && c0 + i < n ? p[c0 + i] : SmpElem<E>::none();
    return x.u;
  }
  // NaN stays: it fails every comparison below, as -inf does
  __device__ __forceinline__ static void unpack(const uint4 &u, float *f) {
    SmpElem<E>::unpack(u, f);
  }
};

// Polynomial of 2^f through the Chebyshev nodes of [-1/2, 1/2], relative error
// below 2e-14; in constant memory, so that a fused multiply-add takes its
// coefficient as an operand.
__constant__ double kSmpExp2[10] = {
    1.00000000000001354e+00, 6.93147180559946174e-01, 2.40226506956403407e-01,
    5.55041086646516774e-02, 9.61812919393430395e-03, 1.33335582007937186e-03,
    1.54034337512549968e-04, 1.52526729253468732e-05, 1.32596452439290570e-06,
    1.02059053204931027e-07};

// Mass of a logit in units of 2^k0: 2^(x c - k0) with c = log2(e) / T and k0
// the integer next to ref * c, so that x c - k0 is rounded once (fma) however
// large the two are. With 1.5 * 2^52 added, the sum's low word is its nearest
// integer n; the rest f is within 1/2, 2^f a polynomial, and n is added to the
// exponent. Masses below 2^-1000 of the reference's are none (2^n would leave the
// normal numbers); all others count, as u = 0 draws the first kept column however
// small its mass. `depth` is the same exponent, falling and in fp32: a monotone
// measure of how far down a logit lies.
// For |ref| c above 2^40 neighbouring fp32 logits differ by a factor of 2^(2^16):
// c is held there, where only the reference's equals keep a mass (`held`).
struct SmpMass {
  double c, k0, k1;
  float ref, xlo, cf;
  bool held;
  __device__ __forceinline__ SmpMass(float ref_, float T) : ref(ref_) {
    const double c0 = 1.4426950408889634 / (double)T, most = 1099511627776.0;
    held = fabs((double)ref) * c0 > most;
    c = held ? most / fabs((double)ref) : c0;
    k0 = rint((double)ref * c);
    k1 = 6755399441055744.0 - k0;
    xlo = fminf((float)((double)ref - 1000.0 / c), nextafterf(ref, -INFINITY));
    cf = fminf((float)(2.0 * c), 3.402823466e38f);
  }
  // halved first: ref - x may pass the largest fp32. Rounded here, so that it
  // is the same number wherever it is used.
  __device__ __forceinline__ float depth(float x) const {
    return __fmul_rn(fmaf(-0.5f, x, 0.5f * ref), cf);
  }
  // for x > xlo (and up to 2^900 above the reference)
  __device__ __forceinline__ double raw(float x) const {
    const double xd = (double)x;
    const double r = fma(xd, c, k1);
    const double f = fma(xd, c, k1 - r);
    double p = kSmpExp2[9];
#pragma unroll
    for (int i = 8; i >= 0; --i) p = fma(p, f, kSmpExp2[i]);
    return __hiloint2double(__double2hiint(p) + (__double2loint(r) << 20), __double2loint(p));
  }
  __device__ __forceinline__ double operator()(float x) const { return x > xlo ? raw(x) : 0.0; }
};

// A prefix of the order: keys above `key`, and the first `ties` equal ones.
struct SmpCut {
  uint32_t key;
  long long ties;
};

// A warp's segment of a row, and how it is walked.
template <typename E, bool CACHED>
struct SmpSpan {
  static constexpr int kVec = SmpElem<E>::kVec;
  static constexpr bool kCached = CACHED;
  SmpRow<E> row;
  int v0, v1;
  int lane;
  uint4 *cache;  // this thread's share of the row in shared memory (CACHED),
  int keep;      // of so many vectors

  // f(vector, kVec values), a lane every 32 vectors, by whole warps: lanes past
  // the segment get -inf. FIRST: the row is read for the first time; a CACHED
  // row then stays in shared memory.
  template <bool FIRST, int kAhead = 4, typename F>
  __device__ __forceinline__ void walk(F f) const {
    constexpr uint32_t no = SmpElem<E>::kNone;
    float x[kVec];
    if constexpr (CACHED) {
      if (FIRST) {
#pragma unroll 1
        for (int i0 = 0; i0 < keep; i0 += 4) {
#pragma unroll
          for (int i = i0; i < i0 + 4; ++i) {
            const int v = v0 + lane + 32 * i;
            if (i < keep)
              cache[kSmpThreads * i] = v < v1 ? row.raw(v) : make_uint4(no, no, no, no);
          }
        }
      }
#pragma unroll 1
      for (int i = 0, v = v0; v < v1; ++i, v += 32) {
        row.unpack(cache[kSmpThreads * i], x);
        f(v + lane, x);
      }
    } else {
      int v = v0;
      for (; v + 32 * kAhead <= v1; v += 32 * kAhead) {
        uint4 u[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) u[i] = row.raw(v + lane + 32 * i);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          row.unpack(u[i], x);
          f(v + lane + 32 * i, x);
        }
      }
#pragma unroll 1
      for (; v < v1; v += 32) {
        row.unpack(v + lane < v1 ? row.raw(v + lane) : make_uint4(no, no, no, no), x);
        f(v + lane, x);
      }
    }
  }
};

template <typename E, bool CACHED>
struct SmpCtx {
  using Elem = E;
  SmpSpan<E, CACHED> span;
  SmpShared &S;
  int rank, size;  // CTA in its cluster
  int phase;       // exchanges so far
  int tid, warp, lane;
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
      if (C.tid < kSmpBands) k += R->x_cnt[b][C.tid];
    }
    C.S.sum_mass[C.tid] = d;
    if (C.tid < kSmpBands) C.S.sum_cnt[C.tid] = k;
  }
  __syncthreads();
}

// Exclusive prefix sum of one double per thread, in a fixed order. (Out of
// line, like the other helpers of the short paths: a launch of few rows waits
// for instructions more than for anything else.)
__device__ __noinline__ double smp_scan(SmpShared &S, double v, double *total) {
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

__device__ __noinline__ int smp_count_scan(SmpShared &S, int v, int *total) {
  return block_exclusive_scan(v, S.scan_i, total);
}

// Sums the threads' bands: one warp a band, lane by lane, then over the cluster.
template <bool MASS, bool CNT, typename Ctx>
__device__ __forceinline__ void smp_band_sums(Ctx &C) {
  SmpShared &S = C.S;
  __syncthreads();
  for (int b = C.warp; b < kSmpBands; b += kSmpWarps) {
    double d = 0.0;
    unsigned long long k = 0ull;
    for (int i = C.lane; i < kSmpThreads; i += 32) {
      if (MASS) d += S.band.mass[b][i];
      if (CNT) k += S.band.cnt[b][i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if (MASS) d += __shfl_xor_sync(0xFFFFFFFFu, d, o);
      if (CNT) k += __shfl_xor_sync(0xFFFFFFFFu, k, o);
    }
    if (C.lane == 0) {
      S.x_mass[C.phase & 1][b] = d;
      S.x_cnt[C.phase & 1][b] = k;
    }
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
  C.span.template walk<false>([&](int, const float *f) {
#pragma unroll
    for (int i = 0; i < decltype(C.span)::kVec; ++i) {
      const uint32_t k = smp_key(f[i]);
      if (k >= lo && k <= hi && f[i] == f[i]) {
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

// Smallest key whose mass is at least min_p times the largest entry's.
__device__ __noinline__ uint32_t smp_min_key(float m, float T, float min_p) {
  const uint32_t top = smp_key(m);
  const double t = log2((double)min_p), c = 1.4426950408889634 / (double)T;
  auto enough = [&](uint32_t k) { return ((double)unmono(k) - (double)m) * c >= t; };
  // bisect the keys; the border's rounded value is nearly always within a step
  uint32_t lo = smp_key(-INFINITY), hi = top;  // lo: too little, hi: enough
  const uint32_t g = smp_key((float)fmin((double)m, (double)m + t / c));
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

// The entries that `hit` marks of a warp's vectors (a lane's first column c0)
// into the warp's part of the list, in column order; n counts on past its end.
template <int kVec>
__device__ __forceinline__ void smp_append(const float *f, int c0, uint32_t hit,
                                           unsigned long long *part, int &n) {
  if (__any_sync(0xFFFFFFFFu, hit)) {
    const unsigned below = (1u << (threadIdx.x & 31)) - 1u;
    int at = n;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const unsigned in = __ballot_sync(0xFFFFFFFFu, (hit >> i) & 1u);
      at += __popc(in & below);
      n += __popc(in);
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if ((hit >> i) & 1u) {
        if (at < kSmpPart)
          part[at] = ((unsigned long long)smp_key(f[i]) << 32) | (uint32_t)(c0 + i);
        ++at;
      }
  }
}

// Exchanges the number of candidates (and x_mass[0..n) of the caller): the
// cluster's total in sum_cnt[0], beyond kSmpList also where one warp found
// more than its part holds.
template <typename Ctx>
__device__ __forceinline__ void smp_count_list(Ctx &C, int masses = 1) {
  SmpShared &S = C.S;
  __syncthreads();
  if (C.warp == 0) {
    int n = C.lane < kSmpWarps ? S.part_n[C.lane] : 0;
    const bool over = __any_sync(0xFFFFFFFFu, n > kSmpPart);
    n = __reduce_add_sync(0xFFFFFFFFu, n);
    if (C.lane == 0) S.x_cnt[C.phase & 1][0] = over ? (unsigned long long)kSmpList + 1ull : n;
  }
  smp_exchange(C, masses);
}

// Rank 0 joins the warps' parts into its list, in column order (a cluster
// barrier before; one after: the other CTAs may go).
template <typename Ctx>
__device__ __forceinline__ void smp_gather(Ctx &C) {
  namespace cg = cooperative_groups;
  cg::cluster_group cl = cg::this_cluster();
  SmpShared &S = C.S;
  if (C.rank == 0) {
    static_assert(kSmpMaxCluster * kSmpWarps <= 64, "two parts per lane");
    const int parts = C.size * kSmpWarps, g = 2 * C.lane;
    const SmpShared *R = cl.map_shared_rank(&S, min(g / kSmpWarps, C.size - 1));
    const int n0 = g < parts ? R->part_n[g % kSmpWarps] : 0;
    const int n1 = g + 1 < parts ? R->part_n[(g + 1) % kSmpWarps] : 0;
    int incl = n0 + n1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xFFFFFFFFu, incl, o);
      if (C.lane >= o) incl += t;
    }
    const int at0 = incl - n0 - n1, at1 = incl - n1;
    for (int q = C.warp; q < parts; q += kSmpWarps) {
      const int base = __shfl_sync(0xFFFFFFFFu, q & 1 ? at1 : at0, q / 2);
      const int cnt = __shfl_sync(0xFFFFFFFFu, q & 1 ? n1 : n0, q / 2);
      const SmpShared *P = cl.map_shared_rank(&S, q / kSmpWarps);
      for (int i = C.lane; i < cnt; i += 32) {
        const unsigned long long e = P->list.part[q % kSmpWarps][i];
        S.list.key[base + i] = (uint32_t)(e >> 32);
        S.list.col[base + i] = (uint32_t)e;
      }
    }
  }
  if (C.size > 1) cl.sync();
  __syncthreads();
}

// Entries in (lo, hi] into the list of rank 0, when they fit; returns their
// number in the cluster. Contains cluster barriers.
template <typename Ctx>
__device__ __forceinline__ int smp_collect(Ctx &C, float lo, float hi) {
  constexpr int kVec = decltype(C.span)::kVec;
  SmpShared &S = C.S;
  __syncthreads();
  int n = 0;
  unsigned long long *part = S.list.part[C.warp];
  C.span.template walk<false>([&](int v, const float *f) {
    uint32_t hit = 0u;
#pragma unroll
    for (int i = 0; i < kVec; ++i) hit |= f[i] > lo && f[i] <= hi ? 1u << i : 0u;
    smp_append<kVec>(f, C.span.row.column(v), hit, part, n);
  });
  if (C.lane == 0) S.part_n[C.warp] = n;
  smp_count_list(C);
  const unsigned long long total = S.sum_cnt[0];
  if (total > (unsigned long long)kSmpList) return kSmpList + 1;
  smp_gather(C);
  return (int)total;
}

// Descending bitonic sort of n2 (a power of two, at most kSmpList) keys by the
// whole CTA. A thread holds kEach = n2 / threads neighbouring keys (one, of
// fewer threads, below that) in registers: short strides stay in a thread,
// those within a warp are shuffles, and only the 6 longest of a full CTA go
// through shared memory.
constexpr int kSmpPer = kSmpList / kSmpThreads;
template <int kEach>
__device__ __noinline__ void smp_sort_n(uint32_t *a, int n2) {
  const int tid = threadIdx.x, base = tid * kEach;
  uint32_t x[kEach];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEach; ++i) x[i] = base + i < n2 ? a[base + i] : 0u;
  const bool live = (tid & ~31) * kEach < n2;  // this warp has keys
#pragma unroll 1
  for (int size = 2; size <= n2; size <<= 1) {
#pragma unroll 1
    for (int step = size >> 1; step >= 32 * kEach; step >>= 1) {
      __syncthreads();
      if (live)
#pragma unroll
        for (int i = 0; i < kEach; ++i) a[base + i] = x[i];
      __syncthreads();
      if (live)
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          // the lower index keeps the larger key in a falling run
          const uint32_t y = a[(base + i) ^ step];
          const bool big = (((base + i) & step) == 0) == (((base + i) & size) == 0);
          x[i] = big ? max(x[i], y) : min(x[i], y);
        }
    }
    if (!live) continue;
#pragma unroll 1
    for (int step = min(size >> 1, 16 * kEach); step >= kEach; step >>= 1) {
      const bool low = (base & step) == 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const uint32_t y = __shfl_xor_sync(0xFFFFFFFFu, x[i], step / kEach);
        const bool big = low == (((base + i) & size) == 0);
        x[i] = big ? max(x[i], y) : min(x[i], y);
      }
    }
#pragma unroll
    for (int step = kEach / 2; step > 0; step >>= 1) {
      if (step >= size) continue;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        if (i & step) continue;
        const bool fall = ((base + i) & size) == 0;
        const uint32_t u = max(x[i], x[i | step]), v = min(x[i], x[i | step]);
        x[i] = fall ? u : v;
        x[i | step] = fall ? v : u;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (base + i < n2) a[base + i] = x[i];
  __syncthreads();
}
__device__ __forceinline__ void smp_sort(uint32_t *a, int n2) {
  static_assert(kSmpPer == 8, "sorts for 1 to 8 keys per thread");
  if (n2 <= kSmpThreads) return smp_sort_n<1>(a, n2);
  if (n2 <= 2 * kSmpThreads) return smp_sort_n<2>(a, n2);
  if (n2 <= 4 * kSmpThreads) return smp_sort_n<4>(a, n2);
  smp_sort_n<8>(a, n2);
}

__device__ __forceinline__ int smp_pow2(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

template <typename E>
__device__ __forceinline__ void smp_emit(const SampleArgs &a, int r, int col, double prob) {
  a.out[r] = a.ids ? (int64_t)a.ids[(long long)r * a.ids_stride + col] : (int64_t)col;
  if (a.prob) a.prob[r] = (float)prob;
}

// The list's prefix (rank 0's CTA): sorts its n keys and cuts them, as the
// caller says, at the first `keep` (counted among the keys above `least`), or at
// the mass `target` (target < 0: p times the prefix's own mass), which the
// entries from `above` on share with mass outside the list. Returns the cut and
// in *total the mass of the first `keep`.
struct SmpPick {
  uint32_t key;
  int ties, keep;
};
__device__ __noinline__ SmpPick smp_pick(SmpShared &S, SmpMass w, int n, uint32_t least,
                                         long long k, double p, double target, double above,
                                         double most, bool *sure) {
  const int tid = threadIdx.x;
  uint32_t *sorted = reinterpret_cast<uint32_t *>(S.list.part[0]);
  const int n2 = smp_pow2(n);
  for (int i = tid; i < n2; i += kSmpThreads) sorted[i] = i < n ? S.list.key[i] : 0u;
  smp_sort(sorted, n2);
  uint32_t key[kSmpPer];
  int in = 0, keep;
#pragma unroll
  for (int i = 0; i < kSmpPer; ++i) {
    const int at = tid * kSmpPer + i;
    key[i] = at < n ? sorted[at] : 0u;
    in += key[i] > least;
  }
  (void)smp_count_scan(S, in, &keep);
  if (k > 0) keep = (int)min(k, (long long)keep);
  if (p < 1.0) {
    double wt[kSmpPer], sum = 0.0, z;
#pragma unroll
    for (int i = 0; i < kSmpPer; ++i) {
      wt[i] = tid * kSmpPer + i < keep ? w(unmono(key[i])) : 0.0;
      sum += wt[i];
    }
    double run = above + smp_scan(S, sum, &z);
    if (target < 0.0) target = p * z;
    int reach = 0, reach_most = 0, all;
#pragma unroll
    for (int i = 0; i < kSmpPer; ++i) {
      const bool valid = tid * kSmpPer + i < keep;
      reach += valid && run < target;
      reach_most += valid && run < most;
      run += wt[i];
    }
    (void)smp_count_scan(S, reach | (reach_most << 16), &all);
    // the cut is the same for the least and the most that the target can be
    if (sure) *sure = (all & 0xFFFF) == (all >> 16) && most < above + z;
    keep = max(1, all & 0xFFFF);
  }
  SmpPick pick;
  pick.keep = keep;
  pick.key = sorted[keep - 1];
  int higher = 0, all;
#pragma unroll
  for (int i = 0; i < kSmpPer; ++i) higher += key[i] > pick.key;
  (void)smp_count_scan(S, higher, &all);
  pick.ties = keep - all;
  return pick;
}

// The draw from the list, cut at `pick` (rank 0's CTA).
template <typename E>
__device__ __noinline__ void smp_draw_list(SmpShared &S, const SampleArgs &a, SmpMass w, int r,
                                           int n, SmpPick pick, double u) {
  const int tid = threadIdx.x;
  if (tid == 0) {
    S.best = 0x7FFFFFFF;
    S.last = -1;
  }
  uint32_t key[kSmpPer];
  int ties = 0, all;
#pragma unroll
  for (int i = 0; i < kSmpPer; ++i) {
    const int at = tid * kSmpPer + i;
    key[i] = at < n ? S.list.key[at] : 0u;
    ties += key[i] == pick.key;
  }
  int left = pick.ties - smp_count_scan(S, ties, &all);
  double wt[kSmpPer], sum = 0.0, total;
#pragma unroll
  for (int i = 0; i < kSmpPer; ++i) {
    const bool keep = key[i] > pick.key || (key[i] == pick.key && left-- > 0);
    wt[i] = keep ? w(unmono(key[i])) : 0.0;
    sum += wt[i];
  }
  double run = smp_scan(S, sum, &total);
  const double target = u * total;
  int best = 0x7FFFFFFF, last = -1;
#pragma unroll
  for (int i = 0; i < kSmpPer; ++i) {
    run += wt[i];
    if (wt[i] > 0.0) {
      last = tid * kSmpPer + i;
      if (run > target) best = min(best, last);
    }
  }
  if (best != 0x7FFFFFFF) atomicMin(&S.best, best);
  if (last >= 0) atomicMax(&S.last, last);
  __syncthreads();
  if (tid == 0) {
    // past the end by rounding: the last entry with a mass
    const int at = S.best != 0x7FFFFFFF ? S.best : S.last;
    smp_emit<E>(a, r, (int)S.list.col[at], w(unmono(S.list.key[at])) / total);
  }
}

// The loops with fp64 exponentials are functions of their own: registers are
// allotted to them alone.
struct SmpSum {
  double sum;
  float top;
  int ties;
};
template <bool FIRST, bool TIES, typename Span>
__device__ __noinline__ SmpSum smp_sum(Span span, SmpMass w, float xc) {
  constexpr int kVec = Span::kVec;
  const float above = fmaxf(xc, w.xlo);
  double sum0 = 0.0, sum1 = 0.0;
  SmpSum r{0.0, -INFINITY, 0};
  span.template walk<FIRST>([&](int, const float *f) {
#pragma unroll
    for (int h = 0; h < kVec; h += 4) {
      double x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = w.raw(f[h + i]);
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        if (f[h + i] > above) sum0 += x[i];
        if (f[h + i + 1] > above) sum1 += x[i + 1];
        if (FIRST) r.top = fmaxf(r.top, fmaxf(f[h + i], f[h + i + 1]));
        if (TIES) r.ties += (f[h + i] == xc) + (f[h + i + 1] == xc);
      }
    }
  });
  r.sum = sum0 + sum1;
  return r;
}

// Kept mass and ties of this warp's segment, for the prefix `cut`; returns
// its largest logit (FIRST).
template <bool FIRST, bool TIES, typename Ctx>
__device__ __forceinline__ float smp_segment(Ctx &C, const SmpMass &w, const SmpCut &cut) {
  SmpSum r = smp_sum<FIRST, TIES>(C.span, w, smp_float(cut.key));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    r.sum += __shfl_xor_sync(0xFFFFFFFFu, r.sum, o);
    if (FIRST) r.top = fmaxf(r.top, __shfl_xor_sync(0xFFFFFFFFu, r.top, o));
    if (TIES) r.ties += __shfl_xor_sync(0xFFFFFFFFu, r.ties, o);
  }
  if (C.lane == 0) {
    C.S.warp_d[C.warp] = r.sum;
    C.S.warp_k[C.warp] = w.k0;
    C.S.warp_i[C.warp] = r.ties;
  }
  return r.top;
}

// The draw from the prefix `cut` of the whole row: the segments' masses are in
// warp_* of every CTA, in units of 2^warp_k; w gives masses in units of 2^w.k0. A
// segment whose largest logit has no mass in those units has none, whatever its sum
// in its own: the walk through the segment of the draw has to find a mass.
template <typename E, typename Ctx>
__device__ __forceinline__ void smp_draw_row(Ctx &C, const SampleArgs &a, const SmpMass &w,
                                             const SmpCut &cut, double tie_w, int r, double u) {
  namespace cg = cooperative_groups;
  cg::cluster_group cl = cg::this_cluster();
  constexpr int kVec = SmpRow<E>::kVec;
  SmpShared &S = C.S;
  const int tid = C.tid;
  const float xc = smp_float(cut.key), above = fmaxf(xc, w.xlo);
  if (tid == 0) {
    S.best = 0x7FFFFFFF;
    S.last = -1;
  }
  // every CTA finds the segment of the draw: thread i has segment i
  const int segs = C.size * kSmpWarps;
  double mass = 0.0;
  int seg_ties = 0;
  if (tid < segs) {
    const SmpShared *R = cl.map_shared_rank(&S, tid / kSmpWarps);
    mass = R->warp_d[tid % kSmpWarps];
    seg_ties = R->warp_i[tid % kSmpWarps];
    const double shift = R->warp_k[tid % kSmpWarps] - w.k0;
    if (shift != 0.0) mass = ldexp(mass, (int)fmax(-2000.0, fmin(shift, 2000.0)));
    if (!(R->warp_f[tid % kSmpWarps] > above)) mass = 0.0;
  }
  long long left = cut.ties;
  if (cut.ties > 0) {
    int all_ties;
    left -= smp_count_scan(S, seg_ties, &all_ties);
    if (left > 0) mass += (double)min(left, (long long)seg_ties) * tie_w;
  }
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
    S.seg_before = before;
    S.seg_left = left;
  }
  __syncthreads();
  if (seg / kSmpWarps != C.rank) return;
  // the segment in pieces of kSmpChunk vectors: their masses, then the vector
  // of the draw, then its entry. The target may lie past the end by rounding:
  // the last entry with a mass then, which any piece may hold.
  const int sv0 = (int)((long long)C.span.row.nv * seg / segs);
  const int sv1 = (int)((long long)C.span.row.nv * (seg + 1) / segs);
  constexpr int kEach = kSmpChunk / kSmpThreads;
  double run = S.seg_before;
  left = S.seg_left;
  // the first entry of vector v beyond the target, or the last kept one; `to`:
  // the mass before it, `ties`: how many equal entries are still kept there
  const auto emit = [&](int v, double to, long long ties) {
    float f[kVec];
    C.span.row.unpack(C.span.row.raw(v), f);
    int col = -1;
    double x = 0.0;
    bool found = false;
#pragma unroll
    for (int q = 0; q < kVec; ++q) {
      double e = 0.0;
      if (f[q] > above)
        e = w.raw(f[q]);
      else if (cut.ties > 0 && f[q] == xc && ties-- > 0)
        e = tie_w;
      to += e;
      if (e > 0.0 && !found) {
        col = C.span.row.column(v) + q;
        x = e;
        found = to > target;
      }
    }
    smp_emit<E>(a, r, col, x / total);
  };
  int kept = -1;  // the last vector with a mass of the pieces so far
  for (int c0 = sv0; c0 < sv1; c0 += kSmpChunk) {
    const int cn = min(kSmpChunk, sv1 - c0);
    __syncthreads();
    if (tid == 0) {
      S.best = 0x7FFFFFFF;
      S.last = -1;
    }
    for (int i = tid; i < cn; i += kSmpThreads) {
      float f[kVec];
      double x[kVec], sum = 0.0;
      int t = 0;
      C.span.row.unpack(C.span.row.raw(c0 + i), f);
#pragma unroll
      for (int q = 0; q < kVec; ++q) x[q] = w.raw(f[q]);
#pragma unroll
      for (int q = 0; q < kVec; ++q) {
        if (f[q] > above) sum += x[q];
        t += f[q] == xc;
      }
      S.vec.mass[i] = sum;
      S.vec.ties[i] = t;
    }
    __syncthreads();
    double m[kEach], sum = 0.0;
    long long l[kEach];  // ties still to be kept at the vector
    if (cut.ties > 0) {
      int t = 0, all;
#pragma unroll
      for (int i = 0; i < kEach; ++i) t += tid * kEach + i < cn ? S.vec.ties[tid * kEach + i] : 0;
      long long lft = left - smp_count_scan(S, t, &all);
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        l[i] = lft;
        lft -= tid * kEach + i < cn ? S.vec.ties[tid * kEach + i] : 0;
      }
      left -= all;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int at = tid * kEach + i;
      m[i] = at < cn ? S.vec.mass[at] : 0.0;
      if (cut.ties > 0 && at < cn && l[i] > 0)
        m[i] += (double)min(l[i], (long long)S.vec.ties[at]) * tie_w;
      sum += m[i];
    }
    double piece;
    const double base = run + smp_scan(S, sum, &piece);
    double before_v = base;
    int hit = 0x7FFFFFFF, last = -1;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (m[i] > 0.0) {
        last = tid * kEach + i;
        if (hit == 0x7FFFFFFF && before_v + m[i] > target) hit = last;
      }
      before_v += m[i];
    }
    if (hit != 0x7FFFFFFF) atomicMin(&S.best, hit);
    if (last >= 0) atomicMax(&S.last, last);
    __syncthreads();
    const int at = S.best;
    const int in = at != 0x7FFFFFFF ? at : S.last;  // the vector to go back to
    if (in >= 0) {
      kept = c0 + in;
      if (in / kEach == tid) {
        double to = base;
        long long ties = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          if (tid * kEach + i < in) to += m[i];
          if (cut.ties > 0 && tid * kEach + i == in) ties = l[i];
        }
        if (at != 0x7FFFFFFF)
          emit(kept, to, ties);
        else
          S.seg_left = ties;
      }
    }
    if (at != 0x7FFFFFFF) return;
    run += piece;
  }
  __syncthreads();
  if (tid == 0) emit(kept, -INFINITY, S.seg_left);
}

// The first pass of the list path: the thread's largest logit, the entries
// above `lo` into the CTA's list and, MASS, the row's mass relative to `ref` in
// fp32, smp_slack of it off at most: with t = (x - ref) c, the difference is
// off by 2^-24 |t| (t > -100, and below 2^-32 nothing counts; above the reference
// up to the row's largest t), c's second word corrects its product, and ex2
// (2^-22), the products and a vector's sum add 2^-20.
constexpr double kSmpSlack = 3.8147e-6;  // 2^-18, where no logit is above `ref`
__device__ __forceinline__ double smp_slack(float m, float ref, double c) {
  const double t = ((double)m - (double)ref) * c;
  return kSmpSlack + (t > 0.0 ? 0x1p-24 * t : 0.0);
}
__device__ __forceinline__ float smp_ex2(float t) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t));
  return y;
}
struct SmpFloat {
  float ref, c_hi, c_lo, xcut;
  __device__ __forceinline__ SmpFloat(float ref_, double c)
      : ref(ref_), c_hi((float)c), c_lo((float)(c - (double)(float)c)),
        xcut(ref_ - 100.f / (float)c) {}
  __device__ __forceinline__ float operator()(float f) const {
    const float x = f - ref, t = x * c_hi;
    const float e = smp_ex2(t), d = fmaf(x, c_lo, fmaf(x, c_hi, -t));
    return fmaf(e, d * 0.69314718f, e);
  }
};
struct SmpFirst {
  double z;
  float top;
};
template <bool MASS, typename Span>
__device__ __noinline__ SmpFirst smp_first(Span span, float lo, float ref, double c,
                                           unsigned long long *part, int *part_n) {
  constexpr int kVec = Span::kVec;
  const SmpFloat e2(ref, c);
  SmpFirst r{0.0, -INFINITY};
  int n = 0;
  span.template walk<true>([&](int v, const float *f) {
    uint32_t hit = 0u;
    float sum = 0.f, top = f[0];
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      if (i) top = fmaxf(top, f[i]);
      if (MASS) {
        const float y = e2(f[i]);
        if (f[i] > e2.xcut) sum += y;
      }
    }
    r.top = fmaxf(r.top, top);
    if (MASS) r.z += (double)sum;
    if (top > lo) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) hit |= f[i] > lo ? 1u << i : 0u;
    }
    smp_append<kVec>(f, span.row.column(v), hit, part, n);
  });
  if (span.lane == 0) *part_n = n;
  return r;
}

// A threshold above which a row in random order has about `want` entries, and
// the largest logit of the sample: one vector per thread, spread over the row
// and the same in every CTA of the cluster. The threshold is the r-th largest
// of the vectors' maxima.
template <typename Ctx>
__device__ __forceinline__ void smp_sample(Ctx &C, float want, float &lo, float &ref) {
  constexpr int kVec = decltype(C.span)::kVec;
  SmpShared &S = C.S;
  float f[kVec];
  C.span.row.unpack(
      C.span.row.raw((int)((long long)C.span.row.nv * C.tid / kSmpThreads)), f);
  float x = f[0];
#pragma unroll
  for (int i = 1; i < kVec; ++i) x = fmaxf(x, f[i]);
  x = fmaxf(x, -INFINITY);  // all NaN
  // its key's upper bits, by halving: a threshold slightly below
  const uint32_t key = smp_key(x);
  const int r = min(kSmpThreads, max(4, (int)(want * (kSmpThreads * kVec) / (float)C.span.row.n)));
  const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, key);
  if (C.lane == 0) S.warp_key[C.warp] = top;
  uint32_t pre = 0u;
#pragma unroll 1
  for (int bit = 31; bit >= 12; --bit) {
    const uint32_t t = pre | (1u << bit);
    if (__syncthreads_count(key >= t) >= r) pre = t;
  }
  uint32_t most = 0u;
#pragma unroll
  for (int i = 0; i < kSmpWarps; ++i) most = max(most, S.warp_key[i]);
  ref = unmono(most);
  // (at most what the r-th largest is, and -inf for -inf)
  lo = pre > smp_key(-INFINITY) ? smp_float(pre) : -INFINITY;
}

// The window of a deep top-p cut: logits up to `hi` in 46 bands of equal width,
// band 0 above it, band 47 below. Band j is (edge(j), edge(j - 1)].
struct SmpWindow {
  float hi, scale;  // scale: bands per logit
  __device__ __forceinline__ int band(float x) const {
    const float y = fminf(fmaxf(fmaf(hi - x, scale, 0.5f), 0.f), (float)(kSmpWin - 1));
    return __float_as_int(y + 8388608.f) & 63;  // the nearest integer
  }
  __device__ __forceinline__ float edge(int j) const { return hi - (float)j / scale; }
};

// Per-thread masses of a window's bands, of the logits above `base`, in fp32
// relative to `ref`; returns the thread's largest logit. (Bands of the thread's
// own: no atomics, a fixed order.) The row's mass is off by kSmpSlack, and 2^-24
// for every addition: the thread's entries (at most 16 more than an equal
// share of the row), and 13 that join the threads' bands.
template <typename Span>
__device__ __noinline__ float smp_window(Span span, SmpWindow win, float base, float ref, double c,
                                         float *mine) {
  constexpr int kVec = Span::kVec;
  const SmpFloat e2(ref, c);
  const float xcut = fmaxf(base, e2.xcut);
  float top = -INFINITY;
#pragma unroll 8
  for (int i = 0; i < kSmpWin; ++i) mine[i * kSmpThreads] = 0.f;
  span.template walk<false>([&](int, const float *f) {
#pragma unroll
    for (int h = 0; h < kVec; h += 4) {
      float e[4];
      int j[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = f[h + i];
        top = fmaxf(top, x);
        e[i] = e2(x);
        e[i] = x > xcut ? e[i] : 0.f;
        j[i] = win.band(x) * kSmpThreads;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) mine[j[i]] += e[i];
    }
  });
  return top;
}

// Sums the threads' window bands over the CTA, in a fixed order.
template <typename Ctx>
__device__ __forceinline__ void smp_window_sums(Ctx &C, double *out) {
  static_assert(kSmpWin % kSmpWarps == 0, "as many bands to every warp");
  __syncthreads();
  float d[kSmpWin / kSmpWarps];
#pragma unroll
  for (int b = 0; b < kSmpWin / kSmpWarps; ++b) {
    d[b] = 0.f;
#pragma unroll
    for (int i = 0; i < kSmpThreads; i += 32)
      d[b] += C.S.win[b * kSmpWarps + C.warp][i + C.lane];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int b = 0; b < kSmpWin / kSmpWarps; ++b) d[b] += __shfl_xor_sync(0xFFFFFFFFu, d[b], o);
  if (C.lane < kSmpWin / kSmpWarps) {
    float mine = d[0];
#pragma unroll
    for (int b = 1; b < kSmpWin / kSmpWarps; ++b) mine = C.lane == b ? d[b] : mine;
    out[C.lane * kSmpWarps + C.warp] = (double)mine;
  }
}

// One pass: exact masses of the logits above `hi` and above `base`, per thread, and
// the entries in (lo, hi] into the warp's part of the list.
struct SmpExact {
  double above, all;
};
template <typename Span>
__device__ __noinline__ SmpExact smp_exact(Span span, SmpMass w, float base, float lo, float hi,
                                           unsigned long long *part, int *part_n) {
  constexpr int kVec = Span::kVec;
  double all0 = 0.0, all1 = 0.0, above0 = 0.0, above1 = 0.0;
  int n = 0;
  span.template walk<false, kVec == 4 ? 2 : 1>([&](int v, const float *f) {
    uint32_t hit = 0u;
#pragma unroll
    for (int i = 0; i < kVec; ++i) hit |= f[i] > lo && f[i] <= hi ? 1u << i : 0u;
#pragma unroll
    for (int h = 0; h < kVec; h += 4) {
      double x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = w.raw(f[h + i]);
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        if (f[h + i] > base) all0 += x[i];
        if (f[h + i + 1] > base) all1 += x[i + 1];
        if (f[h + i] > hi) above0 += x[i];
        if (f[h + i + 1] > hi) above1 += x[i + 1];
      }
    }
    smp_append<kVec>(f, span.row.column(v), hit, part, n);
  });
  if (span.lane == 0) *part_n = n;
  return SmpExact{above0 + above1, all0 + all1};
}

// A deep top-p cut of the logits above `base`: the window's masses, relative to
// `ref`, are in sum_mass; m is the row's largest logit. Finds the bands that hold
// the cut (a window of their own if they hold too many entries). Where that is
// near the top, the candidates are the whole prefix, and a mass known to a
// factor may do (a row in shared memory is summed at once); otherwise one pass gives the exact masses and the candidates,
// then come the cut and the segments' masses for the draw. kDrawn: it has been
// drawn. kLost: nothing but the passes.
enum SmpDeep { kLost, kCut, kDrawn };
template <typename E, typename Ctx>
__device__ __forceinline__ SmpDeep smp_deep(Ctx &C, const SampleArgs &a, const SmpMass &w,
                                            SmpWindow win, float base, float m, float ref,
                                            double c, float p, int r, double u, SmpCut &cut) {
  namespace cg = cooperative_groups;
  cg::cluster_group cl = cg::this_cluster();
  SmpShared &S = C.S;
  const int lane = C.lane;
  const float cf = (float)c;
  float lo = 0.f, hi = 0.f;
  bool whole = false;  // (lo, m] is short enough
  double z;
#pragma unroll 1
  for (int level = 0;; ++level) {
    // lane i has bands 2 i and 2 i + 1
    const bool mine = lane < kSmpWin / 2;
    const double a0 = mine ? S.sum_mass[2 * lane] : 0.0, a1 = mine ? S.sum_mass[2 * lane + 1] : 0.0;
    double incl = a0 + a1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(0xFFFFFFFFu, incl, o);
      if (lane >= o) incl += t;
    }
    z = __shfl_sync(0xFFFFFFFFu, incl, 31);
    // the band that reaches a mass
    const auto reach = [&](double need) {
      const unsigned b0 = __ballot_sync(0xFFFFFFFFu, mine && incl - a1 >= need);
      const unsigned b1 = __ballot_sync(0xFFFFFFFFu, mine && incl >= need);
      const int l = __ffs(b0 | b1) - 1;
      return b0 | b1 ? 2 * l + ((b0 >> l) & 1u ? 0 : 1) : kSmpWin - 1;
    };
    // 2^-12 of room each way
    const int j0 = reach((double)p * z * (1.0 - 0x1p-12));
    const int j1 = reach((double)p * z * (1.0 + 0x1p-12));
    // entries of a band: at most its mass over the least of theirs
    const float n0 = a0 > 0.0 ? (float)a0 * smp_ex2((ref - win.edge(2 * lane)) * cf) : 0.f;
    const float n1 = a1 > 0.0 ? (float)a1 * smp_ex2((ref - win.edge(2 * lane + 1)) * cf) : 0.f;
    float prefix = (2 * lane <= j1 ? n0 : 0.f) + (2 * lane + 1 <= j1 ? n1 : 0.f);
    float in = (2 * lane >= j0 && 2 * lane <= j1 ? n0 : 0.f) +
               (2 * lane + 1 >= j0 && 2 * lane + 1 <= j1 ? n1 : 0.f);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      prefix += __shfl_xor_sync(0xFFFFFFFFu, prefix, o);
      in += __shfl_xor_sync(0xFFFFFFFFu, in, o);
    }
    __syncthreads();
    if (!(z > 0.0)) return kLost;
    const bool last = j1 == kSmpWin - 1;  // (it has no lower edge)
    // (a logit on an edge may be in either band: 1 % of one more each way)
    hi = j0 > 0 ? fminf(win.edge(j0 - 1) + 0.01f / win.scale, m) : m;
    lo = last ? win.edge(kSmpWin - 2) - 24.f / cf : win.edge(j1) - 0.01f / win.scale;
    lo = fmaxf(fminf(lo, nextafterf(hi, -INFINITY)), base);
    const bool fits = !last || lo == base;
    whole = fits && prefix <= (float)kSmpList;
    if (whole || (fits && in <= (float)kSmpList)) break;
    if (level == 3) return kLost;
    win.hi = hi;
    win.scale = (float)(kSmpWin - 2) / (hi - lo);
    if (!(win.scale > 0.f && win.scale < 1e30f)) return kLost;
    smp_window(C.span, win, base, ref, c, &S.win[0][C.tid]);
    smp_window_sums(C, S.x_mass[C.phase & 1]);
    smp_exchange(C, kSmpWin);
  }
  const uint32_t least = cut.key;
  if (whole && decltype(C.span)::kCached) {
    hi = m;
  } else if (whole) {
    const int got = smp_collect(C, lo, m);
    if (got > 0 && got <= kSmpList) {
      hi = m;
      if (C.rank == 0) {
        const double slack = kSmpSlack + 0x1p-24 * (32.0 + (double)C.span.row.n /
                                                               (double)(kSmpThreads * C.size));
        const double target = (double)p * z * exp2(fma((double)ref, w.c, -w.k0));
        bool sure = false;
        const SmpPick pick = smp_pick(S, w, got, least, 0, (double)p, target * (1.0 - slack), 0.0,
                                      target * (1.0 + slack), &sure);
        sure = sure && !w.held && target > 0.0;
        if (C.tid == 0) S.verdict = sure;
        if (sure) smp_draw_list<E>(S, a, w, r, got, pick, u);
      }
      cl.sync();
      const int ok = cl.map_shared_rank(&S, 0)->verdict;
      cl.sync();
      if (ok) return kDrawn;
    }
  }
  hi = fmaxf(hi, w.xlo);  // masses below are none
  SmpExact e = smp_exact(C.span, w, fmaxf(base, w.xlo), lo, hi, S.list.part[C.warp], &S.part_n[C.warp]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    e.above += __shfl_xor_sync(0xFFFFFFFFu, e.above, o);
    e.all += __shfl_xor_sync(0xFFFFFFFFu, e.all, o);
  }
  if (C.lane == 0) {
    S.warp_d[C.warp] = e.above;
    S.warp_k[C.warp] = w.k0;
    S.scan_d[C.warp] = e.all;
  }
  __syncthreads();
  if (C.tid == 0) {
    double above = 0.0, all = 0.0;
    for (int i = 0; i < kSmpWarps; ++i) {
      above += S.warp_d[i];
      all += S.scan_d[i];
    }
    S.x_mass[C.phase & 1][0] = above;
    S.x_mass[C.phase & 1][1] = all;
  }
  smp_count_list(C, 2);
  const double above = S.sum_mass[0], target = (double)p * S.sum_mass[1];
  const unsigned long long listed = S.sum_cnt[0];
  if (listed == 0 || listed > (unsigned long long)kSmpList || !(above < target)) return kLost;
  smp_gather(C);
  if (C.rank == 0) {
    bool sure = false;
    const SmpPick pick = smp_pick(S, w, (int)listed, least, 0, (double)p, target, above, target, &sure);
    if (C.tid == 0) {
      S.cut_key = pick.key;
      S.cut_ties = pick.ties;
      S.verdict = sure;
    }
    if (sure && hi == m) smp_draw_list<E>(S, a, w, r, (int)listed, pick, u);
  }
  cl.sync();
  const SmpShared *R = cl.map_shared_rank(&S, 0);
  if (!R->verdict) {
    cl.sync();
    return kLost;
  }
  if (hi == m) {
    cl.sync();
    return kDrawn;
  }
  cut.key = (uint32_t)R->cut_key;
  cut.ties = R->cut_ties;
  // the segment's kept candidates (rank 0 sorted over its parts: its own lead
  // its list)
  int first = 0;
  for (int i = 0; i < C.warp; ++i) first += S.part_n[i];
  double kept = 0.0;
  int ties = 0;
  for (int i = C.lane; i < S.part_n[C.warp]; i += 32) {
    const uint32_t key = C.rank == 0 ? S.list.key[first + i]
                                     : (uint32_t)(S.list.part[C.warp][i] >> 32);
    if (key > cut.key) kept += w(unmono(key));
    ties += key == cut.key;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    kept += __shfl_xor_sync(0xFFFFFFFFu, kept, o);
    ties += __shfl_xor_sync(0xFFFFFFFFu, ties, o);
  }
  if (C.lane == 0) {
    S.warp_d[C.warp] += kept;
    S.warp_i[C.warp] = ties;
  }
  cl.sync();
  return kCut;
}

// CACHED: every lane's share of the row is at most a.cache vectors, kept in
// shared memory.
template <typename E, bool CACHED>
__global__ void __launch_bounds__(kSmpThreads, CACHED ? kSmpResident / 2 : kSmpResident) k_sample(SampleArgs a) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) unsigned char smp_raw[];
  SmpShared &S = *reinterpret_cast<SmpShared *>(smp_raw);
  cg::cluster_group cl = cg::this_cluster();
  constexpr int kVec = SmpRow<E>::kVec;
  const int size = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int r = blockIdx.x / size;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  SmpCtx<E, CACHED> C{
      {SmpRow<E>(reinterpret_cast<const E *>(a.logits) + (long long)r * a.stride, a.n), 0, 0, lane,
       reinterpret_cast<uint4 *>(smp_raw + sizeof(SmpShared)) + tid, a.cache},
      S, rank, size, 0, tid, warp, lane};
  {
    const int gw = rank * kSmpWarps + warp, warps = size * kSmpWarps;
    C.span.v0 = (int)((long long)C.span.row.nv * gw / warps);
    C.span.v1 = (int)((long long)C.span.row.nv * (gw + 1) / warps);
  }
  float T = a.temperature ? a.temperature[r] : a.temperature0;
  const long long k = a.top_k ? a.top_k[r] : a.top_k0;
  const float p = a.top_p ? a.top_p[r] : a.top_p0;
  const float mp = a.min_p ? a.min_p[r] : a.min_p0;
  double u = a.uniforms[r];
  u = u > 0.0 ? u : 0.0;
  const bool one = !(T > 0.f) || k == 1 || p <= 0.f;  // the first entry
  if (!(T > 0.f)) T = 1.f;
  const bool use_k = !one && k > 0 && k < a.n, use_p = !one && p < 1.f, use_m = !one && mp > 0.f;
  const bool all = !one && !use_k && !use_p && !use_m;  // no filter
  const bool nucleus = use_p && !use_k && !use_m;       // top-p alone
  const uint32_t key_none = smp_key(-INFINITY);
  SmpCut cut{key_none, 0};

  // The first pass: the row's largest logit. Without a filter it sums the
  // masses as well, every warp in units of the largest of its first entries;
  // where a filter keeps few entries it collects those above a threshold that
  // a sample gives (a row in shared memory is better walked twice).
  const bool fast = !CACHED && !one && !all && (!use_k || k <= kSmpMaxK);
  float mt = -INFINITY, m, fast_lo = -INFINITY, ref = 0.f;
  int first = 0x7FFFFFFF;
  SmpMass w(0.f, T);
  int bad = 1;
  const double c = 1.4426950408889634 / (double)T;
  if (all) {
    float f[kVec];
    ref = -INFINITY;
    if (C.span.v0 + lane < C.span.v1) {
      C.span.row.unpack(C.span.row.raw(C.span.v0 + lane), f);
#pragma unroll
      for (int i = 0; i < kVec; ++i) ref = fmaxf(ref, f[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ref = fmaxf(ref, __shfl_xor_sync(0xFFFFFFFFu, ref, o));
    // (0 stands in for first entries that are all masked, or +inf: then the
    // others' masses are good only near it)
    const bool known = fabsf(ref) < INFINITY;
    if (!known) ref = 0.f;
    w = SmpMass(ref, T);
    m = smp_segment<true, false>(C, w, cut);
    const float deep = w.depth(m);
    bad = w.held || deep < -900.f || (!known && m > -INFINITY && deep > 60.f);
  } else if (fast) {
    if (a.n > kSmpList)
      smp_sample(C, use_k ? 1.1f * (float)k + 10.f * sqrtf((float)k) + 32.f : 600.f, fast_lo, ref);
    if (!(fabsf(ref) < INFINITY)) ref = 0.f;
    SmpFirst f;
    unsigned long long *part = S.list.part[warp];
    if (nucleus && a.n > kSmpList)
      f = smp_first<true>(C.span, fast_lo, ref, c, part,
                          &S.part_n[warp]);
    else
      f = smp_first<false>(C.span, fast_lo, ref, 1.0, part, &S.part_n[warp]);
    m = mt = f.top;
    double z;
    smp_scan(S, f.z, &z);
    if (tid == 0) S.x_mass[C.phase & 1][0] = z;
  } else {
    C.span.template walk<true>([&](int v, const float *f) {
      float x = f[0];
#pragma unroll
      for (int i = 1; i < kVec; ++i) x = fmaxf(x, f[i]);
      if (x > mt) {
        mt = x;
        first = v;
      }
    });
    m = mt;
  }
  if (!all) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  }
  if (lane == 0) {
    S.warp_f[warp] = m;
    S.warp_bad[warp] = bad;
  }
  if (fast)
    smp_count_list(C);
  else
    cl.sync();
  bad = 0;
  m = -INFINITY;
  for (int i = lane; i < size * kSmpWarps; i += 32) {
    const SmpShared *R = cl.map_shared_rank(&S, i / kSmpWarps);
    m = fmaxf(m, R->warp_f[i % kSmpWarps]);
    bad |= R->warp_bad[i % kSmpWarps];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  bad = __any_sync(0xFFFFFFFFu, bad);
  if (m == -INFINITY) {  // nothing left in this row
    if (rank == 0 && tid == 0) {
      a.out[r] = -1;
      if (a.prob) a.prob[r] = 0.f;
    }
    cl.sync();
    return;
  }
  const uint32_t key_max = smp_key(m);
  if (one) {
    // the first column of the largest logit
    if (tid == 0) S.best = 0x7FFFFFFF;
    __syncthreads();
    if (mt == m) {
      float f[kVec];
      C.span.row.unpack(C.span.row.raw(first), f);
      int col = 0x7FFFFFFF;
#pragma unroll
      for (int i = kVec - 1; i >= 0; --i)
        if (f[i] == m) col = C.span.row.column(first) + i;
      atomicMin(&S.best, col);
    }
    cl.sync();
    if (rank == 0 && tid == 0) {
      int col = S.best;
      for (int q = 1; q < size; ++q) col = min(col, cl.map_shared_rank(&S, q)->best);
      smp_emit<E>(a, r, col, 1.0);
    }
    cl.sync();
    return;
  }
  if (all) {
    // a common unit for the masses: the row's largest logit
    w = SmpMass(m < INFINITY ? m : 0.f, T);
  } else if (bad) {
    w = SmpMass(m < INFINITY ? m : 0.f, T);
  }
  double tie_w = 1.0;
  if (m == INFINITY) {
    // the +inf entries are equal and have all the mass: every filter counts
    int cnt = 0;
    C.span.template walk<false>([&](int, const float *f) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) cnt += f[i] == INFINITY;
    });
    cnt = __reduce_add_sync(0xFFFFFFFFu, cnt);
    if (lane == 0) S.x_cnt[C.phase & 1][warp] = (unsigned long long)cnt;
    smp_exchange(C, kSmpWarps);
    cut.key = key_max;
    for (int i = 0; i < kSmpWarps; ++i) cut.ties += (long long)S.sum_cnt[i];
    if (use_k) cut.ties = min(cut.ties, k);
    if (use_p) cut.ties = smp_ties((double)p * (double)cut.ties, cut.ties);
    bad = 1;
  } else if (!all) {
    if (use_m) cut.key = smp_min_key(m, T, fminf(mp, 1.f)) - 1u;
    const float xb = smp_float(cut.key);  // the base: logits above
    const bool whole = xb >= fast_lo;     // the list holds all of it
    const unsigned long long listed = fast ? S.sum_cnt[0] : 0ull;
    if (listed > 0 && listed <= (unsigned long long)kSmpList &&
        (whole || nucleus || (use_k && listed >= (unsigned long long)k))) {
      const double z_row = S.sum_mass[0];
      const bool known = whole || !nucleus;
      smp_gather(C);
      if (rank != 0 && known) return;
      if (rank == 0) {
        // a row's mass known to a factor of 1 +- smp_slack is enough, unless the
        // cut falls between the two
        double target = -1.0, most = 0.0;
        bool sure = false;
        if (!known) {
          const double slack = smp_slack(m, ref, c);
          target = (double)p * z_row * exp2(fma((double)ref, w.c, -w.k0));
          most = target * (1.0 + slack);
          target *= 1.0 - slack;
        }
        const SmpPick pick = smp_pick(S, w, (int)listed, cut.key, use_k ? k : 0,
                                      use_p ? (double)p : 1.0, target, 0.0, most, &sure);
        sure = known || (sure && !w.held && target >= 0.0);
        if (tid == 0) S.verdict = sure;
        if (sure) smp_draw_list<E>(S, a, w, r, (int)listed, pick, u);
        if (known) return;
      }
      cl.sync();
      const int ok = cl.map_shared_rank(&S, 0)->verdict;
      cl.sync();
      if (ok) return;
    }
    // What is tried next: the list of the candidates of a top-k or min-p, a
    // deep cut, the cut key by key; kRow: the cut is known.
    enum { kList, kDeep, kKeys, kRow } next;
    float lo = xb;
    bad = 1;
    if (!nucleus && (!use_k || k <= kSmpMaxK)) {
      next = kList;
      if (use_k) {
        // of a row in random order, about `want` entries lie above the
        // threads' rank_t-th largest maximum: a thread's maximum is above it
        // with probability 1 - exp(-want / threads). `want` leaves room for
        // the spread of the count and for the highest of the CTAs' thresholds.
        const float want = 1.1f * (float)k + 10.f * sqrtf((float)k) + 32.f;
        const int rank_t = max(1, (int)(kSmpThreads *
                                        (1.f - __expf(-want / (float)(kSmpThreads * size)))));
        const uint32_t kt = smp_key(mt);
        uint32_t pre = 0u;
#pragma unroll 1
        for (int bit = 31; bit >= 12; --bit) {
          const uint32_t c = pre | (1u << bit);
          if (__syncthreads_count(kt >= c) >= rank_t) pre = c;
        }
        if (size > 1) {
          const int b = C.phase & 1;
          ++C.phase;
          if (tid == 0) S.x_cnt[b][0] = pre;
          cl.sync();
          for (int q = 0; q < size; ++q)
            pre = max(pre, (uint32_t)cl.map_shared_rank(&S, q)->x_cnt[b][0]);
        }
        lo = smp_float(max(cut.key, pre - 1u));
      }
    } else {
      next = use_k ? kKeys : kDeep;
    }
#pragma unroll 1
    while (next != kRow) {
      if (next == kDeep) {
        const SmpWindow win{m, 2.f * (float)c};
        SmpDeep d = kLost;
        if (win.scale < 1e30f) {
          smp_window(C.span, win, xb, m, c, &S.win[0][tid]);
          smp_window_sums(C, S.x_mass[C.phase & 1]);
          smp_exchange(C, kSmpWin);
          d = smp_deep<E>(C, a, w, win, xb, m, m, c, p, r, u, cut);
        }
        if (d == kDrawn) return;
        if (d == kCut) bad = 0;
        next = d == kCut ? kRow : kKeys;
        continue;
      }
      if (next == kKeys) {
        if (use_k) smp_top_k(C, w, cut.key + 1u, key_max, k, cut);
        if (use_p) {
          const SmpCut base = cut;
          smp_top_p(C, w, base, key_max, (double)p, cut);
        }
        break;
      }
      const int got = smp_collect(C, lo, m);
      if (got > 0 && got <= kSmpList && (lo == xb || (long long)got >= k)) {
        if (rank == 0) {
          const SmpPick pick = smp_pick(S, w, got, cut.key, use_k ? k : 0,
                                        use_p ? (double)p : 1.0, -1.0, 0.0, 0.0, nullptr);
          smp_draw_list<E>(S, a, w, r, got, pick, u);
        }
        return;  // drawn; nothing of another CTA is read any more
      }
      // min-p alone keeps a long prefix: its threshold is the cut
      next = use_k ? kKeys : use_p ? kDeep : kRow;
    }
    if (cut.ties > 0) tie_w = w(unmono(cut.key));
  }
  if (bad) {  // the segments' masses are not known yet
    if (cut.ties > 0)
      smp_segment<false, true>(C, w, cut);
    else
      smp_segment<false, false>(C, w, cut);
    cl.sync();
  }
  smp_draw_row<E>(C, a, w, cut, tie_w, r, u);
  cl.sync();
}

}  // namespace fh

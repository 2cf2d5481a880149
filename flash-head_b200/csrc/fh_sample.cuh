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
// w-th contiguous segment of the row. A threshold is found by splitting the
// key range into 16 bands per pass (each thread sums counts and masses in
// bands of its own in shared memory, no atomics) and descending into the band
// that holds the target. The draw sums the kept mass per segment, finds the
// segment, and scans that one.
#pragma once

#include <cooperative_groups.h>

#include "fh_fused.cuh"

namespace fh {

constexpr int kSmpThreads = 512;
constexpr int kSmpWarps = kSmpThreads / 32;
constexpr int kSmpBands = 16;
constexpr int kSmpMaxCluster = 8;

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

struct SmpShared {
  double band_mass[kSmpBands][kSmpThreads];
  uint32_t band_cnt[kSmpBands][kSmpThreads];
  // values exchanged between the CTAs of a cluster, double-buffered so that
  // one cluster barrier per exchange is enough
  double x_mass[2][kSmpBands];
  unsigned long long x_cnt[2][kSmpBands];
  double warp_d[kSmpWarps + 1];
  int warp_i[kSmpWarps + 1];
  float warp_f[kSmpWarps];
  int best;
  int last;
};

// Order of the logits: monotone in x, with -0 equal to +0.
__device__ __forceinline__ uint32_t smp_key(float x) { return mono(x + 0.0f); }

template <typename E>
struct SmpElem;
template <>
struct SmpElem<float> {
  static constexpr int kVec = 4;
  __device__ __forceinline__ static float one(const float *p) { return __ldg(p); }
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
  __device__ __forceinline__ static float one(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
  __device__ __forceinline__ static void unpack(const uint4 &v, float *f) {
    Vec<__nv_bfloat16>::to_float(v, f);
  }
};
template <>
struct SmpElem<__half> {
  static constexpr int kVec = 8;
  __device__ __forceinline__ static float one(const __half *p) { return __half2float(*p); }
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
    nv = (n + mis + kVec - 1) / kVec;
  }
  __device__ __forceinline__ int column(int v) const { return v * kVec - mis; }
  __device__ __forceinline__ void load(int v, float *f) const {
    const int c0 = column(v);
    if (c0 >= 0 && c0 + kVec <= n) {
      SmpElem<E>::unpack(__ldg(reinterpret_cast<const uint4 *>(p + c0)), f);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        f[i] = c0 + i >= 0 && c0 + i < n ? SmpElem<E>::one(p + c0 + i) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) f[i] = f[i] == f[i] ? f[i] : -INFINITY;
  }
};

// Mass of a logit relative to the row's largest. With +inf in the row, the
// +inf entries share all the mass.
struct SmpMass {
  double m, c;
  bool inf;
  __device__ __forceinline__ double operator()(float x) const {
    return inf ? (x == INFINITY ? 1.0 : 0.0) : exp2(((double)x - m) * c);
  }
};

// A prefix of the order: keys above `key`, and the first `ties` equal ones.
struct SmpCut {
  uint32_t key;
  long long ties;
};

template <typename E>
struct SmpCtx {
  SmpRow<E> row;
  SmpShared &S;
  int rank, size;  // CTA in its cluster
  int v0, v1;      // this warp's segment
  int phase;       // exchanges so far
  int tid, warp, lane;
};

// Sums S.x_*[phase & 1][0..n) over the cluster's CTAs, in rank order.
template <typename E>
__device__ __forceinline__ void smp_exchange(SmpCtx<E> &C, int n, double *mass,
                                             unsigned long long *cnt) {
  namespace cg = cooperative_groups;
  cg::cluster_group cl = cg::this_cluster();
  const int b = C.phase & 1;
  ++C.phase;
  cl.sync();
  for (int i = 0; i < n; ++i) {
    double d = 0.0;
    unsigned long long k = 0ull;
    for (int r = 0; r < C.size; ++r) {
      const SmpShared *R = cl.map_shared_rank(&C.S, r);
      d += R->x_mass[b][i];
      k += R->x_cnt[b][i];
    }
    mass[i] = d;
    cnt[i] = k;
  }
}

// Counts and masses of the 16 bands [lo + (i << shift), ...) up to hi of the
// entries of the base prefix (ties of base.key count fully here: the caller
// corrects them). MASS: masses too.
template <bool MASS, typename E>
__device__ __forceinline__ void smp_bands(SmpCtx<E> &C, const SmpMass &w, uint32_t lo, uint32_t hi,
                                          int shift, double *mass, unsigned long long *cnt) {
  constexpr int kVec = SmpRow<E>::kVec;
  SmpShared &S = C.S;
#pragma unroll
  for (int i = 0; i < kSmpBands; ++i) {
    if (MASS) S.band_mass[i][C.tid] = 0.0;
    S.band_cnt[i][C.tid] = 0u;
  }
  for (int v = C.v0 + C.lane; v < C.v1; v += 32) {
    float f[kVec];
    C.row.load(v, f);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const uint32_t k = smp_key(f[i]);
      if (k >= lo && k <= hi) {
        const int b = (int)((k - lo) >> shift);
        S.band_cnt[b][C.tid] += 1u;
        if (MASS) S.band_mass[b][C.tid] += w(f[i]);
      }
    }
  }
  __syncthreads();
  // warp b sums band b
  {
    double d = 0.0;
    unsigned long long k = 0ull;
    for (int i = C.lane; i < kSmpThreads; i += 32) {
      if (MASS) d += S.band_mass[C.warp][i];
      k += S.band_cnt[C.warp][i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      d += __shfl_xor_sync(0xFFFFFFFFu, d, o);
      k += __shfl_xor_sync(0xFFFFFFFFu, k, o);
    }
    if (C.lane == 0) {
      S.x_mass[C.phase & 1][C.warp] = d;
      S.x_cnt[C.phase & 1][C.warp] = k;
    }
  }
  smp_exchange(C, kSmpBands, mass, cnt);
}

__device__ __forceinline__ int smp_shift(uint32_t lo, uint32_t hi) {
  const uint32_t span = hi - lo;
  const int bits = 32 - __clz(span);
  return bits > 4 ? bits - 4 : 0;
}

// First k entries: the key of the k-th largest and how many of its ties.
// Returns false (cut unchanged) when there are fewer than k keys in [lo, hi].
template <typename E>
__device__ __forceinline__ bool smp_top_k(SmpCtx<E> &C, const SmpMass &w, uint32_t lo, uint32_t hi,
                                          long long k, SmpCut &cut) {
  unsigned long long above = 0ull;
  for (int pass = 0; pass < 9; ++pass) {
    double mass[kSmpBands];
    unsigned long long cnt[kSmpBands];
    const int shift = smp_shift(lo, hi);
    smp_bands<false>(C, w, lo, hi, shift, mass, cnt);
    int b = kSmpBands - 1;
    for (; b >= 0; --b) {
      if (above + cnt[b] >= (unsigned long long)k) break;
      above += cnt[b];
    }
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

// Shortest prefix of the base prefix with mass >= p * (its mass).
template <typename E>
__device__ __forceinline__ void smp_top_p(SmpCtx<E> &C, const SmpMass &w, const SmpCut &base,
                                          uint32_t key_max, double p, SmpCut &cut) {
  // the base's ties enter as one more band below its other keys
  const double tie_w = base.ties > 0 ? w(unmono(base.key)) : 0.0;
  double above = 0.0, target = 0.0;
  uint32_t lo = base.key + 1u, hi = key_max;
  if (lo > hi) {  // only ties of one key
    target = p * ((double)base.ties * tie_w);
    double n = ceil(target / tie_w);
    cut.key = base.key;
    cut.ties = n < 1.0 ? 1 : n > (double)base.ties ? base.ties : (long long)n;
    return;
  }
  for (int pass = 0; pass < 9; ++pass) {
    double mass[kSmpBands];
    unsigned long long cnt[kSmpBands];
    const int shift = smp_shift(lo, hi);
    smp_bands<true>(C, w, lo, hi, shift, mass, cnt);
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
      const double n = ceil((target - above) / tie_w);
      cut.key = base.key;
      cut.ties = n < 1.0 ? 1 : n > (double)base.ties ? base.ties : (long long)n;
      return;
    }
    if (b < 0) {  // rounding: the target is the whole band's mass
      b = lowest;
      above = before;
    }
    const uint32_t nlo = lo + ((uint32_t)b << shift);
    if (shift == 0) {
      const double wt = w(unmono(nlo));
      const double n = wt > 0.0 ? ceil((target - above) / wt) : 1.0;
      cut.key = nlo;
      cut.ties = n < 1.0 ? 1 : n > (double)cnt[b] ? (long long)cnt[b] : (long long)n;
      return;
    }
    hi = nlo + min(hi - nlo, (1u << shift) - 1u);
    lo = nlo;
  }
}

// Smallest key whose mass is at least min_p (at most the largest entry's).
__device__ __forceinline__ uint32_t smp_min_key(const SmpMass &w, float m, float min_p) {
  const uint32_t top = smp_key(m);
  if (w.inf) return top;
  const double t = log2((double)min_p);
  auto enough = [&](uint32_t k) { return ((double)unmono(k) - w.m) * w.c >= t; };
  // bisect the keys; the border's rounded value is nearly always within a step
  uint32_t lo = smp_key(-INFINITY), hi = top;  // lo: too little, hi: enough
  const uint32_t g = smp_key((float)fmin((double)m, w.m + t / w.c));
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

template <typename E>
__global__ void __launch_bounds__(kSmpThreads) k_sample(SampleArgs a) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) unsigned char smp_raw[];
  SmpShared &S = *reinterpret_cast<SmpShared *>(smp_raw);
  cg::cluster_group cl = cg::this_cluster();
  constexpr int kVec = SmpRow<E>::kVec;
  const int size = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int r = blockIdx.x / size;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const SmpRow<E> row(reinterpret_cast<const E *>(a.logits) + (long long)r * a.stride, a.n);
  const int gw = rank * kSmpWarps + warp, warps = size * kSmpWarps;
  SmpCtx<E> C{row, S, rank, size, (int)((long long)row.nv * gw / warps),
              (int)((long long)row.nv * (gw + 1) / warps), 0, tid, warp, lane};

  float T = a.temperature ? a.temperature[r] : a.temperature0;
  const long long k = a.top_k ? a.top_k[r] : a.top_k0;
  const float p = a.top_p ? a.top_p[r] : a.top_p0;
  const float mp = a.min_p ? a.min_p[r] : a.min_p0;
  const bool greedy = !(T > 0.f);
  if (greedy) T = 1.f;

  // the row's largest logit
  float m = -INFINITY;
  for (int v = C.v0 + lane; v < C.v1; v += 32) {
    float f[kVec];
    row.load(v, f);
#pragma unroll
    for (int i = 0; i < kVec; ++i) m = fmaxf(m, f[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  if (lane == 0) S.warp_f[warp] = m;
  cl.sync();
  m = -INFINITY;
  for (int q = 0; q < size; ++q) {
    const SmpShared *R = cl.map_shared_rank(&S, q);
    for (int i = 0; i < kSmpWarps; ++i) m = fmaxf(m, R->warp_f[i]);
  }
  const uint32_t key_none = smp_key(-INFINITY);
  if (m == -INFINITY) {  // nothing left in this row
    if (rank == 0 && tid == 0) {
      a.out[r] = -1;
      if (a.prob) a.prob[r] = 0.f;
    }
    cl.sync();
    return;
  }
  const SmpMass w{(double)m, 1.4426950408889634 / (double)T, m == INFINITY};
  const uint32_t key_max = smp_key(m);

  SmpCut cut{key_none, 0};
  if (greedy || k == 1 || p <= 0.f) {
    cut.key = key_max;
    cut.ties = 1;
  } else {
    if (mp > 0.f) cut.key = smp_min_key(w, m, fminf(mp, 1.f)) - 1u;
    if (k > 0 && k < a.n) smp_top_k(C, w, cut.key + 1u, key_max, k, cut);
    if (p < 1.f) {
      const SmpCut base = cut;
      smp_top_p(C, w, base, key_max, (double)p, cut);
    }
  }

  // kept mass and ties of this warp's segment
  double sum = 0.0;
  int ties = 0;
  for (int v = C.v0 + lane; v < C.v1; v += 32) {
    float f[kVec];
    row.load(v, f);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const uint32_t key = smp_key(f[i]);
      if (key > cut.key) sum += w(f[i]);
      ties += key == cut.key;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    ties += __shfl_xor_sync(0xFFFFFFFFu, ties, o);
  }
  if (lane == 0) {
    S.warp_d[warp] = sum;
    S.warp_i[warp] = ties;
  }
  cl.sync();
  // every thread of every CTA finds the segment of the draw
  const double tie_w = cut.ties > 0 ? w(unmono(cut.key)) : 0.0;
  double total = 0.0;
  long long left = cut.ties;
  for (int q = 0; q < size; ++q) {
    const SmpShared *R = cl.map_shared_rank(&S, q);
    for (int i = 0; i < kSmpWarps; ++i) {
      const long long t = min(left, (long long)R->warp_i[i]);
      left -= t;
      total += R->warp_d[i] + (double)t * tie_w;
    }
  }
  double u = a.uniforms[r];
  u = u > 0.0 ? u : 0.0;
  double target = u * total;
  int seg = -1;
  double seg_before = 0.0, run = 0.0;
  long long seg_left = 0;
  left = cut.ties;
  bool found = false;
  for (int q = 0; q < size; ++q) {
    const SmpShared *R = cl.map_shared_rank(&S, q);
    for (int i = 0; i < kSmpWarps; ++i) {
      const long long t = min(left, (long long)R->warp_i[i]);
      const double mass = R->warp_d[i] + (double)t * tie_w;
      if (!found && mass > 0.0) {  // the last one stays if rounding skips them all
        seg = q * kSmpWarps + i;
        seg_before = run;
        seg_left = left;
      }
      run += mass;
      left -= t;
      found = run > target;
    }
  }
  if (seg / kSmpWarps == rank) {
    const int sv0 = (int)((long long)row.nv * seg / warps);
    const int sv1 = (int)((long long)row.nv * (seg + 1) / warps);
    const int per = (sv1 - sv0 + kSmpThreads - 1) / kSmpThreads;
    const int a0 = min(sv1, sv0 + tid * per), a1 = min(sv1, a0 + per);
    double d = 0.0;
    int t = 0;
    for (int v = a0; v < a1; ++v) {
      float f[kVec];
      row.load(v, f);
#pragma unroll
      for (int i = 0; i < kVec; ++i) t += smp_key(f[i]) == cut.key;
    }
    int t_total;
    __shared__ int scan_i[33];
    const int t_before = block_exclusive_scan(t, scan_i, &t_total);
    long long lft = seg_left - t_before;
    for (int v = a0; v < a1; ++v) {
      float f[kVec];
      row.load(v, f);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const uint32_t key = smp_key(f[i]);
        bool keep = key > cut.key;
        if (key == cut.key) keep = lft-- > 0;
        if (keep) d += w(f[i]);
      }
    }
    // exclusive prefix of the threads' masses
    double inc = d;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += x;
    }
    __shared__ double scan_d[kSmpWarps];
    if (lane == 31) scan_d[warp] = inc;
    if (tid == 0) {
      S.best = 0x7FFFFFFF;
      S.last = -1;
    }
    __syncthreads();
    double before = seg_before;
    for (int i = 0; i < warp; ++i) before += scan_d[i];
    before += inc - d;
    lft = seg_left - t_before;
    int best = 0x7FFFFFFF, last = -1;
    for (int v = a0; v < a1; ++v) {
      float f[kVec];
      row.load(v, f);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const uint32_t key = smp_key(f[i]);
        bool keep = key > cut.key;
        if (key == cut.key) keep = lft-- > 0;
        if (keep) {
          const double x = w(f[i]);
          before += x;
          const int col = row.column(v) + i;
          if (x > 0.0) last = col;
          if (before > target && col < best) best = col;
        }
      }
    }
    if (best != 0x7FFFFFFF) atomicMin(&S.best, best);
    if (last >= 0) atomicMax(&S.last, last);
    __syncthreads();
    if (tid == 0) {
      // past the end by rounding: the last kept column
      const int col = S.best != 0x7FFFFFFF ? S.best : S.last;
      a.out[r] = a.ids ? (int64_t)a.ids[(long long)r * a.ids_stride + col] : (int64_t)col;
      if (a.prob) {
        const float x = SmpElem<E>::one(row.p + col);
        a.prob[r] = (float)(w(x) / total);
      }
    }
  }
  cl.sync();
}

}  // namespace fh

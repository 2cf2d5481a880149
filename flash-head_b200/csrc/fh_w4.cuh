// Products with a 4-bit head weight: w[v, k] = (q[v, k] - z[v, g]) * s[v, g],
// q in 0..15, g = k / group_size. The products
//   out[b, v] = sum_g s[v, g] * sum_{k in g} (q[v, k] - z[v, g]) * h[b, k]
// are formed group by group: q - z is a small integer, exact in the 16-bit
// type of the hidden states, so the tensor cores sum exact products in fp32,
// and the scale multiplies the group's fp32 sum. No weight is ever rounded to
// 16 bits.
//
// Layout (made once by the loader, flash_head/w4.py). Rows come in tiles of
// 128, columns in blocks of 128 (both padded; padding has scale 0):
//   qweight u32 [tile][block][4 quads][128 rows][4 words]: word j of quad c
//           holds columns 128 * block + 32 * j + 8 * c + e, e = 0..7, column
//           e = 2i in bits 4i..4i+3 and e = 2i+1 in bits 16+4i..19+4i.
//   scales  16-bit [tile][block][128 rows][groups per block]
//   zeros   u8, same shape (absent: every zero point is 8)
// One tile's block is 8 KB, contiguous (one bulk copy). Lane (g, c) of a warp
// reads 16 bytes of row g and 16 of row g + 8 in quad c: 128-byte runs.
// The nibble order makes (w >> 4i) & 0x000F000F a pair of neighbouring
// columns, i.e. one operand register of mma.m16n8k16 (A: 16 weight rows), and
// the 8 columns of a word are 16 contiguous bytes of a hidden row (B), so
// neither operand is shuffled. Every word lies in one group of 32 or more.
#pragma once

#include "fh_fused.cuh"

namespace fh {

constexpr int kW4Warps = 16;
#ifndef W4_AHEAD
#define W4_AHEAD 2
#endif
constexpr int kW4Ahead = W4_AHEAD;  // blocks a warp loads ahead
constexpr int kW4Block = 128;                   // columns per block
constexpr int kW4Tile = 128;                     // rows per tile
constexpr int kW4RowWords = kW4Block / 8;        // u32 of one row's block

struct W4Args {
  const uint32_t *qw;
  const void *scales;
  const uint8_t *zeros;
  int V;        // weight rows
  int D;        // columns
  int nb;       // 128-column blocks: ceil(D / 128)
  int tiles;    // 128-row tiles: ceil(V / 128)
  const void *hidden;  // [rows, D]
  int rows;
  void *out;    // [rows, ldo]
  long long ldo;
  int ksplit;   // warps that share a unit, each with every ksplit-th block
  // probed clusters (k_w4_probes)
  const int64_t *ci;  // [rows, P]
  int P, K, cap;
};

// Groups per block (128 / group size): the width of one row's scales.
template <int GPK>
struct W4Group;
template <>
struct W4Group<1> {
  using S = uint16_t;
  using Z = uint8_t;
};
template <>
struct W4Group<2> {
  using S = uint32_t;
  using Z = uint16_t;
};
template <>
struct W4Group<4> {
  using S = uint2;
  using Z = uint32_t;
};

template <int GPK>
__device__ __forceinline__ uint32_t w4_scale_bits(typename W4Group<GPK>::S s, int i);
template <>
__device__ __forceinline__ uint32_t w4_scale_bits<1>(uint16_t s, int) {
  return s;
}
template <>
__device__ __forceinline__ uint32_t w4_scale_bits<2>(uint32_t s, int i) {
  return i ? s >> 16 : s & 0xFFFFu;
}
template <>
__device__ __forceinline__ uint32_t w4_scale_bits<4>(uint2 s, int i) {
  const uint32_t w = i < 2 ? s.x : s.y;
  return (i & 1) ? w >> 16 : w & 0xFFFFu;
}

// 16-bit integer arithmetic in the float types: 128 + q (bf16) and 1024 + q
// (fp16) are exact with q in the lowest mantissa bits, and so is their
// difference to 128 + z (1024 + z).
template <typename T>
struct W4Num;
template <>
struct W4Num<__nv_bfloat16> {
  static constexpr uint32_t kMagic = 0x43004300u;
  __device__ __forceinline__ static uint32_t sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&a),
                                     *reinterpret_cast<const __nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
  }
  __device__ __forceinline__ static float scale(uint32_t bits) {
    return __uint_as_float(bits << 16);
  }
};
template <>
struct W4Num<__half> {
  static constexpr uint32_t kMagic = 0x64006400u;
  __device__ __forceinline__ static uint32_t sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&a),
                              *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
  }
  __device__ __forceinline__ static float scale(uint32_t bits) {
    return __half2float(__ushort_as_half((unsigned short)bits));
  }
};

// The four pairs of a word as T x 2 of q - z; zz = magic + z in both halves.
template <typename T>
__device__ __forceinline__ void w4_unpack(uint32_t w, uint32_t zz, uint32_t (&p)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    p[i] = W4Num<T>::sub(((w >> (4 * i)) & 0x000F000Fu) | W4Num<T>::kMagic, zz);
}

// One warp's share of a 16-row block: the words, scales and zero points of
// rows g and g + 8.
template <int GPK, bool ZP>
struct W4Frag {
  uint4 q[2];
  typename W4Group<GPK>::S s[2];
  typename W4Group<GPK>::Z z[2];
};

// First word of a row's quad; i counts rows in [tile][block][row] order.
__device__ __forceinline__ long long w4_word(long long i, int c) {
  return ((i >> 7) * (4 * kW4Tile) + c * kW4Tile + (i & (kW4Tile - 1))) * 4;
}

template <int GPK, bool ZP>
__device__ __forceinline__ void w4_load(const W4Args &a, int kb, int r0, int r1, int c,
                                        W4Frag<GPK, ZP> &f) {
  using S = typename W4Group<GPK>::S;
  using Z = typename W4Group<GPK>::Z;
  // row of the [tile][block][row] order
  const long long i0 = ((long long)(r0 >> 7) * a.nb + kb) * kW4Tile + (r0 & 127);
  const long long i1 = ((long long)(r1 >> 7) * a.nb + kb) * kW4Tile + (r1 & 127);
  f.q[0] = ldg_stream(a.qw + w4_word(i0, c));
  f.q[1] = ldg_stream(a.qw + w4_word(i1, c));
  const S *s = reinterpret_cast<const S *>(a.scales);
  f.s[0] = __ldg(s + i0);
  f.s[1] = __ldg(s + i1);
  if (ZP) {
    const Z *z = reinterpret_cast<const Z *>(a.zeros);
    f.z[0] = __ldg(z + i0);
    f.z[1] = __ldg(z + i1);
  }
}

// acc += the block's products; hb points at the lane's 16 bytes of hidden
// column n = lane / 4 (this block, quad c) and hstride is the distance, in
// bytes, of the next 8 columns of B. LOAD reads 16 bytes of hidden states.
template <typename T, int GPK, bool ZP, int NT, typename Load>
__device__ __forceinline__ void w4_block(const W4Frag<GPK, ZP> &f, Load load, float (&acc)[NT][4]) {
  constexpr int JG = 4 / GPK;  // words per group
#pragma unroll
  for (int gi = 0; gi < GPK; ++gi) {
    uint32_t zz0, zz1;
    if (ZP) {
      const uint32_t z0 = ((uint32_t)f.z[0] >> (8 * gi)) & 0xFFu;
      const uint32_t z1 = ((uint32_t)f.z[1] >> (8 * gi)) & 0xFFu;
      zz0 = W4Num<T>::kMagic | (z0 * 0x00010001u);
      zz1 = W4Num<T>::kMagic | (z1 * 0x00010001u);
    } else {
      zz0 = zz1 = W4Num<T>::kMagic | 0x00080008u;
    }
    float part[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[n][i] = 0.f;
#pragma unroll
    for (int jj = 0; jj < JG; ++jj) {
      const int j = gi * JG + jj;
      const uint32_t w0 = j == 0 ? f.q[0].x : j == 1 ? f.q[0].y : j == 2 ? f.q[0].z : f.q[0].w;
      const uint32_t w1 = j == 0 ? f.q[1].x : j == 1 ? f.q[1].y : j == 2 ? f.q[1].z : f.q[1].w;
      uint32_t p0[4], p1[4];
      w4_unpack<T>(w0, zz0, p0);
      w4_unpack<T>(w1, zz1, p1);
      const uint32_t a0[4] = {p0[0], p1[0], p0[1], p1[1]};
      const uint32_t a1[4] = {p0[2], p1[2], p0[3], p1[3]};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 h = load(n, j);
        const uint32_t b0[2] = {h.x, h.y}, b1[2] = {h.z, h.w};
        mma16816<T>(part[n], a0, b0);
        mma16816<T>(part[n], a1, b1);
      }
    }
    const float s0 = W4Num<T>::scale(w4_scale_bits<GPK>(f.s[0], gi));
    const float s1 = W4Num<T>::scale(w4_scale_bits<GPK>(f.s[1], gi));
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      acc[n][0] = fmaf(s0, part[n][0], acc[n][0]);
      acc[n][1] = fmaf(s0, part[n][1], acc[n][1]);
      acc[n][2] = fmaf(s1, part[n][2], acc[n][2]);
      acc[n][3] = fmaf(s1, part[n][3], acc[n][3]);
    }
  }
}

// Hidden rows in shared memory, 64 bytes of padding per row: the 8 lanes of a
// 128-byte phase of a 16-byte load (2 rows x 4 quads) then hit all 32 banks.
__host__ __device__ inline int w4_row_bytes(int nb) { return nb * kW4Block * 2 + 64; }
__host__ __device__ inline size_t w4_mv_smem_bytes(int nb, int nt) {
  // hidden rows, then the partial sums of the warps that share a unit
  return (size_t)(8 * nt) * w4_row_bytes(nb) + (size_t)kW4Warps * nt * 32 * 8 * sizeof(float);
}

// Dense form for up to 8 * NT hidden rows: one persistent CTA per SM, 16
// warps; a unit is 32 weight rows, taken by ksplit warps (each every
// ksplit-th block of 128 columns). Units go to CTAs round-robin, so every SM
// reads the same share of the weight.
template <typename T, int GPK, bool ZP, int NT>
__global__ void __launch_bounds__(32 * kW4Warps, 1) k_w4_mv(W4Args a) {
  extern __shared__ __align__(16) unsigned char w4_sm[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  const int rb = w4_row_bytes(a.nb);
  // hidden states, zero past the last row and the last column
  {
    const int chunks = a.nb * 16;  // 16-byte chunks of a row
    const int valid = a.D / 8;     // D is a multiple of 32
    for (int i = tid; i < 8 * NT * chunks; i += 32 * kW4Warps) {
      const int r = i / chunks, x = i - r * chunks;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (r < a.rows && x < valid)
        v = ldg_keep(reinterpret_cast<const uint4 *>(a.hidden) + (size_t)r * valid + x);
      *reinterpret_cast<uint4 *>(w4_sm + (size_t)r * rb + x * 16) = v;
    }
  }
  __syncthreads();
  float *red = reinterpret_cast<float *>(w4_sm + (size_t)(8 * NT) * rb);
  const unsigned char *hl = w4_sm + (size_t)g * rb + c * 16;

  const int ks = a.ksplit, kw = warp % ks;
  const int team = warp / ks, teams = kW4Warps / ks;
  const int units = a.tiles * (kW4Tile / 32);
  const int per_round = teams * gridDim.x;
  const int my_nb = (a.nb - kw + ks - 1) / ks;  // blocks of this warp
  const int rounds = (units + per_round - 1) / per_round;
  const int first = team * gridDim.x + blockIdx.x;

  // the warp's blocks, unit after unit, are loaded kW4Ahead steps ahead
  W4Frag<GPK, ZP> f[kW4Ahead][2];
  int l_round = 0, l_b = 0;
  auto fetch = [&](W4Frag<GPK, ZP>(&x)[2]) {
    if (l_round < rounds) {
      const int u = min(first + l_round * per_round, units - 1), kb = kw + l_b * ks;
#pragma unroll
      for (int t = 0; t < 2; ++t)
        w4_load<GPK, ZP>(a, kb, 32 * u + 16 * t + g, 32 * u + 16 * t + g + 8, c, x[t]);
      if (++l_b == my_nb) {
        l_b = 0;
        ++l_round;
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kW4Ahead; ++i) fetch(f[i]);
  float acc[2][NT][4];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[t][n][i] = 0.f;

  const int steps = rounds * my_nb;
  for (int step0 = 0, b = 0, round = 0; step0 < steps; step0 += kW4Ahead) {
#pragma unroll
   for (int ahead = 0; ahead < kW4Ahead; ++ahead) {
    if (step0 + ahead >= steps) break;
    const int kb = kw + b * ks;
    const unsigned char *hk = hl + kb * (kW4Block * 2);
    auto load = [&](int n, int j) { return lds128(hk + (size_t)(8 * n) * rb + j * 64); };
#pragma unroll
    for (int t = 0; t < 2; ++t) w4_block<T, GPK, ZP, NT>(f[ahead][t], load, acc[t]);
    fetch(f[ahead]);
    if (++b < my_nb) continue;
    b = 0;
    const int u = first + round * per_round;
    const bool live = u < units;
    ++round;
    if (ks > 1) {
      // sum the team's partial sums, warp kw = 0 keeps them (fixed order)
      float *mine = red + (size_t)warp * NT * 32 * 8 + lane * (8 * NT);
      if (live && kw > 0) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            *reinterpret_cast<float4 *>(mine + (t * NT + n) * 4) =
                make_float4(acc[t][n][0], acc[t][n][1], acc[t][n][2], acc[t][n][3]);
      }
      __syncthreads();
      if (live && kw == 0) {
        for (int o = 1; o < ks; ++o) {
          const float *other = mine + (size_t)o * NT * 32 * 8;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const float4 v = *reinterpret_cast<const float4 *>(other + (t * NT + n) * 4);
              acc[t][n][0] += v.x;
              acc[t][n][1] += v.y;
              acc[t][n][2] += v.z;
              acc[t][n][3] += v.w;
            }
        }
      }
      __syncthreads();
    }
    if (live && kw == 0) {
      T *out = reinterpret_cast<T *>(a.out);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int v = (2 * u + t) * 16 + g + (i >> 1) * 8;
            const int r = 8 * n + 2 * c + (i & 1);
            if (v < a.V && r < a.rows) out[(long long)r * a.ldo + v] = from_float<T>(acc[t][n][i]);
          }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][n][i] = 0.f;
   }
  }
}

// Probed clusters: out[r, i * cap + s] = logit of weight row ci[r, i] * cap + s
// for hidden row r. A CTA takes 16 candidate slots of one row and its 8 warps
// share the columns. Cluster ids outside [0, K) give -inf.
constexpr int kW4ProbeWarps = 8;

template <typename T, int GPK, bool ZP>
__global__ void __launch_bounds__(32 * kW4ProbeWarps) k_w4_probes(W4Args a) {
  __shared__ float red[kW4ProbeWarps][16];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  const int n = a.P * a.cap;
  const int per_row = (n + 15) / 16;
  const int row = (int)(blockIdx.x / (unsigned)per_row);
  const int s0 = (int)(blockIdx.x - (unsigned)row * (unsigned)per_row) * 16;
  // weight rows of slots s0 + g and s0 + g + 8 (row 0 where there is none)
  int wr[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int s = s0 + g + 8 * i;
    wr[i] = 0;
    if (s < n) {
      const int p = s / a.cap;
      const int64_t cl = a.ci[(size_t)row * a.P + p];
      if (cl >= 0 && cl < a.K) wr[i] = (int)cl * a.cap + (s - p * a.cap);
    }
  }
  const uint4 *h = reinterpret_cast<const uint4 *>(a.hidden) + (size_t)row * (a.D / 8);
  float acc[1][4] = {{0.f, 0.f, 0.f, 0.f}};
  for (int kb = warp; kb < a.nb; kb += kW4ProbeWarps) {
    W4Frag<GPK, ZP> f;
    w4_load<GPK, ZP>(a, kb, wr[0], wr[1], c, f);
    // one hidden row: column n = 0 of B, the other 7 are zero
    auto load = [&](int, int j) {
      const int x = kb * 16 + j * 4 + c;
      return g == 0 && x < a.D / 8 ? ldg_keep(h + x) : make_uint4(0u, 0u, 0u, 0u);
    };
    w4_block<T, GPK, ZP, 1>(f, load, acc);
  }
  if (c == 0) {
    red[warp][g] = acc[0][0];
    red[warp][g + 8] = acc[0][2];
  }
  __syncthreads();
  if (tid < 16 && s0 + tid < n) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kW4ProbeWarps; ++w) v += red[w][tid];
    const int64_t cl = a.ci[(size_t)row * a.P + (s0 + tid) / a.cap];
    if (cl < 0 || cl >= a.K) v = -INFINITY;
    reinterpret_cast<T *>(a.out)[(size_t)row * n + s0 + tid] = from_float<T>(v);
  }
}

}  // namespace fh

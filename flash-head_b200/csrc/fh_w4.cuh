// Products with a 4-bit head weight: w[v, k] = (q[v, k] - z[v, g]) * s[v, g],
// q in 0..15, g = k / group_size. The products
//   out[b, v] = sum_g s[v, g] * sum_{k in g} (q[v, k] - z[v, g]) * h[b, k]
// are formed group by group: q - z is a small integer, exact in the 16-bit
// type of the hidden states, so the tensor cores sum exact products in fp32,
// and the scale multiplies the group's fp32 sum. No weight is ever rounded to
// 16 bits. (More than 8 rows: fh_w4_tc.cuh, fh_w4_split.cuh.)
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
constexpr int kW4Ahead = 2;  // blocks a warp loads ahead
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
  uint32_t mask, magic;  // kW4Mask and W4Num<T>::kMagic (see W4Bits)
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
    uint32_t r;  // a * 1 - b, with b's signs set by the caller
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(0x3F803F80u), "r"(b));
    return r;
  }
  __device__ __forceinline__ static float scale(uint32_t bits) {
    return __uint_as_float(bits << 16);
  }
};
template <>
struct W4Num<__half> {
  static constexpr uint32_t kMagic = 0x64006400u;
  __device__ __forceinline__ static uint32_t sub(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ __forceinline__ static uint32_t fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
  }
  __device__ __forceinline__ static float scale(uint32_t bits) {
    return __half2float(__ushort_as_half((unsigned short)bits));
  }
};

// The mask of a word's nibble pairs and the magic number, as values that the
// compiler cannot know: with both in registers (x & mask) | magic is one
// instruction, with literals it became two, and integer instructions are what
// the unpacking has most of.
constexpr uint32_t kW4Mask = 0x000F000Fu;
struct W4Bits {
  uint32_t mask, magic;
  __device__ __forceinline__ uint32_t low(uint32_t x) const {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(magic));
    return r;
  }
  __device__ __forceinline__ uint32_t high(uint32_t x, uint32_t mask16) const {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask16), "r"(magic));
    return r;
  }
};

// What turns a group's integers into q - z: -(magic + z) in both halves, and for
// fp16 also -(64 + z).
template <typename T>
struct W4Zero {
  uint32_t z, z16;
  __device__ __forceinline__ explicit W4Zero(uint32_t zero) {
    z = (W4Num<T>::kMagic | (zero * 0x00010001u)) ^ 0x80008000u;
    // 64 + z in fp16: 0x5400 is 64, a step 1/16
    z16 = (0x54005400u | (zero * 0x00100010u)) ^ 0x80008000u;
  }
};

// The four pairs of a word as T x 2 of q - z. (Integer operations bound the
// unpacking: fp16 takes the odd pairs where they stand, as 1024 + 16 q, and an
// exact fma, (1024 + 16 q) / 16 - (64 + z), so that a word is shifted once
// instead of three times; bf16 has no bits for it.)
template <typename T>
__device__ __forceinline__ void w4_unpack(uint32_t w, const W4Bits &b, const W4Zero<T> &zero,
                                          uint32_t (&p)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = W4Num<T>::sub(b.low(w >> (4 * i)), zero.z);
}
template <>
__device__ __forceinline__ void w4_unpack<__half>(uint32_t w, const W4Bits &b,
                                                  const W4Zero<__half> &zero, uint32_t (&p)[4]) {
  const uint32_t mask16 = b.mask << 4;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t x = i ? w >> 8 : w;
    p[2 * i] = W4Num<__half>::sub(b.low(x), zero.z);
    p[2 * i + 1] = W4Num<__half>::fma(b.high(x, mask16), 0x2C002C00u, zero.z16);
  }
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

// acc += the products of a block of TILES 16-row tiles; load(j) gives the 16
// bytes of hidden column lane / 4 that belong to word j of the lane's quad.
template <typename T, int GPK, bool ZP, int TILES, typename Load>
__device__ __forceinline__ void w4_block(const W4Frag<GPK, ZP> (&f)[TILES], const W4Bits &bits, Load load,
                                         float (&acc)[TILES][4]) {
  constexpr int JG = 4 / GPK;  // words per group
#pragma unroll
  for (int gi = 0; gi < GPK; ++gi) {
    float part[TILES][4];
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[t][i] = 0.f;
#pragma unroll
    for (int jj = 0; jj < JG; ++jj) {
      const int j = gi * JG + jj;
      const uint4 h = load(j);
      const uint32_t b0[2] = {h.x, h.y}, b1[2] = {h.z, h.w};
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        const uint32_t w0 = j == 0 ? f[t].q[0].x : j == 1 ? f[t].q[0].y : j == 2 ? f[t].q[0].z : f[t].q[0].w;
        const uint32_t w1 = j == 0 ? f[t].q[1].x : j == 1 ? f[t].q[1].y : j == 2 ? f[t].q[1].z : f[t].q[1].w;
        uint32_t p0[4], p1[4];
        const W4Zero<T> z0(ZP ? ((uint32_t)f[t].z[0] >> (8 * gi)) & 0xFFu : 8u);
        const W4Zero<T> z1(ZP ? ((uint32_t)f[t].z[1] >> (8 * gi)) & 0xFFu : 8u);
        w4_unpack<T>(w0, bits, z0, p0);
        w4_unpack<T>(w1, bits, z1, p1);
        const uint32_t a0[4] = {p0[0], p1[0], p0[1], p1[1]};
        const uint32_t a1[4] = {p0[2], p1[2], p0[3], p1[3]};
        mma16816<T>(part[t], a0, b0);
        mma16816<T>(part[t], a1, b1);
      }
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const float s0 = W4Num<T>::scale(w4_scale_bits<GPK>(f[t].s[0], gi));
      const float s1 = W4Num<T>::scale(w4_scale_bits<GPK>(f[t].s[1], gi));
      acc[t][0] = fmaf(s0, part[t][0], acc[t][0]);
      acc[t][1] = fmaf(s0, part[t][1], acc[t][1]);
      acc[t][2] = fmaf(s1, part[t][2], acc[t][2]);
      acc[t][3] = fmaf(s1, part[t][3], acc[t][3]);
    }
  }
}

__device__ __forceinline__ uint4 w4_lds(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(at));
  return v;
}

// Hidden rows in shared memory, 64 bytes of padding per row: the 8 lanes of a
// 128-byte phase of a 16-byte load (2 rows x 4 quads) then hit all 32 banks.
__host__ __device__ inline int w4_row_bytes(int nb) { return nb * kW4Block * 2 + 64; }
__host__ __device__ inline size_t w4_mv_smem_bytes(int nb) {
  // hidden rows, then the partial sums of the warps that share a unit
  return (size_t)8 * w4_row_bytes(nb) + (size_t)kW4Warps * 32 * 8 * sizeof(float);
}

// Dense form for up to 8 hidden rows: one persistent CTA per SM, 16
// warps; a unit is 32 weight rows, taken by ksplit warps (each every
// ksplit-th block of 128 columns). Units go to CTAs round-robin, so every SM
// reads the same share of the weight.
// Bound: no unit is full. Turning nibbles into operands, 9 to 11 instructions a word
// for half an mma, keeps the ALU pipe 56 to 61 % busy, issue 51 to 58 %, DRAM 45
// to 47 %: each of an SM's 16 warps loads, unpacks and multiplies in turn. One row of
// a 2048 x 128256 head, groups of 128 in bf16 and no zero points, 35 us (3.8
// TB/s), 8 rows of 4096 x 128256 69 us.
// mma.sync, not tcgen05: its operand is made in registers, where the words
// arrive, and a tcgen05 tile of 8 columns would wait for the same words.
template <typename T, int GPK, bool ZP>
__global__ void __launch_bounds__(32 * kW4Warps, 1) k_w4_mv(W4Args a) {
  extern __shared__ __align__(16) unsigned char w4_sm[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  const int rb = w4_row_bytes(a.nb);
  // hidden states, zero past the last row and the last column
  {
    const int chunks = a.nb * 16;  // 16-byte chunks of a row
    const int valid = a.D / 8;     // D is a multiple of 32
    for (int i = tid; i < 8 * chunks; i += 32 * kW4Warps) {
      const int r = i / chunks, x = i - r * chunks;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (r < a.rows && x < valid)
        v = ldg_keep(reinterpret_cast<const uint4 *>(a.hidden) + (size_t)r * valid + x);
      *reinterpret_cast<uint4 *>(w4_sm + (size_t)r * rb + x * 16) = v;
    }
  }
  __syncthreads();
  float *red = reinterpret_cast<float *>(w4_sm + (size_t)8 * rb);
  const W4Bits bits{a.mask, a.magic};
  const uint32_t hl = smem_u32(w4_sm) + (uint32_t)(g * rb + c * 16);

  const int ks = a.ksplit, kw = warp % ks;
  const int team = warp / ks, teams = kW4Warps / ks;
  const int units = a.tiles * (kW4Tile / 32);
  const int per_round = teams * gridDim.x;
  const int my_nb = (a.nb - kw + ks - 1) / ks;  // blocks of this warp
  const int first = team * gridDim.x + blockIdx.x;
  const int rounds = first < units ? (units - 1 - first) / per_round + 1 : 0;  // of this team

  // the warp's blocks, unit after unit, are loaded kW4Ahead steps ahead
  W4Frag<GPK, ZP> f[kW4Ahead][2];
  int l_round = 0, l_b = 0;
  using ST = typename W4Group<GPK>::S;
  using ZT = typename W4Group<GPK>::Z;
  const uint32_t *lq = nullptr;  // this lane's words, scales, zero points of the next block
  const ST *ls = nullptr;
  const ZT *lz = nullptr;
  auto fetch = [&](W4Frag<GPK, ZP>(&x)[2]) {
    if (l_round < rounds) {
      if (l_b == 0) {  // a new unit: 32 rows of a tile
        const int u = first + l_round * per_round;  // below units
        const long long blk = (long long)(u >> 2) * a.nb + kw;
        const int row = 32 * (u & 3) + g;
        lq = a.qw + blk * (kW4Tile * kW4RowWords) + (c * kW4Tile + row) * 4;
        ls = reinterpret_cast<const ST *>(a.scales) + blk * kW4Tile + row;
        if (ZP) lz = reinterpret_cast<const ZT *>(a.zeros) + blk * kW4Tile + row;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          x[t].q[i] = ldg_stream(lq + (16 * t + 8 * i) * 4);
          x[t].s[i] = __ldg(ls + 16 * t + 8 * i);
          if (ZP) x[t].z[i] = __ldg(lz + 16 * t + 8 * i);
        }
      lq += ks * (kW4Tile * kW4RowWords);
      ls += ks * kW4Tile;
      if (ZP) lz += ks * kW4Tile;
      if (++l_b == my_nb) {
        l_b = 0;
        ++l_round;
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kW4Ahead; ++i) fetch(f[i]);
  float acc[2][4];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[t][i] = 0.f;

  const int steps = rounds * my_nb;
  for (int step0 = 0, b = 0, round = 0; step0 < steps; step0 += kW4Ahead) {
#pragma unroll
   for (int ahead = 0; ahead < kW4Ahead; ++ahead) {
    if (step0 + ahead >= steps) break;
    const int kb = kw + b * ks;
    const uint32_t hk = hl + (uint32_t)(kb * (kW4Block * 2));
    auto load = [&](int j) { return w4_lds(hk + (uint32_t)(j * 64)); };
    w4_block<T, GPK, ZP, 2>(f[ahead], bits, load, acc);
    fetch(f[ahead]);
    if (++b < my_nb) continue;
    b = 0;
    const int u = first + round * per_round;
    ++round;
    if (ks > 1) {
      // sum the team's partial sums, warp kw = 0 keeps them (fixed order)
      float *mine = red + (size_t)warp * 32 * 8 + lane * 4;
      if (kw > 0) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
          *reinterpret_cast<float4 *>(mine + t * 128) =
              make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]);
      }
      nbar_sync(1 + team, 32 * ks);
      if (kw == 0) {
        for (int o = 1; o < ks; ++o) {
          const float *other = mine + (size_t)o * 32 * 8;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const float4 v = *reinterpret_cast<const float4 *>(other + t * 128);
            acc[t][0] += v.x;
            acc[t][1] += v.y;
            acc[t][2] += v.z;
            acc[t][3] += v.w;
          }
        }
      }
      nbar_sync(1 + team, 32 * ks);
    }
    if (kw == 0) {
      T *out = reinterpret_cast<T *>(a.out);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int v = (2 * u + t) * 16 + g + (i >> 1) * 8;
          const int r = 2 * c + (i & 1);
          if (v < a.V && r < a.rows) out[(long long)r * a.ldo + v] = from_float<T>(acc[t][i]);
        }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[t][i] = 0.f;
   }
  }
}

// Probed clusters: out[r, i * cap + s] = logit of weight row ci[r, i] * cap + s
// for hidden row r. A CTA takes 16 candidate slots of one row and its 8 warps
// share the columns. Cluster ids outside [0, K) give -inf.
// Bound: latency for one row, then the same pipe (60 %) and HBM sectors (29 %): a
// cluster of 16 neighbouring rows is 256 bytes in each quad of a block, and no load
// is issued ahead. 256 clusters of 16, 2048 columns,
// one row 4.7 us; 4096 columns with zero points, 12 rows 40 us (2.7 TB/s of the
// words, scales and zero points of every row's own clusters).
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
    W4Frag<GPK, ZP> f[1];
    w4_load<GPK, ZP>(a, kb, wr[0], wr[1], c, f[0]);
    // one hidden row: column n = 0 of B, the other 7 are zero
    auto load = [&](int j) {
      const int x = kb * 16 + j * 4 + c;
      return g == 0 && x < a.D / 8 ? ldg_keep(h + x) : make_uint4(0u, 0u, 0u, 0u);
    };
    w4_block<T, GPK, ZP, 1>(f, W4Bits{a.mask, a.magic}, load, acc);
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

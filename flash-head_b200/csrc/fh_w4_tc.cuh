// Logits of a 4-bit head for many rows on the 5th-generation tensor cores:
// out[b, v] = sum_k w[v, k] h[b, k], M = 128 weight rows, N = up to 256 hidden
// rows per launch.
//
// The weight's integers become f16 operands: q - z is exact,
// and its product with the group's scale is rounded to f16 once, 2^-11 relative
// (a bf16 scale times a 4-bit integer has at most one bit more than f16 holds).
// That is an eighth of a bf16 output's own rounding; applying the scales to
// fp32 sums instead, as k_w4_mv does, would read every accumulator back once
// per group. Rows of scales are brought to [1, 2) by an exact power of two
// (row_mul), undone in the epilogue, so that no weight leaves f16's range. bf16
// hidden rows are copied to f16 first, each scaled by a power of two likewise
// (k_w4_hidden); f16 ones are read as they are.
//
// The unpacked operand goes to tensor memory, not to shared memory: 16 KB
// written and 16 KB read per 128 x 64 tile were most of the shared-memory
// traffic that bound a first version (64 rows of a 1536 x 151936 head: 92 us).
//
// One persistent CTA per SM, 24 warps:
//   warp 0      lane 0 brings the packed blocks (8 KB of words, the scales and
//               zero points of 128 rows x 128 columns: two or three bulk copies)
//               into a ring of their own, deep enough to keep HBM busy;
//   warp 2      lane 0 brings the hidden tiles of every 128 columns (TMA, two of 64
//               with the 128-byte swizzle) into the stages (a thread of its own: a wait that
//               suspends the one for packed slots must not hold up these);
//   warp 1      allocates TMEM; one lane issues tcgen05.mma (K = 16), 8 per
//               stage, A from tensor memory, B from shared memory;
//   warps 4-19  unpack, in four groups of 4 on successive blocks: a thread has one
//               weight row, i.e. one TMEM lane, reads its 64 bytes of the block
//               and stores 32 columns' pairs (16 TMEM columns) at a time;
//   warps 20-23 epilogue: a thread has one weight row and all hidden rows; up to
//               128 hidden rows the accumulators are double-buffered.
// Bounds: unpacking next to HBM (the packed weight) up to about 64 rows: 64 rows
// of a 1536 x 151936 head 43 us (2.8 TB/s); the tensor cores and the hidden
// tiles' way from L2 at 256: 2048 x 128256 112 us (1.2 PFLOP/s).
// Every wait is bounded; on a timeout the kernel records kErrCopyTimeout,
// drains its own copies and MMAs (bounded) and frees TMEM before it returns.
#pragma once

#include "fh_s1_tc.cuh"
#include "fh_w4.cuh"

namespace fh {

constexpr int kW4tConvWarps = 4;  // unpack one block together, a TMEM quadrant each
constexpr int kW4tGroups = 4;     // of such warps, on successive blocks (a launch may use fewer)
constexpr int kW4tEpiWarps = 4;
constexpr int kW4tFirstConv = 4;  // warp
constexpr int kW4tEpi = kW4tFirstConv + kW4tGroups * kW4tConvWarps;
constexpr int kW4tThreads = 32 * (kW4tFirstConv + kW4tGroups * kW4tConvWarps + kW4tEpiWarps);
constexpr int kW4tMaxN = 256;
constexpr int kW4tMaxStages = 4;
constexpr int kW4tACols = 64;  // TMEM columns of a stage's A tile: 128 f16 per row
constexpr int kW4tMaxPacked = 12;
constexpr int kW4tSmemMax = 227 * 1024;

struct W4TcArgs {
  const uint32_t *qw;
  const void *scales;
  const uint8_t *zeros;
  const float *row_mul;   // [128 * tiles] powers of two
  const float *row_fac;   // [rows] factors of the hidden rows, or null
  int V, D, nb;
  int tiles;
  int rows, n_pad;
  int stages, packed, n_acc, groups;
  int tmem_cols;
  int vec;                // outputs take 16-byte stores (V, ldo and out allow them)
  uint32_t idesc;
  uint32_t mask, magic;   // kW4Mask, W4Num<__half>::kMagic
  void *out;
  long long ldo;
  uint32_t *err;
  uint32_t polls;
};

struct W4TcCtrl {
  uint64_t full[kW4tMaxStages];    // hidden tile landed and A tile written
  uint64_t empty[kW4tMaxStages];   // MMAs done
  uint64_t pfull[kW4tMaxPacked];   // packed block landed
  uint64_t pempty[kW4tMaxPacked];  // packed block unpacked
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t drain;
  uint32_t tmem_base;
  uint32_t s_err;
  alignas(16) float fac[kW4tMaxN];
  uint4 out[kW4tEpiWarps][128];  // 32 hidden rows x 32 weight rows, 16-bit
};

// Groups that may run. A group steps over the others' blocks, so that it knows of
// a barrier's progress only what the order of the work implies; a parity wait
// is unambiguous while the phase before the awaited one is known to be
// complete. Having written block n, a group knows the MMAs up to block
// n - stages, and with them the packed blocks up to there, to be done. Its next
// block n + groups needs the stage's use two rounds back, n + groups - 2 stages,
// and the packed slot's fill one round back, n + groups - packed, among them.
__host__ __device__ inline int w4t_groups(int stages, int packed) {
  int g = kW4tGroups;
  while (g > 0 && (g > stages || packed < g + stages)) --g;
  return g;
}

__host__ __device__ inline int w4t_packed_bytes(int gpk, bool zp) {
  return kW4Tile * kW4RowWords * 4 + kW4Tile * gpk * (zp ? 3 : 2);
}
__host__ __device__ inline size_t w4t_stage_bytes(int n_pad) {
  return (size_t)n_pad * 256;  // two tiles of 64 hidden columns
}
__host__ __device__ inline size_t w4t_smem_bytes(int n_pad, int stages, int packed, int gpk, bool zp) {
  return 1024 + stages * w4t_stage_bytes(n_pad) + (size_t)packed * w4t_packed_bytes(gpk, zp) +
         sizeof(W4TcCtrl);
}

// mbar_wait and tc_commit by shared-memory address.
__device__ __forceinline__ bool w4t_wait(uint32_t bar, uint32_t parity, uint32_t polls) {
  for (uint32_t i = 0; i < polls; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  return false;
}
__device__ __forceinline__ void w4t_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   bar)
               : "memory");
}

__device__ __forceinline__ bool w4t_elect() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}"
               : "=r"(p));
  return p != 0;
}
// D += A . B with A in tensor memory: row m in lane m, two f16 per column.
__device__ __forceinline__ void w4t_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 16 columns of this warp's 32 lanes, a register each.
__device__ __forceinline__ void w4t_st16(uint32_t addr, const uint32_t (&x)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]),
      "r"(x[8]), "r"(x[9]), "r"(x[10]), "r"(x[11]), "r"(x[12]), "r"(x[13]), "r"(x[14]), "r"(x[15])
      : "memory");
}

// f16 copy of bf16 hidden rows, one CTA per row: the row's largest finite
// magnitude is brought to [2^14, 2^15) by a power of two whose inverse goes to
// fac. Infinities and NaN stay. Also clears the error word.
__global__ void __launch_bounds__(256)
    k_w4_hidden(const uint4 *h, uint4 *out, float *fac, int chunks, uint32_t *err) {
  __shared__ uint32_t top[8];
  grid_dep_launch();
  const uint4 *src = h + (size_t)blockIdx.x * chunks;
  uint32_t m = 0u;  // largest finite magnitude, bf16 bits
  for (int i = threadIdx.x; i < chunks; i += 256) {
    const uint4 v = src[i];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = w[j] & 0x7FFFu, hi = (w[j] >> 16) & 0x7FFFu;
      if (lo < 0x7F80u) m = max(m, lo);
      if (hi < 0x7F80u) m = max(m, hi);
    }
  }
  m = __reduce_max_sync(0xFFFFFFFFu, m);
  if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, top[i]);
  // exponent of the largest value (a zero or subnormal row counts as 2^-126)
  const int e = max((int)(m >> 7), 1) - 127;
  // 2^(14 - e) in two factors: it may pass the largest fp32
  const int s0 = (14 - e) / 2, s1 = 14 - e - s0;
  const float f0 = __uint_as_float((uint32_t)(127 + s0) << 23);
  const float f1 = __uint_as_float((uint32_t)(127 + s1) << 23);
  uint4 *dst = out + (size_t)blockIdx.x * chunks;
  for (int i = threadIdx.x; i < chunks; i += 256) {
    const uint4 v = src[i];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float lo = __uint_as_float(w[j] << 16) * f0 * f1;
      const float hi = __uint_as_float(w[j] & 0xFFFF0000u) * f0 * f1;
      const __half2 x = __floats2half2_rn(lo, hi);
      o[j] = *reinterpret_cast<const uint32_t *>(&x);
    }
    dst[i] = make_uint4(o[0], o[1], o[2], o[3]);
  }
  if (threadIdx.x == 0) {
    // the inverse, 2^(e - 14): may be subnormal as one factor, never zero
    fac[blockIdx.x] = ldexpf(1.f, e - 14);
    if (blockIdx.x == 0) *err = 0u;
  }
}

// T: type of the scales and outputs. GPK, ZP as in k_w4_mv.
template <typename T, int GPK, bool ZP>
__global__ void __launch_bounds__(kW4tThreads, 1)
    k_w4_tc(const __grid_constant__ CUtensorMap tm_h, W4TcArgs a) {
  extern __shared__ __align__(1024) unsigned char w4t_sm[];
  const uint32_t raw = smem_u32(w4t_sm);
  unsigned char *ring = w4t_sm + (((raw + 1023u) & ~1023u) - raw);
  const size_t sb = w4t_stage_bytes(a.n_pad);
  unsigned char *pring = ring + (size_t)a.stages * sb;
  constexpr int kWords = kW4Tile * kW4RowWords * 4;  // bytes of packed words
  constexpr int kScales = kW4Tile * GPK * 2, kZeros = ZP ? kW4Tile * GPK : 0;
  constexpr int pb = kWords + kScales + kZeros;
  W4TcCtrl &S = *reinterpret_cast<W4TcCtrl *>(pring + (size_t)a.packed * pb);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);  // uniform
  const int G = gridDim.x, t0 = blockIdx.x;

  if (tid == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&S.full[s], 1 + kW4tConvWarps);
      mbar_init(&S.empty[s], 1);
    }
    for (int s = 0; s < a.packed; ++s) {
      mbar_init(&S.pfull[s], 1);
      mbar_init(&S.pempty[s], kW4tConvWarps);
    }
    for (int j = 0; j < 2; ++j) {
      mbar_init(&S.acc_full[j], 1);
      mbar_init(&S.acc_empty[j], kW4tEpiWarps);
    }
    mbar_init(&S.drain, 1);
    S.s_err = 0u;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&S.tmem_base)),
                 "r"(a.tmem_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, S.tmem_base, 0);
  const uint32_t a_col = (uint32_t)(a.n_acc * a.n_pad);  // first column of the A tiles

  if (warp == 0) {
    if (lane == 0) {
      int issued[kW4tMaxPacked];  // parity of the last fill of each slot, -1: none
      for (int j = 0; j < kW4tMaxPacked; ++j) issued[j] = -1;
      int ps = 0;
      uint32_t ph = 0u;
      bool ok = true;
      for (int t = t0; t < a.tiles && ok; t += G) {
        for (int kb = 0; kb < a.nb; ++kb) {
          if (!mbar_wait(&S.pempty[ps], ph ^ 1u, a.polls)) {
            atomicOr(&S.s_err, kErrCopyTimeout);
            ok = false;
            break;
          }
          unsigned char *p = pring + (size_t)ps * pb;
          const size_t blk = (size_t)t * a.nb + kb;
          mbar_expect_tx(&S.pfull[ps], (uint32_t)pb);
          bulk_g2s(p, reinterpret_cast<const unsigned char *>(a.qw) + blk * kWords, kWords,
                   &S.pfull[ps]);
          bulk_g2s(p + kWords, reinterpret_cast<const unsigned char *>(a.scales) + blk * kScales,
                   kScales, &S.pfull[ps]);
          if (ZP) bulk_g2s(p + kWords + kScales, a.zeros + blk * kZeros, kZeros, &S.pfull[ps]);
          issued[ps] = (int)ph;
          if (++ps == a.packed) {
            ps = 0;
            ph ^= 1u;
          }
        }
      }
      // every copy this thread issued has landed before the CTA may leave
      for (int j = 0; j < a.packed; ++j)
        if (issued[j] >= 0 && !mbar_wait(&S.pfull[j], (uint32_t)issued[j], a.polls))
          atomicOr(&S.s_err, kErrCopyTimeout);
    }
  } else if (warp == 2) {
    if (lane == 0) {
      int issued[kW4tMaxStages];
      for (int j = 0; j < kW4tMaxStages; ++j) issued[j] = -1;
      int s = 0;
      uint32_t ph = 0u;
      bool ok = true;
      grid_dep_wait();  // the f16 copy of the hidden rows
      for (int t = t0; t < a.tiles && ok; t += G) {
        for (int kb = 0; kb < a.nb; ++kb) {
          if (!mbar_wait(&S.empty[s], ph ^ 1u, a.polls)) {
            atomicOr(&S.s_err, kErrCopyTimeout);
            ok = false;
            break;
          }
          const bool two = 128 * kb + 64 < a.D;
          unsigned char *at = ring + (size_t)s * sb;
          mbar_expect_tx(&S.full[s], (uint32_t)(a.n_pad * (two ? 256 : 128)));
          tma_load_2d(at, &tm_h, 128 * kb, 0, &S.full[s]);
          if (two) tma_load_2d(at + a.n_pad * 128, &tm_h, 128 * kb + 64, 0, &S.full[s]);
          issued[s] = (int)ph;
          if (++s == a.stages) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      for (int j = 0; j < a.stages; ++j)
        if (issued[j] >= 0 && !mbar_wait(&S.full[j], (uint32_t)issued[j], a.polls))
          atomicOr(&S.s_err, kErrCopyTimeout);
    }
  } else if (warp == 1) {
    // the whole warp walks the loop, so that descriptors and addresses are
    // uniform; one lane issues (by a single lane inside a branch, an MMA took
    // 50 clocks to issue)
    const bool leader = w4t_elect();
    const uint32_t full0 = smem_u32(&S.full[0]), empty0 = smem_u32(&S.empty[0]);
    const uint64_t bd0 = umma_desc_k(smem_u32(ring)), step = sb >> 4;
    const uint64_t half = (uint64_t)(a.n_pad * 128) >> 4;
    const uint32_t idesc = a.idesc;
    int s = 0;
    uint32_t ph = 0u;
    bool ok = true;
    for (int t = t0, i = 0; t < a.tiles && ok; t += G, ++i) {
      const int buf = i % a.n_acc, use = i / a.n_acc;
      if (use > 0 && !mbar_wait(&S.acc_empty[buf], (uint32_t)((use - 1) & 1), a.polls)) ok = false;
      const uint32_t acc = tmem + (uint32_t)(buf * a.n_pad);
      for (int kb = 0; kb < a.nb && ok; ++kb) {
        if (!w4t_wait(full0 + 8u * s, ph, a.polls)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t bd = bd0 + step * s;
        const uint32_t at = tmem + a_col + (uint32_t)(s * kW4tACols);
        if (leader) {
          if (128 * kb + 128 <= a.D) {
#pragma unroll
            for (int q = 0; q < 8; ++q)
              w4t_mma(acc, at + 8u * q, bd + (q >> 2) * half + 2u * (q & 3), idesc,
                      q > 0 ? 1u : (uint32_t)kb);
          } else {
            for (int q = 0; 128 * kb + 16 * q < a.D; ++q)
              w4t_mma(acc, at + 8u * q, bd + (q >> 2) * half + 2u * (q & 3), idesc,
                      (uint32_t)(kb | q));
          }
          w4t_commit(empty0 + 8u * s);
        }
        __syncwarp();
        if (++s == a.stages) {
          s = 0;
          ph ^= 1u;
        }
      }
      if (ok && leader) tc_commit(&S.acc_full[buf]);
    }
    if (leader) {
      if (!ok) atomicOr(&S.s_err, kErrCopyTimeout);
      tc_commit(&S.drain);
      if (!mbar_wait(&S.drain, 0u, a.polls)) atomicOr(&S.s_err, kErrCopyTimeout);
    }
  } else if (warp >= kW4tFirstConv && warp < kW4tFirstConv + kW4tGroups * kW4tConvWarps) {
    const int group = (warp - kW4tFirstConv) / kW4tConvWarps;
    const int q4 = warp & 3, m = 32 * q4 + lane;  // this thread's row of the tile
    const W4Bits bits{a.mask, a.magic};
    const uint32_t lane_base = tmem + ((uint32_t)(32 * q4) << 16) + a_col;
    int s = 0, ps = 0, turn = 0;
    uint32_t ph = 0u, pph = 0u;
    bool ok = group < a.groups;
    for (int t = t0; t < a.tiles && ok; t += G) {
      const float mul = __ldg(a.row_mul + t * kW4Tile + m);
      for (int kb = 0; kb < a.nb && ok; ++kb) {
        const bool mine = turn == group;
        if (++turn == a.groups) turn = 0;
        if (!mine) {  // another group's block: step over its slot and stages
          if (++ps == a.packed) {
            ps = 0;
            pph ^= 1u;
          }
          if (++s == a.stages) {
            s = 0;
            ph ^= 1u;
          }
          continue;
        }
        if (!mbar_wait(&S.pfull[ps], pph, a.polls)) {
          atomicOr(&S.s_err, kErrCopyTimeout);
          ok = false;
          break;
        }
        const unsigned char *pk = pring + (size_t)ps * pb;
        uint4 q[4];
        uint32_t sc[GPK], zz[GPK];  // scales (f16 pairs), zero points
#pragma unroll
        for (int c = 0; c < 4; ++c) q[c] = lds128(pk + (c * kW4Tile + m) * 16);
#pragma unroll
        for (int g = 0; g < GPK; ++g) {
          const uint16_t bits = reinterpret_cast<const uint16_t *>(pk + kWords)[m * GPK + g];
          const __half2 h = __float2half2_rn(W4Num<T>::scale(bits) * mul);
          sc[g] = *reinterpret_cast<const uint32_t *>(&h);
          zz[g] = ZP ? (uint32_t)pk[kWords + kScales + m * GPK + g] : 8u;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_cta(&S.pempty[ps]);
        if (++ps == a.packed) {
          ps = 0;
          pph ^= 1u;
        }
        if (!mbar_wait(&S.empty[s], ph ^ 1u, a.polls)) {
          atomicOr(&S.s_err, kErrCopyTimeout);
          ok = false;
        }
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int g = j * GPK / 4;
          const W4Zero<__half> zero(zz[g]);
          uint32_t x[16];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t w = j == 0 ? q[c].x : j == 1 ? q[c].y : j == 2 ? q[c].z : q[c].w;
            uint32_t y[4];
            w4_unpack<__half>(w, bits, zero, y);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const __half2 v = __hmul2(*reinterpret_cast<const __half2 *>(&y[e]),
                                        *reinterpret_cast<const __half2 *>(&sc[g]));
              x[4 * c + e] = *reinterpret_cast<const uint32_t *>(&v);
            }
          }
          w4t_st16(lane_base + (uint32_t)(s * kW4tACols + 16 * j), x);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cta(&S.full[s]);
        if (++s == a.stages) {
          s = 0;
          ph ^= 1u;
        }
      }
    }
  } else if (warp > 3) {
    const int q = warp & 3;  // TMEM lane quadrant of this warp
    const int et = tid - 32 * (kW4tFirstConv + kW4tGroups * kW4tConvWarps);
    grid_dep_wait();
    for (int i = et; i < kW4tMaxN; i += 32 * kW4tEpiWarps)
      S.fac[i] = a.row_fac && i < a.rows ? a.row_fac[i] : 1.f;
    nbar_sync(1, 32 * kW4tEpiWarps);
    bool ok = true;
    for (int t = t0, i = 0; t < a.tiles && ok; t += G, ++i) {
      const int buf = i % a.n_acc, use = i / a.n_acc;
      if (!mbar_wait(&S.acc_full[buf], (uint32_t)(use & 1), a.polls)) {
        atomicOr(&S.s_err, kErrCopyTimeout);
        ok = false;
      }
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (!ok) break;
      tc_fence_after();
      const int v0 = t * kW4Tile + 32 * q, v = v0 + lane;
      const float back = 1.f / __ldg(a.row_mul + v);  // a power of two
      T *out = reinterpret_cast<T *>(a.out);
      T *stage = reinterpret_cast<T *>(S.out[warp - kW4tEpi]);
      const uint32_t base = tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(buf * a.n_pad);
      for (int c = 0; c < a.n_pad; c += 32) {
        uint32_t x[2][16];
        tc_ld16(base + (uint32_t)c, x[0]);
        if (c + 16 < a.n_pad) tc_ld16(base + (uint32_t)(c + 16), x[1]);
        float4 fac[8];  // read before the stores below, which may alias them
#pragma unroll
        for (int j = 0; j < 8; ++j) fac[j] = *reinterpret_cast<const float4 *>(&S.fac[c + 4 * j]);
        tc_wait_ld();
        // through shared memory: 16-byte stores instead of 2-byte ones
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float4 f = fac[j >> 2];
          const float fj = (j & 3) == 0 ? f.x : (j & 3) == 1 ? f.y : (j & 3) == 2 ? f.z : f.w;
          stage[32 * j + lane] = from_float<T>(__uint_as_float(x[j >> 4][j & 15]) * back * fj);
        }
        __syncwarp();
        if (a.vec) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = c + 8 * i + (lane >> 2), vv = v0 + 8 * (lane & 3);
            if (r < a.rows && vv < a.V)
              *reinterpret_cast<uint4 *>(out + (long long)r * a.ldo + vv) =
                  S.out[warp - kW4tEpi][32 * i + lane];
          }
        } else if (v < a.V) {
          for (int j = 0; j < 32 && c + j < a.rows; ++j)
            out[(long long)(c + j) * a.ldo + v] = stage[32 * j + lane];
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cta(&S.acc_empty[buf]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(a.tmem_cols)
                 : "memory");
  }
  if (tid == 0 && S.s_err) atomicOr(a.err, S.s_err);
}

}  // namespace fh

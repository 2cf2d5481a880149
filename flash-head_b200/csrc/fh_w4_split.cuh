// Logits of a 4-bit head with scale groups of 32 or 64 columns for many rows, on
// the 5th-generation tensor cores:
// out[b, v] = sum_k w[v, k] h[b, k], M = 128 weight rows, N = up to 128 hidden
// rows per launch. (Groups of 128: fh_w4_tc.cuh, which is faster for them: with one
// accumulator for both parts, 64 rows of a 1536 x 151936 head 54 us against 60, 256
// of 2048 x 128256 148 against 176, but reads accumulators back once per group:
// with groups of 32, 64 rows of 2048 x 128256 took it 137 us against 72 here, with
// groups of 64 128 rows 139 against 105.)
//
// A weight (q - z) s is the product of an integer of up to 4 bits and a scale of 8
// (bf16) or 11 (fp16): it has up to 15 bits, more than the hidden states' 16-bit
// type holds. It is the exact sum of two numbers of that type: hi, the product
// rounded, and lo, what was rounded off, which one fused multiply-add gives. Both
// are operands, so that no weight and no hidden state is rounded, however far
// apart scales or hidden states lie, and logits differ from k_w4_mv's only in the
// order of their fp32 sums. Each part has an accumulator of its own: the tensor
// core truncates its fp32 sum at every step, of which one accumulator would see
// twice as many, and an infinite hidden state times a lo of 0 would make NaN of an
// infinite logit.
// 15 s may pass the type's largest number: rows with a scale above 2^12 (fp16) or
// 2^124 (bf16) are brought down by 2^-4 (row_mul), undone in the epilogue.
//
// The unpacked operands go to tensor memory, not to shared memory (fh_w4_tc.cuh).
//
// One persistent CTA per SM, 20 warps:
//   warp 0      lane 0 brings the packed blocks (8 KB of words, the scales and
//               zero points of 128 rows x 128 columns: two or three bulk copies)
//               into a ring of their own, deep enough to keep HBM busy;
//   warp 2      lane 0 brings the hidden tiles of every 128 columns (TMA, two of 64
//               with the 128-byte swizzle) into the stages;
//   warp 1      allocates TMEM; one lane issues tcgen05.mma (K = 16), 16 per
//               stage, A from tensor memory, B from shared memory;
//   warps 4-15  unpack, in three groups of 4 on successive blocks: a thread has one
//               weight row, i.e. one TMEM lane, reads its 64 bytes of the block
//               and stores 32 columns' pairs, hi and lo (16 TMEM columns each) at a
//               time;
//   warps 16-19 epilogue: a thread has one weight row and all hidden rows; up to
//               32 hidden rows the accumulators are double-buffered.
// Bound: the issue of the MMAs, some 46 clocks each whatever N is (twice the warps
// that unpack changed nothing). 2048 x 128256, zero points: 16 rows 62 us, 64
// 72 us, 128 105 us, 256 217 us in two launches (183 in one, with one accumulator).
// Every wait is bounded; on a timeout the CTA drains its own copies and MMAs
// (bounded), frees TMEM, fills the logits of its tiles with NaN and records
// kErrCopyTimeout.
#pragma once

#include "fh_w4_tc.cuh"

namespace fh {

constexpr int kW4sConvWarps = 4;  // unpack one block together, a TMEM quadrant each
constexpr int kW4sGroups = 3;     // of such warps, on successive blocks (a launch may use fewer)
constexpr int kW4sEpiWarps = 4;
constexpr int kW4sFirstConv = 4;  // warp
constexpr int kW4sEpi = kW4sFirstConv + kW4sGroups * kW4sConvWarps;
constexpr int kW4sThreads = 32 * (kW4sFirstConv + kW4sGroups * kW4sConvWarps + kW4sEpiWarps);
constexpr int kW4sMaxN = 128;
constexpr int kW4sMaxStages = 3;
constexpr int kW4sACols = 128;  // TMEM columns of a stage's A tiles: 128 numbers per row, hi and lo
constexpr int kW4sMaxPacked = 12;

struct W4SplitArgs {
  const uint32_t *qw;
  const void *scales;
  const uint8_t *zeros;
  const float *row_mul;   // [128 * tiles] powers of two
  int V, D, nb;
  int tiles;
  int rows, n_pad;
  int stages, packed, n_acc, groups;
  int tmem_cols;
  int vec;                // outputs take 16-byte stores (V, ldo and out allow them)
  uint32_t idesc;
  uint32_t mask, magic;   // kW4Mask, W4Num<T>::kMagic
  void *out;
  long long ldo;
  uint32_t *err;
  uint32_t polls;
};

struct W4SplitCtrl {
  uint64_t full[kW4sMaxStages];    // hidden tile landed and A tile written
  uint64_t empty[kW4sMaxStages];   // MMAs done
  uint64_t pfull[kW4sMaxPacked];   // packed block landed
  uint64_t pempty[kW4sMaxPacked];  // packed block unpacked
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t drain;
  uint32_t tmem_base;
  uint32_t s_err;
  alignas(16) uint4 out[kW4sEpiWarps][128];  // 32 hidden rows x 32 weight rows, 16-bit
};

// Groups that may run. A group steps over the others' blocks, so that it knows of
// a barrier's progress only what the order of the work implies; a parity wait
// is unambiguous while the phase before the awaited one is known to be
// complete. Having written block n, a group knows the MMAs up to block
// n - stages, and with them the packed blocks up to there, to be done. Its next
// block n + groups needs the stage's use two rounds back, n + groups - 2 stages,
// and the packed slot's fill one round back, n + groups - packed, among them.
__host__ __device__ inline int w4s_groups(int stages, int packed) {
  int g = kW4sGroups;
  while (g > 0 && (g > stages || packed < g + stages)) --g;
  return g;
}

__host__ __device__ inline size_t w4s_smem_bytes(int n_pad, int stages, int packed, int gpk, bool zp) {
  return 1024 + stages * w4_stage_bytes(n_pad) + (size_t)packed * w4_packed_bytes(gpk, zp) +
         sizeof(W4SplitCtrl);
}

// Pairs of a type: products, and what their rounding lost.
template <typename T>
struct W4Pair;
template <>
struct W4Pair<__nv_bfloat16> {
  __device__ __forceinline__ static uint32_t twice(float s) {
    const __nv_bfloat162 v = __float2bfloat162_rn(s);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  __device__ __forceinline__ static void split(uint32_t x, uint32_t s, uint32_t &hi, uint32_t &lo) {
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"(x), "r"(s));
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(lo) : "r"(x), "r"(s), "r"(hi ^ 0x80008000u));
  }
};
template <>
struct W4Pair<__half> {
  __device__ __forceinline__ static uint32_t twice(float s) {
    const __half2 v = __float2half2_rn(s);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  __device__ __forceinline__ static void split(uint32_t x, uint32_t s, uint32_t &hi, uint32_t &lo) {
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(x), "r"(s));
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(lo) : "r"(x), "r"(s), "r"(hi ^ 0x80008000u));
  }
};

// T: type of the hidden states, scales and outputs. GPK, ZP as in k_w4_mv.
template <typename T, int GPK, bool ZP>
__global__ void __launch_bounds__(kW4sThreads, 1)
    k_w4_split(const __grid_constant__ CUtensorMap tm_h, W4SplitArgs a) {
  extern __shared__ __align__(1024) unsigned char w4s_sm[];
  const uint32_t raw = smem_u32(w4s_sm);
  unsigned char *ring = w4s_sm + (((raw + 1023u) & ~1023u) - raw);
  const size_t sb = w4_stage_bytes(a.n_pad);
  unsigned char *pring = ring + (size_t)a.stages * sb;
  constexpr int kWords = kW4Tile * kW4RowWords * 4;  // bytes of packed words
  constexpr int kScales = kW4Tile * GPK * 2, kZeros = ZP ? kW4Tile * GPK : 0;
  constexpr int pb = kWords + kScales + kZeros;
  W4SplitCtrl &S = *reinterpret_cast<W4SplitCtrl *>(pring + (size_t)a.packed * pb);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);  // uniform
  const int G = gridDim.x, t0 = blockIdx.x;

  if (tid == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&S.full[s], 1 + kW4sConvWarps);
      mbar_init(&S.empty[s], 1);
    }
    for (int s = 0; s < a.packed; ++s) {
      mbar_init(&S.pfull[s], 1);
      mbar_init(&S.pempty[s], kW4sConvWarps);
    }
    for (int j = 0; j < 2; ++j) {
      mbar_init(&S.acc_full[j], 1);
      mbar_init(&S.acc_empty[j], kW4sEpiWarps);
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
  const uint32_t a_col = (uint32_t)(2 * a.n_acc * a.n_pad);  // first column of the A tiles

  if (warp == 0) {
    if (lane == 0) {
      int issued[kW4sMaxPacked];  // parity of the last fill of each slot, -1: none
      for (int j = 0; j < kW4sMaxPacked; ++j) issued[j] = -1;
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
        if (issued[j] >= 0 && !mbar_wait(&S.pfull[j], (uint32_t)issued[j], kW4DrainPolls))
          atomicOr(&S.s_err, kErrCopyTimeout);
    }
  } else if (warp == 2) {
    if (lane == 0) {
      int issued[kW4sMaxStages];
      for (int j = 0; j < kW4sMaxStages; ++j) issued[j] = -1;
      int s = 0;
      uint32_t ph = 0u;
      bool ok = true;
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
        if (issued[j] >= 0 && !mbar_wait(&S.full[j], (uint32_t)issued[j], kW4DrainPolls))
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
      if (use > 0)
        ok = w4t_wait_all(smem_u32(&S.acc_empty[buf]), (uint32_t)((use - 1) & 1), a.polls);
      const uint32_t acc = tmem + (uint32_t)(2 * buf * a.n_pad);
      const uint32_t acc_lo = acc + (uint32_t)a.n_pad;
      for (int kb = 0; kb < a.nb && ok; ++kb) {
        ok = w4t_wait_all(full0 + 8u * s, ph, a.polls);
        if (!ok) break;
        tc_fence_after();
        const uint64_t bd = bd0 + step * s;
        const uint32_t at = tmem + a_col + (uint32_t)(s * kW4sACols);
        if (leader) {
          if (128 * kb + 128 <= a.D) {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const uint64_t b = bd + (q >> 2) * half + 2u * (q & 3);
              w4t_mma(acc, at + 8u * q, b, idesc, q > 0 ? 1u : (uint32_t)kb);
              w4t_mma(acc_lo, at + 64u + 8u * q, b, idesc, q > 0 ? 1u : (uint32_t)kb);
            }
          } else {
            for (int q = 0; 128 * kb + 16 * q < a.D; ++q) {
              const uint64_t b = bd + (q >> 2) * half + 2u * (q & 3);
              w4t_mma(acc, at + 8u * q, b, idesc, (uint32_t)(kb | q));
              w4t_mma(acc_lo, at + 64u + 8u * q, b, idesc, (uint32_t)(kb | q));
            }
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
      if (!mbar_wait(&S.drain, 0u, kW4DrainPolls)) atomicOr(&S.s_err, kErrCopyTimeout);
    }
  } else if (warp >= kW4sFirstConv && warp < kW4sFirstConv + kW4sGroups * kW4sConvWarps) {
    const int group = (warp - kW4sFirstConv) / kW4sConvWarps;
    const int q4 = warp & 3, m = 32 * q4 + lane;  // this thread's row of the tile
    const W4Bits bits{a.mask, a.magic};
    const uint32_t lane_base = tmem + ((uint32_t)(32 * q4) << 16) + a_col;
    int s = 0, ps = 0, turn = 0;
    uint32_t ph = 0u, pph = 0u;
    const bool idle = group >= a.groups;
    bool ok = true;
    for (int t = t0; t < a.tiles && ok && !idle; t += G) {
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
        ok = w4t_wait_all(smem_u32(&S.pfull[ps]), pph, a.polls);
        if (!ok) break;
        const unsigned char *pk = pring + (size_t)ps * pb;
        uint4 q[4];
        uint32_t sc[GPK], zz[GPK];  // scales (twice each), zero points
#pragma unroll
        for (int c = 0; c < 4; ++c) q[c] = lds128(pk + (c * kW4Tile + m) * 16);
#pragma unroll
        for (int g = 0; g < GPK; ++g) {
          const uint16_t bits = reinterpret_cast<const uint16_t *>(pk + kWords)[m * GPK + g];
          sc[g] = W4Pair<T>::twice(W4Num<T>::scale(bits) * mul);
          zz[g] = ZP ? (uint32_t)pk[kWords + kScales + m * GPK + g] : 8u;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_cta(&S.pempty[ps]);
        if (++ps == a.packed) {
          ps = 0;
          pph ^= 1u;
        }
        ok = w4t_wait_all(smem_u32(&S.empty[s]), ph ^ 1u, a.polls);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int g = j * GPK / 4;
          const W4Zero<T> zero(zz[g]);
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t w = j == 0 ? q[c].x : j == 1 ? q[c].y : j == 2 ? q[c].z : q[c].w;
            uint32_t y[4];
            w4_unpack<T>(w, bits, zero, y);
#pragma unroll
            for (int e = 0; e < 4; ++e) W4Pair<T>::split(y[e], sc[g], hi[4 * c + e], lo[4 * c + e]);
          }
          const uint32_t to = lane_base + (uint32_t)(s * kW4sACols + 16 * j);
          w4t_st16(to, hi);
          w4t_st16(to + 64u, lo);
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
    if (!ok && lane == 0) atomicOr(&S.s_err, kErrCopyTimeout);
  } else if (warp > 3) {
    const int q = warp & 3;  // TMEM lane quadrant of this warp
    bool ok = true;
    for (int t = t0, i = 0; t < a.tiles && ok; t += G, ++i) {
      const int buf = i % a.n_acc, use = i / a.n_acc;
      ok = w4t_wait_all(smem_u32(&S.acc_full[buf]), (uint32_t)(use & 1), a.polls);
      if (!ok) break;
      tc_fence_after();
      const int v0 = t * kW4Tile + 32 * q, v = v0 + lane;
      const float back = 1.f / __ldg(a.row_mul + v);  // a power of two
      T *out = reinterpret_cast<T *>(a.out);
      T *stage = reinterpret_cast<T *>(S.out[warp - kW4sEpi]);
      const uint32_t base = tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(2 * buf * a.n_pad);
      for (int c = 0; c < a.n_pad; c += 32) {
        // through shared memory: 16-byte stores instead of 2-byte ones
        __syncwarp();
#pragma unroll
        for (int half = 0; half < 32; half += 16) {
          if (c + half >= a.n_pad) break;
          uint32_t hi[16], lo[16];
          tc_ld16(base + (uint32_t)(c + half), hi);
          tc_ld16(base + (uint32_t)(a.n_pad + c + half), lo);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            // (an infinite hidden state times a lo of 0 is NaN: hi says what it is)
            float x = __uint_as_float(hi[j]);
            if (fabsf(x) < INFINITY) x += __uint_as_float(lo[j]);
            stage[32 * (half + j) + lane] = from_float<T>(x * back);
          }
        }
        __syncwarp();
        if (a.vec) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = c + 8 * i + (lane >> 2), vv = v0 + 8 * (lane & 3);
            if (r < a.rows && vv < a.V)
              *reinterpret_cast<uint4 *>(out + (long long)r * a.ldo + vv) =
                  S.out[warp - kW4sEpi][32 * i + lane];
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
    if (!ok && lane == 0) atomicOr(&S.s_err, kErrCopyTimeout);
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
  if (S.s_err) {
    w4t_fill(reinterpret_cast<T *>(a.out), a.ldo, a.rows, a.V, t0, a.tiles, G);
    if (tid == 0) atomicOr(a.err, S.s_err);
  }
}

}  // namespace fh

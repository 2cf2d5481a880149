// Logits of a 4-bit head with scale groups of 128 columns for many rows, on the
// 5th-generation tensor cores:
// out[b, v] = sum_g s[v, g] sum_{k in g} (q[v, k] - z[v, g]) h[b, k], M = 128
// weight rows, N = up to 128 hidden rows per launch. (Smaller groups:
// fh_w4_split.cuh.)
//
// The products are k_w4_mv's: the operands are the integers q - z, exact in
// the hidden states' own 16-bit type, and those hidden states as they are; a
// group's products are summed in fp32 in an accumulator of their own, and the
// group's scale multiplies that sum in fp32. No weight and no hidden state is
// rounded, however far apart scales or hidden states lie. (Scales multiplied
// into one f16 operand need no accumulator per group and take 45 us where this
// takes 54, but round weights to 11 bits and lose scales 2^-14 below their row's
// largest.)
//
// The unpacked operand goes to tensor memory, not to shared memory: 16 KB
// written and 16 KB read per 128 x 64 tile were most of the shared-memory
// traffic that bound a first version.
//
// One persistent CTA per SM, 28 warps; its blocks (128 columns, one scale group, of
// a tile of 128 weight rows) are numbered in the order of the work:
//   warp 0      lane 0 brings the packed blocks (8 KB of words, the scales and zero
//               points: two or three bulk copies) into a ring of their own, deep
//               enough to keep HBM busy;
//   warp 2      lane 0 brings the hidden tiles of every block (TMA, two of 64 columns
//               with the 128-byte swizzle) into the stages (a thread of its own: a wait that
//               suspends the one for packed slots must not hold up these);
//   warps 1, 3  issue tcgen05.mma (K = 16), 8 a block, A from tensor memory, B
//               from shared memory: warp 1 the even blocks, warp 3 the odd ones, each
//               into accumulators of its own. Warp 1 also allocates TMEM;
//   warps 4-27  six groups of 4 (a TMEM quadrant each). The last one to four, one
//               for every 32 hidden rows, sum and store: a thread has one weight
//               row and 32 hidden rows, whose logits it keeps in registers. The
//               first ones (4 or 2) unpack, on successive blocks: a thread has one
//               weight row, reads its 64 bytes of the block and stores 32
//               columns' pairs (16 TMEM columns) at a time; it also hands the
//               scale on, in shared memory.
// More than 128 rows take several launches: two more sets of accumulators would
// not fit beside the operand, nor their sums in the registers.
// Bound: the chain of barriers that every block passes (a wait costs some 130
// clocks, met or not) and the issue slots (73 to 75 %): 9 rows of a 2048 x 128256 head
// 49 us, 64 of a 1536 x 151936 one 54 us (2.2 TB/s), 128 and 256 of 2048 x 128256
// 75 and 148 us (0.9 PFLOP/s). Tried and slower: polls with a time hint, fp32x2
// multiply-adds, half as many warps that sum 64 rows each, and twice as many that
// take every other block.
// Every wait is bounded; on a timeout the CTA drains its own copies and MMAs
// (bounded), frees TMEM, fills the logits of its tiles with NaN and records
// kErrCopyTimeout.
#pragma once

#include "fh_s1_tc.cuh"
#include "fh_w4.cuh"

namespace fh {

constexpr int kW4tConvWarps = 4;  // unpack one block together, a TMEM quadrant each
constexpr int kW4tGroups = 4;     // of such warps, on successive blocks (a launch may use fewer)
constexpr int kW4tTeams = 6;      // groups of 4 warps that unpack, or sum and store
constexpr int kW4tFirst = 4;      // their first warp
constexpr int kW4tThreads = 32 * (kW4tFirst + 4 * kW4tTeams);
constexpr int kW4tCols = 32;      // hidden rows of a group that sums
constexpr int kW4tMaxN = 128;
constexpr int kW4tStages = 4;     // blocks of hidden columns and unpacked weights
constexpr int kW4tMaxAcc = 2;     // accumulators of an issuing warp
constexpr int kW4tACols = 64;  // TMEM columns of a stage's A tile: 128 16-bit numbers per row
constexpr int kW4tMaxPacked = 12;
// Blocks of scales handed on. Block n's are written when the MMAs of block
// n - stages are done, which were issued when the block 2 * n_acc before had been
// summed (n_acc accumulators in each of two warps): the slot's last use, 8 blocks
// before, is over.
constexpr int kW4tScaleSlots = 8;
static_assert(kW4tScaleSlots >= kW4tStages + 2 * kW4tMaxAcc, "a slot may still be read");
constexpr int kW4tOutBytes = 32 * 16 * 2;  // a warp's outputs, 16 hidden rows at a time
constexpr int kW4SmemMax = 227 * 1024;
// Polls for copies and MMAs in flight before a CTA leaves: milliseconds, for what
// takes microseconds. (The limit of the other waits may be set to less.)
constexpr uint32_t kW4DrainPolls = 1u << 14;

struct W4TcArgs {
  const uint32_t *qw;
  const void *scales;
  const uint8_t *zeros;
  int V, D, nb;
  int tiles;
  int rows, n_pad;
  int packed;  // slots of packed blocks
  int n_acc;   // accumulators of an issuing warp (1 or 2)
  int groups;  // groups that unpack
  int sums;    // groups that sum and store
  int tmem_cols;
  int vec;                // outputs take 16-byte stores (V, ldo and out allow them)
  uint32_t idesc;
  uint32_t mask, magic;   // kW4Mask, W4Num<T>::kMagic
  void *out;
  long long ldo;
  uint32_t *err;
  uint32_t polls;
};

struct W4TcCtrl {
  uint64_t hfull[kW4tStages];   // hidden tile landed
  uint64_t full[kW4tStages];    // A tile written
  uint64_t empty[kW4tStages];   // MMAs done
  uint64_t pfull[kW4tMaxPacked];   // packed block landed
  uint64_t pempty[kW4tMaxPacked];  // packed block unpacked
  uint64_t acc_full[2][kW4tMaxAcc];
  uint64_t acc_empty[2][kW4tMaxAcc];
  uint64_t drain;
  uint32_t tmem_base;
  uint32_t s_err;
};

// Groups that may unpack: as many as divide the stages and the packed slots, so
// that a stage and a slot are always the same group's. A parity wait cannot tell
// a phase from the one two before it: a group that did not see every phase of
// a barrier might pass one early.
__host__ __device__ inline int w4t_groups(int stages, int packed) {
  int g = kW4tGroups;
  while (g > 0 && (g > stages || packed < g + stages || stages % g || packed % g)) --g;
  return g;
}

__host__ __device__ inline int w4_packed_bytes(int gpk, bool zp) {
  return kW4Tile * kW4RowWords * 4 + kW4Tile * gpk * (zp ? 3 : 2);
}
__host__ __device__ inline size_t w4_stage_bytes(int n_pad) {
  return (size_t)n_pad * 256;  // two tiles of 64 hidden columns
}
// Everything but the packed ring.
__host__ __device__ inline size_t w4t_other_bytes(int n_pad, int sums) {
  return 1024 + kW4tStages * w4_stage_bytes(n_pad) + (size_t)kW4tScaleSlots * kW4Tile * 2 +
         (size_t)sums * 4 * kW4tOutBytes + sizeof(W4TcCtrl);
}

// NaN in the rows x 128 logits of a CTA's tiles t, t + step, ...
template <typename T>
__device__ __noinline__ void w4t_fill(T *out, long long ldo, int rows, int V, int t, int tiles,
                                      int step) {
  const T nan = from_float<T>(__int_as_float(0x7FFFFFFF));
  for (; t < tiles; t += step)
    for (int i = threadIdx.x; i < rows * kW4Tile; i += blockDim.x) {
      const int v = t * kW4Tile + i % kW4Tile;
      if (v < V) out[(long long)(i / kW4Tile) * ldo + v] = nan;
    }
}

// mbar_wait by shared-memory address.
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
// The same by a whole warp, with one outcome for all its lanes.
__device__ __forceinline__ bool w4t_wait_all(uint32_t bar, uint32_t parity, uint32_t polls) {
  return __all_sync(0xFFFFFFFFu, w4t_wait(bar, parity, polls));
}
// The same by a group of 4 warps (named barrier `id`): its first warp polls, the
// others are held by the barrier, which brings them the outcome. (28 warps that
// poll took a third of the issue slots.)
__device__ __forceinline__ bool w4t_wait_group(uint32_t bar, uint32_t parity, uint32_t polls,
                                               int id, bool first) {
  const uint32_t failed = first && !w4t_wait(bar, parity, polls);
  uint32_t any;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n"
      " barrier.cta.red.or.pred q, %2, 128, p;\n selp.u32 %0, 1, 0, q;\n}"
      : "=r"(any)
      : "r"(failed), "r"(id)
      : "memory");
  return any == 0u;
}
__device__ __forceinline__ void w4t_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   bar)
               : "memory");
}
__device__ __forceinline__ void w4t_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ bool w4t_elect() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}"
               : "=r"(p));
  return p != 0;
}
// D += A . B with A in tensor memory: row m in lane m, two 16-bit numbers per column.
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

// A position in a ring of n barriers and the parity of its current round.
struct W4tRing {
  int at = 0;
  uint32_t phase = 0u;
  __device__ __forceinline__ void next(int n) {
    if (++at == n) {
      at = 0;
      phase ^= 1u;
    }
  }
};

// A block's accumulator among the n_acc (1 or 2) of the warp that issues its MMAs.
struct W4tUse {
  uint32_t at, phase;
  __device__ __forceinline__ W4tUse(uint32_t block, uint32_t n_acc) {
    const uint32_t use = block >> 1;
    at = use & (n_acc - 1u);
    phase = (n_acc == 2u ? use >> 1 : use) & 1u;
  }
};

// T: type of the hidden states, scales and outputs. ZP: with zero points.
template <typename T, bool ZP>
__global__ void __launch_bounds__(kW4tThreads, 1)
    k_w4_tc(const __grid_constant__ CUtensorMap tm_h, W4TcArgs a) {
  extern __shared__ __align__(1024) unsigned char w4t_sm[];
  const uint32_t raw = smem_u32(w4t_sm);
  unsigned char *ring = w4t_sm + (((raw + 1023u) & ~1023u) - raw);
  const size_t sb = w4_stage_bytes(a.n_pad);
  constexpr int kWords = kW4Tile * kW4RowWords * 4;  // bytes of packed words
  constexpr int kScales = kW4Tile * 2, kZeros = ZP ? kW4Tile : 0;
  constexpr int pb = kWords + kScales + kZeros;
  unsigned char *pring = ring + (size_t)kW4tStages * sb;
  unsigned char *sring = pring + (size_t)a.packed * pb;
  unsigned char *oring = sring + kW4tScaleSlots * kScales;
  W4TcCtrl &S = *reinterpret_cast<W4TcCtrl *>(oring + (size_t)a.sums * 4 * kW4tOutBytes);
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);  // uniform
  const int G = gridDim.x, t0 = blockIdx.x;
  const int team = (warp - kW4tFirst) >> 2;

  if (tid == 0) {
    for (int s = 0; s < kW4tStages; ++s) {
      mbar_init(&S.hfull[s], 1);
      mbar_init(&S.full[s], kW4tConvWarps);
      mbar_init(&S.empty[s], 1);
    }
    for (int s = 0; s < a.packed; ++s) {
      mbar_init(&S.pfull[s], 1);
      mbar_init(&S.pempty[s], kW4tConvWarps);
    }
    for (int i = 0; i < 2; ++i)
      for (int j = 0; j < a.n_acc; ++j) {
        mbar_init(&S.acc_full[i][j], 1);
        mbar_init(&S.acc_empty[i][j], 4 * a.sums);
      }
    mbar_init(&S.drain, 2);
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
      uint32_t sent = 0u;  // slots filled, and the parity of their last fill
      uint32_t parity = 0u;
      W4tRing p;
      bool ok = true;
      for (int t = t0; t < a.tiles && ok; t += G) {
        for (int kb = 0; kb < a.nb; ++kb) {
          if (!mbar_wait(&S.pempty[p.at], p.phase ^ 1u, a.polls)) {
            atomicOr(&S.s_err, kErrCopyTimeout);
            ok = false;
            break;
          }
          unsigned char *to = pring + (size_t)p.at * pb;
          const size_t blk = (size_t)t * a.nb + kb;
          mbar_expect_tx(&S.pfull[p.at], (uint32_t)pb);
          bulk_g2s(to, reinterpret_cast<const unsigned char *>(a.qw) + blk * kWords, kWords,
                   &S.pfull[p.at]);
          bulk_g2s(to + kWords, reinterpret_cast<const unsigned char *>(a.scales) + blk * kScales,
                   kScales, &S.pfull[p.at]);
          if (ZP)
            bulk_g2s(to + kWords + kScales, a.zeros + blk * kZeros, kZeros, &S.pfull[p.at]);
          sent |= 1u << p.at;
          parity = (parity & ~(1u << p.at)) | (p.phase << p.at);
          p.next(a.packed);
        }
      }
      // every copy this thread issued has landed before the CTA may leave
      for (int j = 0; j < a.packed; ++j)
        if ((sent >> j) & 1u && !mbar_wait(&S.pfull[j], (parity >> j) & 1u, kW4DrainPolls))
          atomicOr(&S.s_err, kErrCopyTimeout);
    }
  } else if (warp == 2) {
    if (lane == 0) {
      uint32_t sent = 0u, parity = 0u;
      W4tRing p;
      bool ok = true;
      for (int t = t0; t < a.tiles && ok; t += G) {
        for (int kb = 0; kb < a.nb; ++kb) {
          if (!mbar_wait(&S.empty[p.at], p.phase ^ 1u, a.polls)) {
            atomicOr(&S.s_err, kErrCopyTimeout);
            ok = false;
            break;
          }
          unsigned char *at = ring + (size_t)p.at * sb;
          mbar_expect_tx(&S.hfull[p.at], (uint32_t)(a.n_pad * 256));
          tma_load_2d(at, &tm_h, 128 * kb, 0, &S.hfull[p.at]);
          tma_load_2d(at + a.n_pad * 128, &tm_h, 128 * kb + 64, 0, &S.hfull[p.at]);
          sent |= 1u << p.at;
          parity = (parity & ~(1u << p.at)) | (p.phase << p.at);
          p.next(kW4tStages);
        }
      }
      for (int j = 0; j < kW4tStages; ++j)
        if ((sent >> j) & 1u && !mbar_wait(&S.hfull[j], (parity >> j) & 1u, kW4DrainPolls))
          atomicOr(&S.s_err, kErrCopyTimeout);
    }
  } else if (warp == 1 || warp == 3) {
    // the whole warp walks the loop, so that descriptors and addresses are
    // uniform; one lane issues (by a single lane inside a branch, an MMA took
    // 50 clocks to issue)
    const bool leader = w4t_elect();
    const int mine = warp >> 1;
    const uint32_t hfull0 = smem_u32(&S.hfull[0]), full0 = smem_u32(&S.full[0]);
    const uint32_t empty0 = smem_u32(&S.empty[0]);
    const uint32_t afull0 = smem_u32(&S.acc_full[mine][0]);
    const uint32_t aempty0 = smem_u32(&S.acc_empty[mine][0]);
    const uint32_t acc0 = tmem + (uint32_t)(mine * a.n_acc * a.n_pad);
    const uint64_t bd0 = umma_desc_k(smem_u32(ring)), step = sb >> 4;
    const uint64_t half = (uint64_t)(a.n_pad * 128) >> 4;
    const uint32_t idesc = a.idesc;
    const uint32_t n_acc = (uint32_t)a.n_acc;
    uint32_t block = 0u;
    bool ok = true;
    for (int t = t0; t < a.tiles && ok; t += G) {
      for (int kb = 0; kb < a.nb; ++kb, ++block) {
        if ((block & 1u) != (uint32_t)mine) continue;
        const uint32_t st = block % kW4tStages, phase = (block / kW4tStages) & 1u;
        ok = w4t_wait_all(hfull0 + 8u * st, phase, a.polls) &&
             w4t_wait_all(full0 + 8u * st, phase, a.polls);
        if (!ok) break;
        const W4tUse ac(block, n_acc);
        ok = w4t_wait_all(aempty0 + 8u * ac.at, ac.phase ^ 1u, a.polls);
        if (!ok) break;
        tc_fence_after();
        const uint64_t bd = bd0 + step * st;
        const uint32_t at = tmem + a_col + st * kW4tACols;
        const uint32_t acc = acc0 + ac.at * (uint32_t)a.n_pad;
        if (leader) {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            w4t_mma(acc, at + 8u * q, bd + (q >> 2) * half + 2u * (q & 3), idesc, q > 0);
          w4t_commit(afull0 + 8u * ac.at);
          w4t_commit(empty0 + 8u * st);
        }
        __syncwarp();
      }
    }
    if (leader) {
      if (!ok) atomicOr(&S.s_err, kErrCopyTimeout);
      tc_commit(&S.drain);
      if (!mbar_wait(&S.drain, 0u, kW4DrainPolls)) atomicOr(&S.s_err, kErrCopyTimeout);
    }
  } else if (team < a.groups) {
    const int q4 = warp & 3, m = 32 * q4 + lane;  // this thread's row of the tile
    const W4Bits bits{a.mask, a.magic};
    const uint32_t lane_base = tmem + ((uint32_t)(32 * q4) << 16) + a_col;
    W4tRing st, pk;
    int turn = 0;
    uint32_t block = 0u;
    bool ok = true;
    for (int t = t0; t < a.tiles && ok; t += G) {
      for (int kb = 0; kb < a.nb; ++kb, ++block) {
        const bool mine = turn == team;
        if (++turn == a.groups) turn = 0;
        if (!mine) {  // another group's block: step over its slot and stage
          pk.next(a.packed);
          st.next(kW4tStages);
          continue;
        }
        ok = w4t_wait_group(smem_u32(&S.pfull[pk.at]), pk.phase, a.polls, 1 + team, q4 == 0);
        if (!ok) break;
        const unsigned char *p = pring + (size_t)pk.at * pb;
        uint4 q[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) q[c] = lds128(p + (c * kW4Tile + m) * 16);
        const uint16_t scale = reinterpret_cast<const uint16_t *>(p + kWords)[m];
        const W4Zero<T> zero(ZP ? (uint32_t)p[kWords + kScales + m] : 8u);
        __syncwarp();
        if (lane == 0) mbar_arrive_cta(&S.pempty[pk.at]);
        pk.next(a.packed);
        ok = w4t_wait_group(smem_u32(&S.empty[st.at]), st.phase ^ 1u, a.polls, 1 + team, q4 == 0);
        if (!ok) break;
        tc_fence_after();
        reinterpret_cast<uint16_t *>(sring + (block % kW4tScaleSlots) * kScales)[m] = scale;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t x[16];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t w = j == 0 ? q[c].x : j == 1 ? q[c].y : j == 2 ? q[c].z : q[c].w;
            uint32_t y[4];
            w4_unpack<T>(w, bits, zero, y);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * c + e] = y[e];
          }
          w4t_st16(lane_base + (uint32_t)(st.at * kW4tACols + 16 * j), x);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cta(&S.full[st.at]);
        st.next(kW4tStages);
      }
    }
    if (!ok && lane == 0) atomicOr(&S.s_err, kErrCopyTimeout);
  } else if (team >= kW4tTeams - a.sums) {
    const int q4 = warp & 3, m = 32 * q4 + lane;
    const int e = team - (kW4tTeams - a.sums), c0 = kW4tCols * e;  // first hidden row
    const bool two = c0 + 16 < a.n_pad;
    const uint32_t base = tmem + ((uint32_t)(32 * q4) << 16) + (uint32_t)c0;
    const uint32_t afull0 = smem_u32(&S.acc_full[0][0]), aempty0 = smem_u32(&S.acc_empty[0][0]);
    unsigned char *stage8 = oring + (size_t)(4 * e + q4) * kW4tOutBytes;
    T *stage = reinterpret_cast<T *>(stage8);
    T *out = reinterpret_cast<T *>(a.out);
    const uint32_t n_acc = (uint32_t)a.n_acc;
    uint32_t block = 0u;
    bool ok = true;
    for (int t = t0; t < a.tiles && ok; t += G) {
      float sum[kW4tCols];
#pragma unroll
      for (int j = 0; j < kW4tCols; ++j) sum[j] = 0.f;
      for (int kb = 0; kb < a.nb && ok; ++kb, ++block) {
        const uint32_t odd = block & 1u;
        const W4tUse ac(block, n_acc);
        const uint32_t bar = 8u * (odd * kW4tMaxAcc + ac.at);
        ok = w4t_wait_group(afull0 + bar, ac.phase, a.polls, 1 + team, q4 == 0);
        if (!ok) break;
        tc_fence_after();
        const uint32_t acc = base + (odd * n_acc + ac.at) * (uint32_t)a.n_pad;
        uint32_t x[16];
        tc_ld16(acc, x);
        // (written before the MMAs that the wait was for)
        const float scale = W4Num<T>::scale(
            reinterpret_cast<const uint16_t *>(sring + (block % kW4tScaleSlots) * kScales)[m]);
        tc_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j) sum[j] = fmaf(scale, __uint_as_float(x[j]), sum[j]);
        if (two) {
          tc_ld16(acc + 16u, x);
          tc_wait_ld();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) w4t_arrive(aempty0 + bar);
        if (two)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            sum[16 + j] = fmaf(scale, __uint_as_float(x[j]), sum[16 + j]);
      }
      if (!ok) break;
      // through shared memory: 16-byte stores instead of 2-byte ones
      const int v0 = t * kW4Tile + 32 * q4, v = v0 + lane;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h == 1 && !two) break;
        const int r0 = c0 + 16 * h;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 16; ++j) stage[32 * j + lane] = from_float<T>(sum[16 * h + j]);
        __syncwarp();
        if (a.vec) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = r0 + 8 * i + (lane >> 2), vv = v0 + 8 * (lane & 3);
            if (r < a.rows && vv < a.V)
              *reinterpret_cast<uint4 *>(out + (long long)r * a.ldo + vv) =
                  lds128(stage8 + (32 * i + lane) * 16);
          }
        } else if (v < a.V) {
          for (int j = 0; j < 16 && r0 + j < a.rows; ++j)
            out[(long long)(r0 + j) * a.ldo + v] = stage[32 * j + lane];
        }
      }
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

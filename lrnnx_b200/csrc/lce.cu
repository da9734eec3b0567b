// Softmax cross entropy of hidden W^T without the logits (b200_lce_fwd / b200_lce_bwd), sm_100a.
//
//     z = H W^T   (rows x classes, H rows x features, W classes x features)
//     lse_r = log sum_v exp z_rv,     loss_r = lse_r - z_{r, label_r}
//     dz_rv = s_r (exp(z_rv - lse_r) - [v = label_r]),     dH = dz W,     dW = dz^T H
//
// The forward is one product whose tiles never leave the SM: each 128 x 256 tile of z is reduced to a running maximum
// and sum of a row's half (float32, natural units scaled by log2 e), a second kernel joins them.  The backward makes z
// again in pieces of the vocabulary, writes a piece of dz in the operands' type and multiplies it from both sides; the
// piece's columns are chosen so that dz stays below kPieceBytes.  dz is kept in units of the largest |s_r|, float16 in a
// 2^15th of it, so that a float16 dz neither overflows under a scaled loss nor vanishes under a mean over many rows or where
// probabilities are small: below 2^-29 of the largest weight it loses bits, below 2^-40 it is zero.  The products are scaled back
// in 32 bits.  s_r = 0 (ignored labels) makes an exact zero row.
//
// The products run on tcgen05 with accumulators in TMEM, one kernel with three epilogues.  Pairs of thread blocks
// (cta_group::2) take tiles of 256 x 256 in turn, each block with its 128 rows of both operands: in each, warp 0 issues TMA
// loads into a 6-stage ring (64 of the contraction a stage) and warps 4-11 empty one of two 256-column accumulators while
// the other is filled; warp 1 of the first block issues the MMAs for both.  A single block's tile of 128 x 256 takes 96 bytes
// a clock from L2 where a pair takes 64, and its MMAs waited for loads a quarter of the time (16384 x 50280 x 768: the
// product with W 488 -> 456 us, 90 % of the tensor pipe's cycles; the forward 849 -> 844 us, 1.5 PFLOP/s).
// Either operand may have the contraction along its rows (z) or across them (dz W, dz^T H): both are 128-byte
// swizzled tiles, of K-major or of MN-major layout.
//
// float32 operands are split into three bfloat16 (8 bits of mantissa each) and multiplied as six products of the
// planes, the small ones first; what is left out is below 2^-24.  (An infinite float32 operand gives NaN
// where its product with the rest of a split is none.)
//
// The tensor core truncates when it adds into its accumulator, an error to one side that grows with the length of the chain: over
// 8192 features a loss came out 3e-5 too small.  So the contractions of float32 are cut into chains of at most kSegSteps stages, and that of z into
// chains of kSegSteps16 for 16-bit operands, whose sums are added up in the epilogue's registers, rounded to nearest (through
// memory they cost dz W 32 us of 204 at 2031 x 16411 x 509).  The gradients of 16-bit operands are rounded to 2^-8 or 2^-11 and stay one
// chain, and so does z where one chain holds it: cut in two, the forward over 2048 features takes 2.5 % longer (333 x 50280 float16
// 88.1 -> 90.5 us, 4096 x 50280 bfloat16 543 -> 557 us).
//
// Measured (one B200, 16384 x 50280 x 768 bfloat16, forward and backward 4.34 ms, 1.17 PFLOP/s over the four products, under the power
// limit as a library product would be): z and its log-sum-exp 827-844 us (tensor pipe 82 %), the two pieces of dz 479 us each
// (74 %: the epilogue's stores), dz W 439-456 us each (90 %), dz^T H 510 and 438 us (80 %: 297
// tiles on 74 pairs), with pieces of equal size; cut as piece_of does, 65 us less for the whole.  float32,
// 2031 x 16411 x 509: 0.82 ms, six times the products: z 131 us, dz 153, dz W 163, dz^T H 171, operands split in both passes 57.
#include "common.cuh"
#include "dispatch.h"
#include "tc_common.cuh"
#include <algorithm>
#include <cstring>

namespace b200 {
namespace {

using namespace tc;

__device__ int g_lce_status = 0;

constexpr int TM = 128, TN = 256, TK = 64;       // a block's rows of the result, columns, contraction of a stage
constexpr int NST = 6;
constexpr int A_BYTES = TM * TK * 2, B_BYTES = TN / 2 * TK * 2;      // a block's half of the pair's operands
constexpr int ST_BYTES = A_BYTES + B_BYTES;      // 32 KB
constexpr int STAGING = 32 * 128;                // a warp's 32 rows x 64 columns of dz on their way out
constexpr int LCE_THREADS = 384;                 // 4 warps that issue, 8 that empty accumulators
constexpr int LCE_SMEM = NST * ST_BYTES + 8 * STAGING + 1024;
constexpr uint32_t LCE_WAIT = 1u << 24;
constexpr int64_t kPieceBytes = int64_t(1) << 30;
constexpr int kSegSteps = 8;              // float32: most stages (of 64) of the contraction in one accumulation chain, which has their six products
constexpr int kSegSteps16 = 16;           // float16 and bfloat16: the same of z
constexpr int kPieceStages = 64;           // what a piece costs besides, in stages: launches, the sums of dH read and written
constexpr int kMaxSplits = 32;            // blocks that share the contraction of a tile

enum { EPI_LSE = 0, EPI_DZ = 1, EPI_OUT = 2 };

struct LceGemm {
  CUtensorMap a, b, out;       // (inner, rows, plane); out: dz
  int mt, nt, nk;              // tiles, stages of 64 along the contraction
  int seg;                     // stages a chain, nk where it is not cut
  int passes;                  // 1, or 6 products of the planes of a split
  int a_mn, b_mn;              // operand has the contraction across its rows
  int b_row0;                  // first row (K-major) of the piece within W
  int bk_row0;                 // the same where W's rows are the contraction
  uint32_t idesc;
  // epilogues
  int rows, cols;              // of the result
  int64_t classes, ignore_index;
  const int64_t *labels;
  float2 *part;                // LSE: (slot, rows)
  float *target;               // LSE: (rows)
  const float *lse, *rs, *common;
  int col0;                    // first class of this piece
  int dtype;                   // of the operands and gradients
  float *acc;                  // OUT: float32 sums, pitch acc_rs
  int64_t acc_rs;
  void *dst;
  int64_t dst_rs;
  int add, last;               // OUT: acc holds earlier pieces; this is the last one
  int splits, per;             // OUT: blocks that share a tile's contraction, and their stages; each has its sums at acc + split rows acc_rs
};

__device__ __forceinline__ void tma_st_3d(const CUtensorMap *map, const void *src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x),
               "r"(y), "r"(z), "r"(smem_u32(src))
               : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the first block's barrier at the place of `bar` in this one's shared memory
__device__ __forceinline__ uint32_t of_first(const uint64_t *bar) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(bar)));
  return a;
}
__device__ __forceinline__ void arrive_at(uint32_t bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
// a load into this block's shared memory that counts on a barrier of the pair
__device__ __forceinline__ void tma_3d_pair(void *dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// arrives at both blocks' barrier once the products issued so far are done
__device__ __forceinline__ void commit_pair(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct LcePipe {
  uint64_t full[NST], empty[NST], acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  int fail;
};

// planes of a product of splits: the small ones first
__device__ __forceinline__ int plane_a(int passes, int p) { return passes == 1 ? 0 : (0x021010 >> (4 * (5 - p))) & 15; }
__device__ __forceinline__ int plane_b(int passes, int p) { return passes == 1 ? 0 : (0x201100 >> (4 * (5 - p))) & 15; }

// The largest finite |s_r|, which dz is kept in units of; 1 where there is none to divide by.
__device__ __forceinline__ float unit_of(const float *common) {
  const float c = *common;
  return c > 0.f ? c : 1.f;
}
// A float16 dz, at most 1 in that unit, is kept 2^15 times as large, near the top of the type's range (65504): its probabilities would
// otherwise lie in the lower half of the range, and at 50280 classes the mean one below the smallest normal number, 2^-14.
__host__ __device__ constexpr float dz_up(int dtype) { return dtype == B200_F16 ? 32768.f : 1.f; }
// what a sum over dz is multiplied by
__device__ __forceinline__ float unit_back(const float *common, int dtype) { return unit_of(common) / dz_up(dtype); }

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// 64 columns of this warp's 32 rows, a row per lane, into the swizzled staging tile and out
template <typename T>
__device__ __forceinline__ void store_dz(const LceGemm &p, unsigned char *staging, const float (&v)[64], int col, int row, int plane, int lane) {
  if (lane == 0) bulk_wait_read<0>();
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint4 w;
    w.x = pack2<T>(v[8 * j], v[8 * j + 1]);
    w.y = pack2<T>(v[8 * j + 2], v[8 * j + 3]);
    w.z = pack2<T>(v[8 * j + 4], v[8 * j + 5]);
    w.w = pack2<T>(v[8 * j + 6], v[8 * j + 7]);
    *reinterpret_cast<uint4 *>(staging + lane * 128 + ((j ^ (lane & 7)) << 4)) = w;
  }
  fence_proxy_async();
  __syncwarp();
  if (lane == 0 && col < p.cols && row < p.rows) {
    tma_st_3d(&p.out, staging, col, row, plane);
    bulk_commit();
  }
}

template <typename T> __device__ __forceinline__ void store_row(T *dst, const float (&v)[32], int n, bool vec) {
  if (vec && n >= 32) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      reinterpret_cast<uint4 *>(dst)[j] = make_uint4(pack2<T>(v[8 * j], v[8 * j + 1]), pack2<T>(v[8 * j + 2], v[8 * j + 3]),
                                                     pack2<T>(v[8 * j + 4], v[8 * j + 5]), pack2<T>(v[8 * j + 6], v[8 * j + 7]));
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < n) {
        const uint32_t w = pack2<T>(v[j], 0.f);
        reinterpret_cast<uint16_t *>(dst)[j] = (uint16_t)w;
      }
  }
}

// CUT: the contraction of a tile is more than one chain, whose sums are kept in registers
template <int EPI, bool CUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(LCE_THREADS, 1) lce_gemm_kernel(const __grid_constant__ LceGemm p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ LcePipe pipe;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tiles = p.mt * p.nt * (EPI >= EPI_OUT ? p.splits : 1), pairs = gridDim.x >> 1, pair = blockIdx.x >> 1;
  const int rank = (int)cluster_rank();
  if (tid == 0) {
    for (int s = 0; s < NST; ++s) {
      mbar_init(&pipe.full[s], 1);
      mbar_init(&pipe.empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&pipe.acc_full[s], 1);
      mbar_init(&pipe.acc_empty[s], 16);               // the epilogue warps of both blocks
    }
    pipe.fail = 0;
    mbar_fence_init();
    fence_proxy_async();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&pipe.tmem_base)), "r"(2 * TN) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();                                      // the other block's barriers are set up
  tc_fence_after();
  const uint32_t tmem = pipe.tmem_base;
  // z and dz: neighbouring blocks share W's tile; products of dz: they share dz's
  const auto m_of = [&](int t) { return EPI >= EPI_OUT ? t / p.nt % p.mt : t % p.mt; };
  const auto n_of = [&](int t) { return EPI >= EPI_OUT ? t % p.nt : t / p.mt; };
  // the stages of a block's part of the contraction
  const auto k_from = [&](int t) { return EPI >= EPI_OUT ? t / (p.nt * p.mt) * p.per : 0; };
  const auto k_to = [&](int t) { return EPI >= EPI_OUT ? min(p.nk, k_from(t) + p.per) : p.nk; };

  if (warp == 0 && lane == 0) {
    // ------------------------------------------------------------------ loads
    int g = 0;
    bool ok = true;
    for (int t = pair; t < tiles && ok; t += pairs) {
      const int m0 = (m_of(t) * 2 + rank) * TM, n0 = n_of(t) * TN + rank * (TN / 2);      // this block's halves
      const int ke = k_to(t);
      for (int k0 = k_from(t); k0 < ke && ok; k0 += p.seg) {
        const int k1 = min(ke, k0 + p.seg);
        for (int ps = 0; ps < p.passes && ok; ++ps) {
          const int pa = plane_a(p.passes, ps), pb = plane_b(p.passes, ps);
          for (int k = k0; k < k1; ++k, ++g) {
            const int s = g % NST;
            if (g >= NST && !mbar_wait(&pipe.empty[s], ((g / NST) - 1) & 1, LCE_WAIT)) { ok = false; break; }
            unsigned char *st = smem + (size_t)s * ST_BYTES;
            const uint32_t full = of_first(&pipe.full[s]);
            if (rank == 0) mbar_expect_tx(&pipe.full[s], 2 * ST_BYTES);      // of both blocks
            if (p.a_mn) {
#pragma unroll
              for (int j = 0; j < TM / 64; ++j) tma_3d_pair(st + j * 8192, &p.a, m0 + 64 * j, k * TK, pa, full);
            } else {
              tma_3d_pair(st, &p.a, k * TK, m0, pa, full);
            }
            if (p.b_mn) {
#pragma unroll
              for (int j = 0; j < TN / 128; ++j) tma_3d_pair(st + A_BYTES + j * 8192, &p.b, n0 + 64 * j, p.bk_row0 + k * TK, pb, full);
            } else {
              tma_3d_pair(st + A_BYTES, &p.b, k * TK, p.b_row0 + n0, pb, full);
            }
          }
        }
      }
    }
    if (!ok) {
      atomicExch(&pipe.fail, 1);
      for (int i = 0; i < 1 << 12; ++i) __nanosleep(256);        // copies in flight: a millisecond, many times what they take
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ------------------------------------------------------------------ products
    int g = 0, ch = 0;
    bool ok = true;
    const uint32_t a_lbo = p.a_mn ? 8192 : 16, b_lbo = p.b_mn ? 8192 : 16;
    const uint32_t a_step = p.a_mn ? 2048 : 32, b_step = p.b_mn ? 2048 : 32;      // bytes to the next 16 of the contraction
    for (int t = pair; t < tiles && ok; t += pairs) {
      const int ke = k_to(t);
      for (int k0 = k_from(t); k0 < ke && ok; k0 += p.seg, ++ch) {
        const int n = (min(ke, k0 + p.seg) - k0) * p.passes;
        const uint32_t d = tmem + (ch & 1) * TN;
        if (ch >= 2 && !mbar_wait(&pipe.acc_empty[ch & 1], ((ch >> 1) - 1) & 1, LCE_WAIT)) { ok = false; break; }
        tc_fence_after();
        for (int i = 0; i < n; ++i, ++g) {
          const int s = g % NST;
          if (!mbar_wait(&pipe.full[s], (g / NST) & 1, LCE_WAIT)) { ok = false; break; }
          tc_fence_after();
          const uint32_t st = smem_u32(smem + (size_t)s * ST_BYTES);
#pragma unroll
          for (int kk = 0; kk < TK / 16; ++kk)
            mma_pair(d, smem_desc(st + kk * a_step, a_lbo, 1024, 2), smem_desc(st + A_BYTES + kk * b_step, b_lbo, 1024, 2), p.idesc, i > 0 || kk > 0 ? 1u : 0u);
          commit_pair(&pipe.empty[s]);
        }
        if (ok) commit_pair(&pipe.acc_full[ch & 1]);
      }
    }
    if (!ok) atomicExch(&pipe.fail, 1);
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ epilogues
    const int q = warp & 3, half = (warp - 4) >> 2;
    unsigned char *staging = smem + NST * ST_BYTES + (warp - 4) * STAGING;
    int ch = 0;
    bool ok = true;
    for (int t = pair; t < tiles && ok; t += pairs) {
      const int m0 = (m_of(t) * 2 + rank) * TM, n0 = n_of(t) * TN;
      const int row = m0 + q * 32 + lane, c0 = n0 + half * (TN / 2);      // this thread's row and 128 columns
      const bool in = row < p.rows;
      const int kb = k_from(t), ke = k_to(t);
      float sums[CUT ? TN / 64 : 1][32] = {};
      for (int k0 = kb; k0 < ke; k0 += p.seg, ++ch) {
        const bool whole = !CUT || k0 + p.seg >= ke;                     // the tile's last chain
        // what the epilogue needs besides is loaded before the wait
        float lse2 = 0.f, sc = 0.f;
        int at = -1;                                                     // the label's column within this thread's columns
        if (EPI < EPI_OUT && in && whole) {
          const int64_t label = p.labels[row];
          if (label != p.ignore_index && label >= 0 && label < p.classes) {
            const int64_t c = label - p.col0 - c0;
            if (c >= 0 && c < TN / 2) at = (int)c;
          }
          if (EPI == EPI_DZ) {
            lse2 = p.lse[row] * kLog2e;
            sc = p.rs[row] / unit_of(p.common) * dz_up(p.dtype);
          }
        }
        if (!mbar_wait(&pipe.acc_full[ch & 1], (ch >> 1) & 1, LCE_WAIT)) { ok = false; break; }
        tc_fence_after();
        const uint32_t ta = tmem + (ch & 1) * TN + ((uint32_t)(q * 32) << 16) + half * (TN / 2);
        const auto emptied = [&]() {                                     // the accumulator has been read
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_at(of_first(&pipe.acc_empty[ch & 1]));
        };
        if constexpr (CUT) {
#pragma unroll
          for (int c = 0; c < TN / 32; ++c) {           // 16 at a time: with 32 more registers beside the 128 sums are spilled
            float v[16];
            __syncwarp();                              // lanes come from their own waits, and from the last tile's stores
            tmem_ld16(ta + c * 16, v);
#pragma unroll
            for (int j = 0; j < 16; ++j) sums[c >> 1][(c & 1) * 16 + j] += v[j];
          }
          emptied();
          if (!whole) continue;
        }
        if constexpr (EPI == EPI_LSE) {
          float m = -INFINITY, sum = 0.f, target = 0.f;                   // m in units of log2
          const auto take = [&](float (&v)[32], int c) {
            const int left = p.cols - (c0 + c * 32);
            if (left < 32) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = j < left ? v[j] : -INFINITY;
            }
            if ((at >> 5) == c) {
              const uint32_t one = 1u << (at & 31);                       // (an index into v would put all of it into memory)
#pragma unroll
              for (int j = 0; j < 32; ++j) target = one & (1u << j) ? v[j] : target;
            }
            float vm = v[0];
#pragma unroll
            for (int j = 1; j < 32; ++j) vm = fmaxf(vm, v[j]);
            const float nm = fmaxf(m, vm * kLog2e), off = nm == -INFINITY ? 0.f : nm;
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              s0 += ex2(fmaf(v[j], kLog2e, -off));
              s1 += ex2(fmaf(v[j + 1], kLog2e, -off));
            }
            sum = fmaf(sum, ex2(m - off), s0 + s1);                       // the first time 0 * 2^-inf
            m = nm;
          };
#pragma unroll
          for (int c = 0; c < TN / 64; ++c) {
            if constexpr (CUT) {
              take(sums[c], c);
            } else {
              float v[32];
              __syncwarp();
              tmem_ld32(ta + c * 32, v);
              take(v, c);
            }
          }
          if constexpr (!CUT) emptied();
          if (in) {
            p.part[(int64_t)(n_of(t) * 2 + half) * p.rows + row] = make_float2(m, sum);
            if (at >= 0) p.target[row] = target;
          }
        } else if constexpr (EPI == EPI_DZ) {
          const auto give = [&](float (&v)[64], int c) {
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = ex2(fmaf(v[j], kLog2e, -lse2));
            if ((at >> 6) == c) {
#pragma unroll
              for (int j = 0; j < 64; ++j) v[j] = j == (at & 63) ? v[j] - 1.f : v[j];
            }
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = sc == 0.f ? 0.f : v[j] * sc;
            const int col = c0 + c * 64, r0 = m0 + q * 32;
            if (p.dtype == B200_BF16) store_dz<__nv_bfloat16>(p, staging, v, col, r0, 0, lane);
            else if (p.dtype == B200_F16) store_dz<__half>(p, staging, v, col, r0, 0, lane);
            else {
#pragma unroll 1
              for (int pl = 0; pl < 3; ++pl) {
                store_dz<__nv_bfloat16>(p, staging, v, col, r0, pl, lane);
#pragma unroll
                for (int j = 0; j < 64; ++j) v[j] -= __bfloat162float(__float2bfloat16_rn(v[j]));
              }
            }
          };
          if constexpr (CUT) {
#pragma unroll
            for (int c = 0; c < TN / 128; ++c) give(*reinterpret_cast<float(*)[64]>(sums[2 * c]), c);
          } else {
#pragma unroll 1
            for (int c = 0; c < TN / 128; ++c) {
              float v[64];
              __syncwarp();
              tmem_ld32(ta + c * 64, *reinterpret_cast<float(*)[32]>(v));
              tmem_ld32(ta + c * 64 + 32, *reinterpret_cast<float(*)[32]>(v + 32));
              give(v, c);
            }
            emptied();
          }
        } else {
          float *acc = p.acc + (int64_t)(t / (p.nt * p.mt)) * p.rows * p.acc_rs;
          const float unit = unit_back(p.common, p.dtype);
          if constexpr (CUT) {
            // 32 x 32 of them, a row a lane, are turned over in shared memory, so that a row leaves as one line
            float *turn = reinterpret_cast<float *>(staging);
            const int r0 = m0 + q * 32, n = min(32, p.rows - r0);
#pragma unroll
            for (int c = 0; c < TN / 64; ++c) {
              const int col = c0 + c * 32 + lane;
              __syncwarp();
#pragma unroll
              for (int j = 0; j < 32; ++j) turn[lane * 32 + (j ^ lane)] = sums[c][j];
              __syncwarp();
              if (col >= p.cols) continue;
              float *sum = acc + (int64_t)r0 * p.acc_rs + col, *dst = reinterpret_cast<float *>(p.dst) + (int64_t)r0 * p.dst_rs + col;
#pragma unroll 8
              for (int i = 0; i < n; ++i) {
                float x = turn[i * 32 + (lane ^ i)];
                if (p.add) x += sum[i * p.acc_rs];
                if (p.last) dst[i * p.dst_rs] = x * unit;
                else sum[i * p.acc_rs] = x;
              }
            }
          } else {
            // one chain: a row a lane, which writes the whole line of a bfloat16 or float16 row by itself
            const bool vec = (p.dst_rs * 2) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.dst) & 15) == 0;
#pragma unroll 1
            for (int c = 0; c < TN / 64; ++c) {
              float v[32];
              __syncwarp();
              tmem_ld32(ta + c * 32, v);
              const int col = c0 + c * 32, n = min(32, p.cols - col);
              if (!in || n <= 0) continue;
              float4 *o = reinterpret_cast<float4 *>(acc + (int64_t)row * p.acc_rs + col);
              if (p.add) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                  if (4 * j < n) {
                    const float4 w = o[j];
                    v[4 * j] += w.x;
                    v[4 * j + 1] += w.y;
                    v[4 * j + 2] += w.z;
                    v[4 * j + 3] += w.w;
                  }
              }
              if (!p.last) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                  if (4 * j < n) o[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
              } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] *= unit;
                const int64_t i = (int64_t)row * p.dst_rs + col;
                if (p.dtype == B200_BF16) store_row<__nv_bfloat16>(reinterpret_cast<__nv_bfloat16 *>(p.dst) + i, v, n, vec);
                else store_row<__half>(reinterpret_cast<__half *>(p.dst) + i, v, n, vec);
              }
            }
            emptied();
          }
        }
      }
    }
    if (EPI == EPI_DZ && lane == 0) bulk_wait<0>();
    if (!ok) atomicExch(&pipe.fail, 1);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();                                      // neither block leaves while the other uses its memory
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * TN) : "memory");
  if (tid == 0 && pipe.fail) atomicExch(&g_lce_status, 7);
}

__device__ __forceinline__ bool is_target(int64_t label, int64_t ignore, int classes) { return label != ignore && label >= 0 && label < classes; }

// Rows of 16-byte pitch from rows of any: a copy for 16-bit types, three bfloat16 planes for float32.  With labels, rows without a
// target become zeros: whatever they hold (NaN in the padding of a batch) is then in no product.
__global__ void __launch_bounds__(256) lce_pack_kernel(const void *src, int64_t rs, int64_t rows, int cols, int pitch, int split, int wide, const int64_t *labels,
                                                      int64_t ignore, int classes, uint16_t *dst) {
  const int per = pitch / (wide ? 8 : 2);
  const int64_t n = rows * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * (wide ? 8 : 2);
    const bool on = !labels || is_target(labels[r], ignore, classes);
    if (wide) {                                          // 16-bit rows of 16-byte pitch
      uint4 w = make_uint4(0, 0, 0, 0);
      if (on) {
        w = __ldg(reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(src) + r * rs + c));
        uint32_t *x = reinterpret_cast<uint32_t *>(&w);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + j >= cols) x[j >> 1] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
      }
      *reinterpret_cast<uint4 *>(dst + r * pitch + c) = w;
    } else if (!split) {
      const uint16_t *s = reinterpret_cast<const uint16_t *>(src) + r * rs;
      const uint32_t lo = on && c < cols ? s[c] : 0, hi = on && c + 1 < cols ? s[c + 1] : 0;
      *reinterpret_cast<uint32_t *>(dst + r * pitch + c) = lo | hi << 16;
    } else {
      const float *s = reinterpret_cast<const float *>(src) + r * rs;
      float a = on && c < cols ? s[c] : 0.f, b = on && c + 1 < cols ? s[c + 1] : 0.f;
#pragma unroll
      for (int pl = 0; pl < 3; ++pl) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        *reinterpret_cast<__nv_bfloat162 *>(dst + ((int64_t)pl * rows + r) * pitch + c) = v;
        a = isfinite(a) ? a - __bfloat162float(v.x) : 0.f;
        b = isfinite(b) ? b - __bfloat162float(v.y) : 0.f;
      }
    }
  }
}

// Joins the partial maxima and sums of 32 rows: a warp reads the same slot of 32 rows.
constexpr int JOIN_WARPS = 32;
__global__ void __launch_bounds__(JOIN_WARPS * 32) lce_join_kernel(const float2 *part, const float *target, const int64_t *labels, int64_t ignore, int classes, int rows,
                                                                  int slots, float *lse, float *loss) {
  __shared__ float2 sh[JOIN_WARPS][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, row = blockIdx.x * 32 + lane;
  float m = -INFINITY, s = 0.f;
  const auto join = [&](float2 v) {
    const float nm = fmaxf(m, v.x), off = nm == -INFINITY ? 0.f : nm;
    s = s * ex2(m - off) + v.y * ex2(v.x - off);
    m = nm;
  };
  if (row < rows) {
#pragma unroll 8
    for (int i = w; i < slots; i += JOIN_WARPS) join(part[(int64_t)i * rows + row]);
  }
  sh[w][lane] = make_float2(m, s);
  __syncthreads();
  const int r = blockIdx.x * 32 + w;                   // a warp a row
  const float2 v = sh[lane][w];
  m = v.x;
  s = v.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) join(make_float2(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o)));
  if (lane == 0 && r < rows) {
    const float l = m / kLog2e + logf(s);
    lse[r] = l;
    loss[r] = is_target(labels[r], ignore, classes) ? l - target[r] : 0.f;
  }
}

// Sum of the rows' losses (over the count of labels that are not ignored), one block in a fixed order.
__global__ void __launch_bounds__(1024) lce_sum_kernel(const float *loss, const int64_t *labels, int64_t ignore, int rows, int mean, float *out, float *count) {
  __shared__ double ss[32];
  __shared__ int sc[32];
  double s = 0.0;
  int n = 0;
#pragma unroll 4
  for (int i = threadIdx.x; i < rows; i += 1024) {
    s += (double)loss[i];
    n += labels[i] != ignore;
  }
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  if (lane == 0) { ss[w] = s; sc[w] = n; }
  __syncthreads();
  if (w == 0) {
    s = ss[lane];
    n = sc[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      n += __shfl_xor_sync(0xffffffffu, n, o);
    }
    if (lane == 0) {
      const int c = n > 0 ? n : 1;
      if (count) *count = (float)c;
      if (out) *out = (float)(mean ? s / c : s);
    }
  }
}

// s_r, and the largest finite |s_r| by an atomic maximum of its bits (any order gives the same; the word was cleared).
__global__ void __launch_bounds__(256) lce_scale_kernel(const float *dloss, int per_row, const float *count, const int64_t *labels, int64_t ignore, int classes,
                                                       int rows, float *rs, unsigned *common) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  float s = 0.f;
  if (r < rows) {
    if (is_target(labels[r], ignore, classes)) s = dloss[per_row ? r : 0] / (count ? *count : 1.f);
    rs[r] = s;
  }
  const unsigned m = __reduce_max_sync(0xffffffffu, isfinite(s) ? __float_as_uint(fabsf(s)) : 0u);
  if ((threadIdx.x & 31) == 0 && m) atomicMax(common, m);
}

// The blocks' parts of a product, added up in their order, scaled and rounded.
__global__ void __launch_bounds__(256) lce_fold_kernel(const float *acc, int splits, int64_t rows, int cols, int64_t acc_rs, const float *common, int dtype, void *dst,
                                                      int64_t dst_rs) {
  const int64_t n = rows * (acc_rs / 4), plane = rows * acc_rs;
  const float unit = unit_back(common, dtype);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / (acc_rs / 4);
    const int c = (int)(i - r * (acc_rs / 4)) * 4;
    const float *a = acc + r * acc_rs + c;
    float4 s = *reinterpret_cast<const float4 *>(a);
#pragma unroll 4
    for (int k = 1; k < splits; ++k) {
      const float4 w = *reinterpret_cast<const float4 *>(a + k * plane);
      s.x += w.x;
      s.y += w.y;
      s.z += w.z;
      s.w += w.w;
    }
    const float v[4] = {s.x * unit, s.y * unit, s.z * unit, s.w * unit};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < cols) st_act(dst, dtype, r * dst_rs + c + j, v[j]);
  }
}

// ------------------------------------------------------------------------------------------------ host

int64_t up(int64_t n, int64_t unit) { return (n + unit - 1) / unit * unit; }

bool map16(CUtensorMap *m, int dtype, const void *base, uint64_t inner, uint64_t rows, uint64_t pitch, int planes, uint32_t box_rows) {
  EncodeTiledFn enc = encoder();
  if (!enc) return false;
  const cuuint64_t dims[3] = {inner, rows, (cuuint64_t)planes};
  const cuuint64_t strides[2] = {pitch * 2, pitch * 2 * rows};
  const cuuint32_t box[3] = {64, box_rows, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return enc(m, dtype == B200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// how the operands are read: in place where their rows allow TMA, else from packed (or split) copies
struct Plan {
  int planes, Dp;
  bool pack_h, pack_w;
  int64_t pack_bytes_h, pack_bytes_w;
  int piece, n_pieces;            // columns of dz at a time (a multiple of 256), pieces
  int64_t dz_pitch, dz_bytes, acc_h_bytes, acc_w_bytes;
  int64_t Da;                     // pitch of the float32 sums
  int seg;
  int splits_h, per_h, splits_w, per_w;
};

// How many blocks share the contraction of `stages` for each of `tiles` tiles: as few as fill the SMs (at least 8 stages
// each, to be worth 128 KB of sums).
// Returns the stages that pass until all is done.
int64_t split_of(int64_t tiles, int stages, int &splits, int &per) {
  const int64_t pairs = sm_count_current() / 2;
  splits = 1;
  per = stages;
  int64_t best = (tiles + pairs - 1) / pairs * stages;
  for (int s = 2; s <= kMaxSplits && stages / s >= 8 && tiles * (s - 1) < pairs; ++s) {
    const int p = (stages + s - 1) / s;
    if ((int64_t)(s - 1) * p >= stages) continue;
    const int64_t cost = (tiles * s + pairs - 1) / pairs * p;
    if (cost * 100 < best * 90) { best = cost; splits = s; per = p; }
  }
  return best;
}

// The classes of a piece, in tiles of 256, where dz has to be made in pieces of at most `most`: the number for which the
// products with dz, taken a wave of tiles after the other, take the fewest stages (16384 x 50280 x 768 on 74 pairs: pieces
// of 99 and 98 leave dz^T H one tile for a fifth wave, 510 + 438 us; 123 and 74 fill five and three, see the figures above).
int64_t piece_of(const b200_lce_args &a, int64_t total, int64_t most) {
  if (total <= most) return total;
  const int64_t least = (total + (total + most - 1) / most) / ((total + most - 1) / most + 1), step = most / 256 + 1;
  const int64_t dt = (a.features + TN - 1) / TN, mt = (a.rows + 2 * TM - 1) / (2 * TM), pairs = sm_count_current() / 2;
  int64_t best = most, cost = INT64_MAX;
  for (int64_t p = most; p >= least; p -= step) {
    const int64_t full = total / p, rest = total % p;
    int s, per;
    int64_t c = (mt * total / pairs + full + 1) * ((a.features + TK - 1) / TK) + (full + (rest > 0)) * kPieceStages;
    c += full * split_of(mt * dt, (int)(p * (TN / TK)), s, per);
    if (rest) c += (mt * dt * s + pairs - 1) / pairs * std::min<int64_t>(per, rest * (TN / TK));
    c += full * split_of(p * dt, (int)((a.rows + TK - 1) / TK), s, per);
    if (rest) c += (rest * dt * s + pairs - 1) / pairs * per;                      // a last, smaller piece is split as the others
    if (c < cost) { cost = c; best = p; }
  }
  return best;
}

bool in_place(const void *p, int64_t rs, int cols) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && rs % 8 == 0 && rs >= cols && rs < (int64_t(1) << 36);
}

Plan plan_of(const b200_lce_args &a, bool bwd) {
  Plan q;
  const bool f32 = a.dtype == B200_F32;
  q.planes = f32 ? 3 : 1;
  q.Dp = (int)up(a.features, 8);
  q.pack_h = f32 || bwd || !in_place(a.hidden, a.hidden_rs, a.features);      // backwards: a copy without the rows that have no target
  q.pack_w = f32 || !in_place(a.weight, a.weight_rs, a.features);
  q.pack_bytes_h = q.pack_h ? up(2 * q.planes * a.rows * q.Dp, 256) : 0;
  q.pack_bytes_w = q.pack_w ? up(2 * q.planes * (int64_t)a.classes * q.Dp, 256) : 0;
  q.seg = f32 ? kSegSteps : 1 << 30;
  q.Da = up(a.features, 4);
  const int64_t most = kPieceBytes / (2 * q.planes * a.rows) / TN;
  q.piece = bwd ? (int)piece_of(a, (a.classes + TN - 1) / TN, most < 1 ? 1 : most) * TN : TN;
  q.n_pieces = (a.classes + q.piece - 1) / q.piece;
  q.dz_pitch = q.piece;
  q.dz_bytes = up(2 * q.planes * a.rows * q.dz_pitch, 256);
  const int64_t dt = (a.features + TN - 1) / TN;
  // by the stages of the first piece, which has all the classes where it is the only one: each of its blocks has a part then, and writes its sums
  split_of((a.rows + 2 * TM - 1) / (2 * TM) * dt, (std::min(q.piece, a.classes) + TK - 1) / TK, q.splits_h, q.per_h);
  split_of((q.piece + 2 * TM - 1) / (2 * TM) * dt, (int)((a.rows + TK - 1) / TK), q.splits_w, q.per_w);
  // float32 sums: of dH over the pieces and the blocks that share a tile, of dW over the blocks
  q.acc_h_bytes = q.n_pieces > 1 || q.splits_h > 1 ? up(4 * q.splits_h * a.rows * q.Da, 256) : 0;
  q.acc_w_bytes = q.splits_w > 1 ? up(4 * q.splits_w * (int64_t)q.piece * q.Da, 256) : 0;
  return q;
}

int slots_of(const b200_lce_args &a) { return (a.classes + TN - 1) / TN * 2; }

int check_lce(const b200_lce_args &a) {
  B200_REQUIRE(a.hidden && a.weight && a.labels, B200_ERR_NULL, "lce: hidden, weight and labels must be non-null");
  B200_REQUIRE(a.rows > 0 && a.classes > 0 && a.features > 0, B200_ERR_SHAPE, "lce: sizes must be positive");
  B200_REQUIRE(a.dtype == B200_F32 || a.dtype == B200_F16 || a.dtype == B200_BF16, B200_ERR_DTYPE, "lce: unknown dtype %d", a.dtype);
  B200_REQUIRE(a.reduction >= 0 && a.reduction <= 2, B200_ERR_DTYPE, "lce: unknown reduction %d", a.reduction);
  B200_REQUIRE(a.rows < (int64_t(1) << 30) && a.classes < (1 << 30) && a.features <= (1 << 20) &&
                   ((a.rows + TM - 1) / TM) * ((int64_t)(a.classes + TN - 1) / TN) < (int64_t(1) << 30),
               B200_ERR_SHAPE, "lce: sizes too large (rows %lld, classes %d, features %d)", (long long)a.rows, a.classes, a.features);
  B200_REQUIRE(a.hidden_rs >= a.features && a.weight_rs >= a.features, B200_ERR_SHAPE, "lce: row pitches must be at least the features");
  B200_REQUIRE((reinterpret_cast<uintptr_t>(a.work) & 255) == 0, B200_ERR_ALIGN, "lce: work must be 256-byte aligned");
  return 0;
}

int pack(const void *src, int64_t rs, int64_t rows, const b200_lce_args &a, const Plan &q, bool masked, void *dst, cudaStream_t st) {
  const bool wide = a.dtype != B200_F32 && in_place(src, rs, a.features) && rs >= q.Dp;
  const int64_t n = rows * (q.Dp / (wide ? 8 : 2));
  const int64_t blocks = (n + 255) / 256, most = (int64_t)sm_count_current() * 32;
  lce_pack_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, st>>>(src, rs, rows, a.features, q.Dp, a.dtype == B200_F32, wide,
                                                                            masked ? reinterpret_cast<const int64_t *>(a.labels) : nullptr, a.ignore_index, a.classes,
                                                                            reinterpret_cast<uint16_t *>(dst));
  return launch_status();
}

template <int EPI, bool CUT> int launch_gemm_of(const LceGemm &g, cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(lce_gemm_kernel<EPI, CUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, LCE_SMEM);
  if (e != cudaSuccess) { set_error("cudaFuncSetAttribute: %s", cudaGetErrorString(e)); return (int)e; }
  const int tiles = g.mt * g.nt * (EPI >= EPI_OUT ? g.splits : 1), sms = sm_count_current();
  lce_gemm_kernel<EPI, CUT><<<(unsigned)(2 * (tiles < sms / 2 ? tiles : sms / 2)), LCE_THREADS, LCE_SMEM, st>>>(g);
  return launch_status();
}

// (the sums of float32 gradients take the same path when they are one chain: their results leave a row a line)
template <int EPI> int launch_gemm(const LceGemm &g, cudaStream_t st) {
  const bool cut = EPI == EPI_OUT ? g.dtype == B200_F32 : g.seg < g.nk;
  return cut ? launch_gemm_of<EPI, true>(g, st) : launch_gemm_of<EPI, false>(g, st);
}

uint32_t idesc_of(int dtype, bool a_mn, bool b_mn) { return idesc_f16(dtype == B200_F16 ? 0u : 1u, a_mn, b_mn, 2 * TM, TN); }

int fold(const LceGemm &g, cudaStream_t st) {
  const int64_t n = (int64_t)g.rows * (g.acc_rs / 4), most = (int64_t)sm_count_current() * 16, blocks = (n + 255) / 256;
  lce_fold_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, st>>>(g.acc, g.splits, g.rows, g.cols, g.acc_rs, g.common, g.dtype, g.dst, g.dst_rs);
  return launch_status();
}

struct Operands { const void *h, *w; int64_t h_pitch, w_pitch; };

// z = H W^T for classes c0 .. c0 + cols
int gemm_z(LceGemm &g, const b200_lce_args &a, const Plan &q, const Operands &o, int c0, int cols) {
  memset(&g, 0, sizeof(g));
  B200_REQUIRE(map16(&g.a, a.dtype, o.h, a.features, a.rows, o.h_pitch, q.planes, TM) && map16(&g.b, a.dtype, o.w, a.features, a.classes, o.w_pitch, q.planes, TN / 2),
               B200_ERR_UNSUPPORTED, "lce: tensor-map encoding failed");
  g.mt = (int)((a.rows + 2 * TM - 1) / (2 * TM));
  g.nt = (cols + TN - 1) / TN;
  g.nk = (a.features + TK - 1) / TK;
  const int chains = (g.nk + (q.planes == 3 ? kSegSteps : kSegSteps16) - 1) / (q.planes == 3 ? kSegSteps : kSegSteps16);
  g.seg = (g.nk + chains - 1) / chains;
  g.passes = q.planes == 3 ? 6 : 1;
  g.b_row0 = c0;
  g.idesc = idesc_of(a.dtype, false, false);
  g.rows = (int)a.rows;
  g.cols = cols;
  g.classes = a.classes;
  g.ignore_index = a.ignore_index;
  g.labels = reinterpret_cast<const int64_t *>(a.labels);
  g.col0 = c0;
  g.dtype = a.dtype;
  return 0;
}

}  // namespace

int lce_status_read() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_lce_status, sizeof(int)) != cudaSuccess) return -1;
  return v;
}

}  // namespace b200

using namespace b200;

extern "C" int64_t b200_lce_fwd_work_bytes(const b200_lce_args *args) {
  if (!args || check_lce(*args)) return 0;
  const b200_lce_args &a = *args;
  const Plan q = plan_of(a, false);
  return q.pack_bytes_h + q.pack_bytes_w + up(8 * a.rows * slots_of(a), 256) + 2 * up(4 * a.rows, 256);
}

extern "C" int64_t b200_lce_bwd_work_bytes(const b200_lce_args *args) {
  if (!args || check_lce(*args)) return 0;
  const b200_lce_args &a = *args;
  const Plan q = plan_of(a, true);
  return q.pack_bytes_h + q.pack_bytes_w + q.dz_bytes + (a.dhidden ? q.acc_h_bytes : 0) + (a.dweight ? q.acc_w_bytes : 0) + up(4 * a.rows, 256) + 256;
}

extern "C" int b200_lce_fwd(const b200_lce_args *args, void *stream) {
  B200_REQUIRE(args, B200_ERR_NULL, "lce_fwd: null argument block");
  const b200_lce_args &a = *args;
  if (int e = check_lce(a)) return e;
  B200_REQUIRE(a.lse && a.loss && a.work && (a.reduction != 1 || a.count), B200_ERR_NULL, "lce_fwd: lse, loss, work and (for a mean) count must be non-null");
  const Plan q = plan_of(a, false);
  B200_REQUIRE(a.work_bytes >= b200_lce_fwd_work_bytes(args), B200_ERR_TOO_LARGE, "lce_fwd: work has %lld bytes, %lld are needed", (long long)a.work_bytes,
               (long long)b200_lce_fwd_work_bytes(args));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  unsigned char *w = reinterpret_cast<unsigned char *>(a.work);
  Operands o = {a.hidden, a.weight, a.hidden_rs, a.weight_rs};
  if (q.pack_h) { o.h = w; o.h_pitch = q.Dp; if (int e = pack(a.hidden, a.hidden_rs, a.rows, a, q, false, w, st)) return e; }
  w += q.pack_bytes_h;
  if (q.pack_w) { o.w = w; o.w_pitch = q.Dp; if (int e = pack(a.weight, a.weight_rs, a.classes, a, q, false, w, st)) return e; }
  w += q.pack_bytes_w;
  LceGemm g;
  if (int e = gemm_z(g, a, q, o, 0, a.classes)) return e;
  g.part = reinterpret_cast<float2 *>(w);
  w += up(8 * a.rows * slots_of(a), 256);
  g.target = reinterpret_cast<float *>(w);
  w += up(4 * a.rows, 256);
  float *row_loss = a.reduction == 0 ? reinterpret_cast<float *>(a.loss) : reinterpret_cast<float *>(w);
  if (int e = launch_gemm<EPI_LSE>(g, st)) return e;
  lce_join_kernel<<<(unsigned)((a.rows + 31) / 32), JOIN_WARPS * 32, 0, st>>>(g.part, g.target, g.labels, a.ignore_index, a.classes, (int)a.rows, slots_of(a),
                                                                reinterpret_cast<float *>(a.lse), row_loss);
  if (int e = launch_status()) return e;
  if (a.reduction != 0)
    lce_sum_kernel<<<1, 1024, 0, st>>>(row_loss, g.labels, a.ignore_index, (int)a.rows, a.reduction == 1, reinterpret_cast<float *>(a.loss),
                                       reinterpret_cast<float *>(a.count));
  return launch_status();
}

extern "C" int b200_lce_bwd(const b200_lce_args *args, void *stream) {
  B200_REQUIRE(args, B200_ERR_NULL, "lce_bwd: null argument block");
  const b200_lce_args &a = *args;
  if (int e = check_lce(a)) return e;
  B200_REQUIRE(a.lse && a.dloss && a.work && (a.reduction != 1 || a.count), B200_ERR_NULL, "lce_bwd: lse, dloss, work and (for a mean) count must be non-null");
  B200_REQUIRE(a.dhidden || a.dweight, B200_ERR_NULL, "lce_bwd: dhidden or dweight must be non-null");
  B200_REQUIRE((!a.dhidden || a.dhidden_rs >= a.features) && (!a.dweight || a.dweight_rs >= a.features), B200_ERR_SHAPE,
               "lce_bwd: row pitches must be at least the features");
  const Plan q = plan_of(a, true);
  B200_REQUIRE(a.work_bytes >= b200_lce_bwd_work_bytes(args), B200_ERR_TOO_LARGE, "lce_bwd: work has %lld bytes, %lld are needed", (long long)a.work_bytes,
               (long long)b200_lce_bwd_work_bytes(args));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  unsigned char *w = reinterpret_cast<unsigned char *>(a.work);
  Operands o = {a.hidden, a.weight, a.hidden_rs, a.weight_rs};
  o.h = w;
  o.h_pitch = q.Dp;
  if (int e = pack(a.hidden, a.hidden_rs, a.rows, a, q, true, w, st)) return e;
  w += q.pack_bytes_h;
  if (q.pack_w) { o.w = w; o.w_pitch = q.Dp; if (int e = pack(a.weight, a.weight_rs, a.classes, a, q, false, w, st)) return e; }
  w += q.pack_bytes_w;
  void *dz = w;
  w += q.dz_bytes;
  float *acc_h = reinterpret_cast<float *>(w);
  if (a.dhidden) w += q.acc_h_bytes;
  float *acc_w = reinterpret_cast<float *>(w);
  if (a.dweight) w += q.acc_w_bytes;
  float *rs = reinterpret_cast<float *>(w);
  w += up(4 * a.rows, 256);
  float *common = reinterpret_cast<float *>(w);
  cudaError_t ce = cudaMemsetAsync(common, 0, 4, st);
  if (ce != cudaSuccess) { set_error("cudaMemsetAsync: %s", cudaGetErrorString(ce)); return (int)ce; }
  lce_scale_kernel<<<(unsigned)((a.rows + 255) / 256), 256, 0, st>>>(reinterpret_cast<const float *>(a.dloss), a.reduction == 0,
                                                                    a.reduction == 1 ? reinterpret_cast<const float *>(a.count) : nullptr,
                                                                    reinterpret_cast<const int64_t *>(a.labels), a.ignore_index, a.classes, (int)a.rows, rs,
                                                                    reinterpret_cast<unsigned *>(common));
  if (int e = launch_status()) return e;
  const int esz = a.dtype == B200_F32 ? 4 : 2;
  for (int pc = 0; pc < q.n_pieces; ++pc) {
    const int c0 = pc * q.piece, cols = a.classes - c0 < q.piece ? a.classes - c0 : q.piece;
    LceGemm g;
    if (int e = gemm_z(g, a, q, o, c0, cols)) return e;
    B200_REQUIRE(map16(&g.out, a.dtype, dz, cols, a.rows, q.dz_pitch, q.planes, 32), B200_ERR_UNSUPPORTED, "lce: tensor-map encoding failed");
    g.lse = reinterpret_cast<const float *>(a.lse);
    g.rs = rs;
    g.common = common;
    if (int e = launch_gemm<EPI_DZ>(g, st)) return e;
    g.seg = q.seg;
    g.nt = (a.features + TN - 1) / TN;
    g.cols = a.features;
    g.acc_rs = q.Da;
    g.b_mn = 1;
    g.b_row0 = 0;
    if (a.dhidden) {                                             // dz W: contraction over the piece's classes
      B200_REQUIRE(map16(&g.a, a.dtype, dz, cols, a.rows, q.dz_pitch, q.planes, TM) && map16(&g.b, a.dtype, o.w, a.features, a.classes, o.w_pitch, q.planes, 64),
                   B200_ERR_UNSUPPORTED, "lce: tensor-map encoding failed");
      g.nk = (cols + TK - 1) / TK;
      g.splits = q.splits_h;                                     // of a shorter piece after the first some blocks have no part; their sums stay
      g.per = q.per_h;
      if (g.seg > g.nk) g.seg = g.nk;
      g.a_mn = 0;
      g.bk_row0 = c0;
      g.idesc = idesc_of(a.dtype, false, true);
      g.acc = acc_h;
      g.dst = a.dhidden;
      g.dst_rs = a.dhidden_rs;
      g.add = pc > 0;
      g.last = pc == q.n_pieces - 1 && g.splits == 1;
      if (int e = launch_gemm<EPI_OUT>(g, st)) return e;
      if (g.splits > 1 && pc == q.n_pieces - 1)
        if (int e = fold(g, st)) return e;
    }
    if (a.dweight) {                                             // dz^T H: contraction over the rows
      B200_REQUIRE(map16(&g.a, a.dtype, dz, cols, a.rows, q.dz_pitch, q.planes, 64) && map16(&g.b, a.dtype, o.h, a.features, a.rows, o.h_pitch, q.planes, 64),
                   B200_ERR_UNSUPPORTED, "lce: tensor-map encoding failed");
      g.mt = (cols + 2 * TM - 1) / (2 * TM);
      g.nk = (int)((a.rows + TK - 1) / TK);
      g.seg = q.seg < g.nk ? q.seg : g.nk;
      g.a_mn = 1;
      g.bk_row0 = 0;
      g.idesc = idesc_of(a.dtype, true, true);
      g.rows = cols;
      g.acc = acc_w;
      g.dst = reinterpret_cast<unsigned char *>(a.dweight) + (int64_t)c0 * a.dweight_rs * esz;
      g.dst_rs = a.dweight_rs;
      g.add = 0;
      g.splits = q.splits_w;
      g.per = q.per_w;
      g.last = g.splits == 1;
      if (int e = launch_gemm<EPI_OUT>(g, st)) return e;
      if (g.splits > 1)
        if (int e = fold(g, st)) return e;
    }
  }
  return 0;
}

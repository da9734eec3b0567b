// Linear attention with a decay for each head (b200_linattn_fwd / bwd / step), sm_100a.
//
//     S_t = exp(g_t) S_{t-1} + k_t v_t^T   (dk x dv, float32),      o_t = scale S_t^T q_t
//
// A sequence is walked in chunks of 64 or 128 steps.  With G_i the sum of g from the chunk's start to step i and S the state
// before the chunk,
//     o_i = exp(G_i) q_i S + sum_{j <= i} exp(G_i - G_j) (q_i . k_j) v_j,
//     S' = exp(G_end) S + sum_j exp(G_end - G_j) k_j v_j^T,
// products of small matrices.  Every exponent is a difference of sums of the same chunk and is formed from sums in two floats
// (48 bits), so that strong decays do not cost the weak ones their precision; a decay of -inf (an empty state) counts
// as one of -300, whose exponential is zero in float32 all the same.
//
// All the gradients are the same walk with the operands in other roles:
//     dq: (q, k, v) -> (do, v, k) forwards;   dk: (v, do, q) backwards;   dv: (k, q, do) backwards,
// where backwards in time the decay of a step is that of the step after it.  dg_t is the sum over all pairs of a step s
// before t and a step r not before it of (what s puts into the state) . (what r takes from it), decayed from s to r.
// Sums of q . dq - k . dk would give it too, but as a small difference of long sums (an error of 3.4e-6 where this has
// 6e-7); instead, for a chunk: pairs within it, from the products of their two scores; pairs with one step outside, from the
// dots of q with the state's part of dq and of k with that of dk; and pairs on both sides of it, from the product of
// the two walks' states, which they save every 512 steps.
//
// One thread block walks 64 output columns of a (batch, head); where these are too few for the GPU the sequence is cut
// into segments: a first pass forms each segment's own state, a scan joins them, and every segment then starts from the
// state that the earlier ones lead to.  A single pass with the state on the chip moves what the operands and results are, where
// a state written for every chunk would move several times that (8 x 2048 steps x 24 heads of 128 x 64: 100 MB of
// states beside 110 MB).
//
// Measured (one B200, bfloat16, 8 x 2048 steps, 24 heads, keys of 128 shared by all, values of 64): o and dv 114 us each,
// dq 234 us and dk 328 us (two blocks for the 128 columns, float32 results for each head, dots and states for the gradient
// of g), each alone, the two sums over the heads 37 us each; the whole forward and backward 818 us.  Bound by the latency of a chunk's
// chain (products, decays, products; 8900 clocks alone, 13000 with two blocks on an SM): issue slots 42-48 % busy, the tensor pipe
// 19-26 %, DRAM below 20 %.  With 192 blocks 44 of 148 SMs have two.  16 heads of 128 x 128 over 16384 steps: 9 segments, 83 +
// 131 us and the scan.
#include "common.cuh"
#include "dispatch.h"
#include "tc_common.cuh"
#include <algorithm>
#include <cstring>

namespace b200 {
namespace {

using namespace tc;

constexpr int CH = 64;                    // steps of a chunk
constexpr int DO = 64;                    // output columns of a block
constexpr int MAX_D = 128;
constexpr int PP = CH + 4, PV = DO + 8;   // pitches of scores and of values / state (in floats)
constexpr int kSnapSteps = 512;           // steps between the states that the gradient of g is anchored at
constexpr int kSnap = kSnapSteps / CH;
constexpr int kMaxSeg = 64;               // segments of a sequence

struct Walk {
  // operands (batch, length, heads or groups, size), sizes contiguous; strides in elements
  const void *q, *k, *v, *x;              // x: dotted with the result
  int64_t q_bs, q_ls, q_hs, k_bs, k_ls, k_hs, v_bs, v_ls, v_hs, x_bs, x_ls, x_hs;
  int q_div, k_div, v_div, x_div;         // head / div: which of the operand's heads
  const void *g;
  int64_t g_bs, g_ls, g_hs;
  int g_dtype;
  int batch, length, heads, di, dout;     // sizes of q, k and of v
  int ch, chunks, rev;                    // steps of a chunk; rev: from the last chunk to the first, and backwards within each
  float s_inter, s_intra, s_update;
  const float *s0;                        // state at the start: (batch, heads, di, dout) by strides
  int64_t s0_bs, s0_hs, s0_is, s0_os;
  float *last;                            // state at the end, nullable
  int64_t last_bs, last_hs, last_is, last_os;
  int last_decay;                         // rev: times exp(g_0)
  void *out;
  int64_t o_bs, o_ls, o_hs;
  int out_f32;
  // for the gradient of g, nullable together (x is given then)
  float *run;                             // (tile, batch heads, length): what the pairs of steps across each step give, within its chunk
  float *sum;                             // (tile, batch heads, chunks): sums of the dots of a chunk
  float *snap;                            // (batch heads, snapshots, di, dout): states at every kSnap-th border of chunks
  int tiles, nseg, seg_chunks;            // blocks for a sequence's columns; segments and their chunks
  float *seg;                             // (batch heads, nseg, di, dout): states
  double *seg_g;                          // (batch heads, nseg): sums of g
  int beside;                             // host: needs nothing of the walk launched before it
};

// The walks of a backward pass need nothing of one another: the next one's blocks take the places that the last blocks of
// this one leave free.  One block waits for the walk before at its end, so that a walk is complete only after those before
// it, and what follows the last one follows all.  8 x 2048 steps, 24 heads: 940 us one after the other, 856 from the shortest
// blocks to the longest, 818 from the longest to the shortest.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ float ex2a(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A sum in two floats (the second what the first leaves out): 48 bits, at a tenth of the latency of 64-bit arithmetic in a
// chain that a whole block waits for.  The error of a rounded sum by Knuth's two-sum (The Art of Computer Programming, 2, 4.2.2),
// numbers of two parts added as Dekker does (Numerische Mathematik 18, 1971).
struct Two { float h, l; };
__device__ __forceinline__ Two two(float x) { return Two{x, 0.f}; }
__device__ __forceinline__ Two operator+(Two a, Two b) {
  const float s = a.h + b.h, t = s - a.h;
  const float e = ((a.h - (s - t)) + (b.h - t)) + (a.l + b.l);
  const float h = s + e;
  return Two{h, e - (h - s)};
}
__device__ __forceinline__ Two operator-(Two a) { return Two{-a.h, -a.l}; }
__device__ __forceinline__ Two shfl_up2(Two a, int d) { return Two{__shfl_up_sync(0xffffffffu, a.h, d), __shfl_up_sync(0xffffffffu, a.l, d)}; }
__device__ __forceinline__ Two shfl_down2(Two a, int d) { return Two{__shfl_down_sync(0xffffffffu, a.h, d), __shfl_down_sync(0xffffffffu, a.l, d)}; }
__device__ __forceinline__ float minus(Two a, Two b) { return (a.h - b.h) + (a.l - b.l); }
// 2^x in 64 bits: the series of 2^f for the fraction f, |f| <= 1/2, to 2^-38
__device__ __forceinline__ double exp2_two(Two x) {
  if (!(x.h > -1000.f && x.h < 1000.f)) return exp2((double)x.h);
  const float n = rintf(x.h);
  const double f = ((double)(x.h - n) + (double)x.l) * 0.6931471805599453;
  double y = 1.0 / 3628800;
#pragma unroll
  for (int k = 9; k >= 0; --k) {
    constexpr double inv[10] = {1.0, 1.0, 1.0 / 2, 1.0 / 6, 1.0 / 24, 1.0 / 120, 1.0 / 720, 1.0 / 5040, 1.0 / 40320, 1.0 / 362880};
    y = fma(y, f, inv[k]);
  }
  return ldexp(y, (int)n);
}

__device__ __forceinline__ float load_g(const void *g, int dtype, int64_t i) { return ld_act(g, dtype, i); }

// the time of the walk's step i (past the sequence's end where there is none)
__device__ __forceinline__ int time_of(const Walk &p, int i) { return p.rev ? p.chunks * p.ch - 1 - i : i; }

// a log decay in units of log2, bounded below; NaN stays
__device__ __forceinline__ Two to_log2(float g) {
  const float x = g != g ? g : fmaxf(g, -300.f), y = x * 1.44269504f;      // log2 e in two floats
  return Two{y, fmaf(x, 1.92596303e-8f, fmaf(x, 1.44269504f, -y))};
}
__device__ __forceinline__ Two log2_of(const Walk &p, int b, int h, int t) { return to_log2(load_g(p.g, p.g_dtype, b * p.g_bs + t * p.g_ls + h * p.g_hs)); }
// the decay before the walk's step i: backwards that of the step after it in time
__device__ __forceinline__ Two log2_decay(const Walk &p, int b, int h, int i) {
  const int t = p.rev ? p.chunks * p.ch - i : i;
  return t < p.length ? log2_of(p, b, h, t) : two(0.f);
}

// What the chunk's decays come to, by one warp, two steps a lane: sums from the chunk's start in two floats, their
// exponentials, and what is left of each step at the chunk's end.
struct Decays {
  float hi[CH], lo[CH], in[CH], out[CH];
  float keep, keep_lo;                    // of the state over the chunk, in two floats: it is multiplied up over all chunks
  Two total;
};
template <typename D> __device__ __forceinline__ void keep_of(D &d, Two end) {
  const double keep = exp2_two(end);
  d.keep = (float)keep;
  d.keep_lo = end.h <= 0.f ? (float)(keep - (double)d.keep) : 0.f;
  d.total = end;
}
__device__ __forceinline__ Two inclusive(Two s, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Two u = shfl_up2(s, o);
    if (lane >= o) s = s + u;
  }
  return s;
}
__device__ __forceinline__ Two from_lane(Two s, int lane) { return Two{__shfl_sync(0xffffffffu, s.h, lane), __shfl_sync(0xffffffffu, s.l, lane)}; }
__device__ __forceinline__ void chunk_decays(const Walk &p, int b, int h, int i0, int lane, Decays &d) {
  const Two a0 = log2_decay(p, b, h, i0 + 2 * lane), a1 = log2_decay(p, b, h, i0 + 2 * lane + 1);
  const Two s = inclusive(a0 + a1, lane), end = from_lane(s, 31);
  Two before = shfl_up2(s, 1);
  if (lane == 0) before = two(0.f);
  const Two G[2] = {before + a0, s};                 // (s less a1 would be NaN where a1 is infinite or NaN, a step before it)
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = 2 * lane + j;
    d.hi[i] = G[j].h;
    d.lo[i] = G[j].l;
    d.in[i] = ex2a(G[j].h);
    d.out[i] = ex2a(minus(end, G[j])) * p.s_update;
  }
  if (lane == 0) keep_of(d, end);
}
// exp(G_r - G_c)
__device__ __forceinline__ float decay_between(const Decays &d, int r, int c) { return ex2a((d.hi[r] - d.hi[c]) + (d.lo[r] - d.lo[c])); }

// The dots of a chunk's steps become what the pairs of steps on both sides of a step give to its decay, by one warp, N steps a
// lane, summed in two floats and kept as one.  Forwards (x . dq, pairs whose earlier step is before the chunk): the sum from the step on.  Backwards (x . dk,
// pairs whose later step is after the chunk, and pairs within it, by row and column sums without the diagonal): the sum
// over the steps before it in time.
template <int N> __device__ __forceinline__ void chunk_runs(const Walk &p, int tile, int bh, int i0, int lane, const Two (&v)[N], float dots) {
  Two s = v[N - 1];
#pragma unroll
  for (int j = N - 2; j >= 0; --j) s = s + v[j];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Two u = shfl_down2(s, o);
    if (lane + o < 32) s = s + u;
  }
  const int64_t row = (int64_t)tile * p.batch * p.heads + bh;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int t = time_of(p, i0 + N * lane + j);
    const Two next = s + -v[j], r = p.rev ? next : s;
    if (t < p.length) p.run[row * p.length + t] = r.h;
    s = next;
  }
  dots = warp_sum(dots);
  if (lane == 0) p.sum[row * p.chunks + (p.rev ? p.chunks - 1 - i0 / p.ch : i0 / p.ch)] = dots;
}

// One 16 x 8 x 8 product on TF32 operands given as float32 bit patterns.
__device__ __forceinline__ void mma8(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ uint32_t tf32(float x) {
  uint32_t y;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(y) : "f"(x));
  return y;
}

// acc (16 x 8 NT of a warp) += A (16 x K) B (K x 8 NT).  A(m, k) = a[m * AM + k * AK] * wk[k] (wk nullable), B(k, n) = b[k * BK + n * BN].
// An operand whose values have at most 11 bits (16-bit inputs) is exact in TF32; others are split in two: a b ~ a_hi b_hi + a_lo b_hi + a_hi b_lo.
template <bool SPLIT_A, bool SPLIT_B, int AM, int AK, int BK, int BN, int NT>
__device__ __forceinline__ void product(float (&acc)[NT][4], const float *a, const float *wk, const float *b, int K, int lane) {
  const int g = lane >> 2, t = lane & 3;
  a += g * AM + t * AK;
  b += t * BK + g * BN;
#pragma unroll 4
  for (int k0 = 0; k0 < K; k0 += 8, a += 8 * AK, b += 8 * BK) {
    float av[4] = {a[0], a[8 * AM], a[4 * AK], a[8 * AM + 4 * AK]};
    if (wk) {
      const float w0 = wk[k0 + t], w1 = wk[k0 + t + 4];
      av[0] *= w0;
      av[1] *= w0;
      av[2] *= w1;
      av[3] *= w1;
    }
    uint32_t ah[4], al[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ah[i] = SPLIT_A ? tf32(av[i]) : __float_as_uint(av[i]);
      al[i] = SPLIT_A ? tf32(av[i] - __uint_as_float(ah[i])) : 0u;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float bv[2] = {b[n * 8 * BN], b[n * 8 * BN + 4 * BK]};
      uint32_t bh[2], bl[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        bh[i] = SPLIT_B ? tf32(bv[i]) : __float_as_uint(bv[i]);
        bl[i] = SPLIT_B ? tf32(bv[i] - __uint_as_float(bh[i])) : 0u;
      }
      // the unit truncates when it adds: each step's products start from zero, the small ones first, and are added rounded
      float c[4] = {0.f, 0.f, 0.f, 0.f};
      if (SPLIT_A) mma8(c, al, bh);
      if (SPLIT_B) mma8(c, ah, bl);
      mma8(c, ah, bh);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] += c[i];
    }
  }
}

// 64 rows of an operand from step i0 on into shared memory as float32, zero past the sequence and past its size: 16 threads a
// row, 4 columns each.  Returns whether one of them is infinite or NaN.
template <typename T, int WT>
__device__ __forceinline__ bool load_rows(const Walk &p, const void *base, int64_t off, int64_t ls, int i0, int col0, int size, int width, int pitch, float *dst) {
  const T *src = reinterpret_cast<const T *>(base) + off + col0;
  const bool vec = ((reinterpret_cast<uintptr_t>(src) | (uintptr_t)(ls * sizeof(T))) & (4 * sizeof(T) - 1)) == 0;
  const int r0 = threadIdx.x >> 4;
  float zero = 0.f;
  for (int c = (threadIdx.x & 15) * 4; c < width; c += 64) {
    const int left = size - col0 - c;
    float4 v[CH / (WT / 16)];
#pragma unroll
    for (int i = 0; i < CH / (WT / 16); ++i) {
      const int t = time_of(p, i0 + r0 + i * (WT / 16));
      const T *s = src + (int64_t)t * ls + c;
      const bool in = t < p.length;
      v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (vec && left >= 4) {
        if (in) {
          if constexpr (sizeof(T) == 4) v[i] = __ldg(reinterpret_cast<const float4 *>(s));
          else {
            const uint2 w = __ldg(reinterpret_cast<const uint2 *>(s));
            const T *x = reinterpret_cast<const T *>(&w);
            v[i] = make_float4((float)x[0], (float)x[1], (float)x[2], (float)x[3]);
          }
        }
      } else if (in) {
        if (left > 0) v[i].x = (float)s[0];
        if (left > 1) v[i].y = (float)s[1];
        if (left > 2) v[i].z = (float)s[2];
        if (left > 3) v[i].w = (float)s[3];
      }
    }
#pragma unroll
    for (int i = 0; i < CH / (WT / 16); ++i) {
      *reinterpret_cast<float4 *>(dst + (r0 + i * (WT / 16)) * pitch + c) = v[i];
      zero = fmaf(v[i].x, 0.f, fmaf(v[i].y, 0.f, fmaf(v[i].z, 0.f, fmaf(v[i].w, 0.f, zero))));
    }
  }
  return zero != 0.f;
}

// the cache lines of the rows: four threads a row, 32 columns apart
template <typename T>
__device__ __forceinline__ void prefetch_rows(const Walk &p, const void *base, int64_t off, int64_t ls, int i0, int col0, int size) {
  const int t = time_of(p, i0 + (threadIdx.x >> 2)), c = (threadIdx.x & 3) * 32;
  if (threadIdx.x < CH * 4 && t < p.length && c < min(size - col0, MAX_D))
    asm volatile("prefetch.global.L1 [%0];" ::"l"(reinterpret_cast<const T *>(base) + off + (int64_t)t * ls + col0 + c));
}

// WT threads: a warp has 16 x 8 NT scores and results.  With 512 a block is done with a chunk sooner; where there are
// more blocks than SMs and two fit (up to 64 rows of state), two of 256 get through more (2 x 640 steps x 128 heads of 64 x
// 64, float16, with gradients: 966 -> 720 us; 2 x 100 steps x 8 heads 102 -> 117 us).
template <typename T, int DI, int WT, bool STATE_ONLY> __global__ void __launch_bounds__(WT, WT == 256 ? 2 : 1) linattn_walk_kernel(const Walk p) {
  constexpr int NT = 1024 / WT, NW = 8 / NT;             // NW: warps along 64 columns
  constexpr bool F32 = sizeof(T) == 4;
  extern __shared__ __align__(16) float sm[];
  constexpr int PQ = DI + 4;
  const int dip = (p.di + 15) / 16 * 16;                // rows and columns in use, of DI
  float *sk = sm, *sv = sk + CH * PQ, *S = sv + CH * PV, *sq = S + DI * PV, *sp = sq + CH * PQ, *sx = sp + CH * PP;
  __shared__ Decays dd[2];
  __shared__ float dots[NW][CH], rows_[NW][CH], cols_[4][CH];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gq = lane >> 2, tq = lane & 3;
  const int tile = blockIdx.x % p.tiles, bh = blockIdx.x / p.tiles % (p.batch * p.heads), seg = blockIdx.x / p.tiles / (p.batch * p.heads);
  const int b = bh / p.heads, h = bh % p.heads, col0 = tile * DO;
  const int i_begin = seg * p.seg_chunks * CH, i_end = min(p.chunks, (seg + 1) * p.seg_chunks) * CH;
  const int snaps = (p.chunks + kSnap - 1) / kSnap;
  const auto snapshot = [&](int c, float f) {            // at the border before chunk c in time
    for (int e = tid; e < p.di * DO; e += WT) {
      const int r = e / DO, col = e % DO;
      if (col0 + col < p.dout) p.snap[(((int64_t)bh * snaps + c / kSnap) * p.di + r) * p.dout + col0 + col] = S[r * PV + col] * f;
    }
  };
  let_next_start();
  // the state before the first step
  for (int e = tid; e < dip * DO; e += WT) {
    const int r = e / DO, c = e % DO;
    float s = 0.f;
    if (!STATE_ONLY && r < p.di && col0 + c < p.dout) {
      if (p.nseg > 1) s = p.seg[(((int64_t)bh * p.nseg + seg) * p.di + r) * p.dout + col0 + c];
      else if (p.s0) s = p.s0[b * p.s0_bs + h * p.s0_hs + r * p.s0_is + (col0 + c) * p.s0_os];
    }
    S[r * PV + c] = s;
  }
  double total = 0.0;
  if (warp == 4) chunk_decays(p, b, h, i_begin, lane, dd[0]);
  for (int i0 = i_begin, it = 0; i0 < i_end; i0 += CH, ++it) {
    __syncthreads();                                 // the last chunk's reads and writes are done
    const int chunk = p.rev ? p.chunks - 1 - i0 / CH : i0 / CH;
    const Decays &d = dd[it & 1];
    if (!STATE_ONLY && p.run && !p.rev && chunk % kSnap == 0) snapshot(chunk, 1.f);
    load_rows<T, WT>(p, p.k, b * p.k_bs + h / p.k_div * p.k_hs, p.k_ls, i0, 0, p.di, dip, PQ, sk);
    bool odd = load_rows<T, WT>(p, p.v, b * p.v_bs + h / p.v_div * p.v_hs, p.v_ls, i0, col0, p.dout, DO, PV, sv);
    if (!STATE_ONLY) {
      load_rows<T, WT>(p, p.q, b * p.q_bs + h / p.q_div * p.q_hs, p.q_ls, i0, 0, p.di, dip, PQ, sq);
      if (p.run) load_rows<T, WT>(p, p.x, b * p.x_bs + h / p.x_div * p.x_hs, p.x_ls, i0, col0, p.dout, DO, PP, sx);
    }
    odd = __syncthreads_or(odd);                     // some value is infinite or NaN
    const int m0 = (warp & 3) * 16, n0 = (warp >> 2) * 8 * NT;  // this warp's scores and results
    if (i0 + CH < i_end) {                           // the next chunk's rows into the first-level cache
      prefetch_rows<T>(p, p.k, b * p.k_bs + h / p.k_div * p.k_hs, p.k_ls, i0 + CH, 0, p.di);
      prefetch_rows<T>(p, p.v, b * p.v_bs + h / p.v_div * p.v_hs, p.v_ls, i0 + CH, col0, p.dout);
      if (!STATE_ONLY) {
        prefetch_rows<T>(p, p.q, b * p.q_bs + h / p.q_div * p.q_hs, p.q_ls, i0 + CH, 0, p.di);
        if (p.run) prefetch_rows<T>(p, p.x, b * p.x_bs + h / p.x_div * p.x_hs, p.x_ls, i0 + CH, col0, p.dout);
      }
    }
    // the next chunk's decays, by a warp whose scores are all zero
    if (warp == 4 && i0 + CH < i_end) chunk_decays(p, b, h, i0 + CH, lane, dd[(it + 1) & 1]);
    if (!STATE_ONLY) {
      float acc[NT][4] = {};
      const bool any = n0 <= m0 + 15;
      if (any) product<F32, F32, PQ, 1, 1, PQ, NT>(acc, sq + m0 * PQ, nullptr, sk + n0 * PQ, dip, lane);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = m0 + gq + (e >> 1) * 8, c = n0 + n * 8 + tq * 2 + (e & 1);
          acc[n][e] = c <= r ? acc[n][e] * decay_between(d, r, c) * p.s_intra : 0.f;
          sp[r * PP + c] = acc[n][e];
        }
      if (p.run && p.rev) {                          // products of a pair's two scores, without the diagonal
        float x[NT][4] = {};
        if (any) product<F32, F32, PP, 1, 1, PV, NT>(x, sx + m0 * PP, nullptr, sv + n0 * PV, DO, lane);
        float row[2] = {0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e1 = 0; e1 < 2; ++e1) {
            const int c = n0 + n * 8 + tq * 2 + e1;
            float col = 0.f;
#pragma unroll
            for (int e2 = 0; e2 < 2; ++e2) {
              const float m = c == m0 + gq + e2 * 8 ? 0.f : acc[n][e2 * 2 + e1] * x[n][e2 * 2 + e1];
              row[e2] += m;
              col += m;
            }
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) col += __shfl_xor_sync(0xffffffffu, col, o);
            if (gq == 0) cols_[warp & 3][c] = col;
          }
#pragma unroll
        for (int e2 = 0; e2 < 2; ++e2) {
          row[e2] += __shfl_xor_sync(0xffffffffu, row[e2], 1);
          row[e2] += __shfl_xor_sync(0xffffffffu, row[e2], 2);
          if (tq == 0) rows_[warp >> 2][m0 + gq + e2 * 8] = row[e2];
        }
      }
      __syncthreads();
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
      product<F32, true, PQ, 1, PV, 1, NT>(acc, sq + m0 * PQ, nullptr, S + n0, dip, lane);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][e] *= d.in[m0 + gq + (e >> 1) * 8] * p.s_inter;
      if (p.run) {
#pragma unroll
        for (int e2 = 0; e2 < 2; ++e2) {
          const int r = m0 + gq + e2 * 8;
          float s = 0.f;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e1 = 0; e1 < 2; ++e1) s = fmaf(acc[n][e2 * 2 + e1], sx[r * PP + n0 + n * 8 + tq * 2 + e1], s);
          s += __shfl_xor_sync(0xffffffffu, s, 1);
          s += __shfl_xor_sync(0xffffffffu, s, 2);
          if (tq == 0) dots[warp >> 2][r] = s;
        }
      }
      if (!odd) product<true, F32, PP, 1, PV, 1, NT>(acc, sp + m0 * PP, nullptr, sv + n0, min(CH, m0 + 16), lane);
      else                                           // one by one: a zero score of a later step would carry it to earlier ones
        for (int e2 = 0; e2 < 2; ++e2) {
          const int r = m0 + gq + e2 * 8;
          for (int j = 0; j <= r; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e1 = 0; e1 < 2; ++e1)
                if (e2 == 0) acc[n][e1] = fmaf(sp[r * PP + j], sv[j * PV + n0 + n * 8 + tq * 2 + e1], acc[n][e1]);
                else acc[n][2 + e1] = fmaf(sp[r * PP + j], sv[j * PV + n0 + n * 8 + tq * 2 + e1], acc[n][2 + e1]);
        }
#pragma unroll
      for (int e2 = 0; e2 < 2; ++e2) {
        const int t = time_of(p, i0 + m0 + gq + e2 * 8);
        if (t >= p.length) continue;
        const int64_t o = b * p.o_bs + t * p.o_ls + h * p.o_hs;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e1 = 0; e1 < 2; ++e1) {
            const int c = col0 + n0 + n * 8 + tq * 2 + e1;
            if (c >= p.dout) continue;
            const float v = acc[n][e2 * 2 + e1];
            if (p.out_f32) reinterpret_cast<float *>(p.out)[o + c] = v;
            else reinterpret_cast<T *>(p.out)[o + c] = T(v);
          }
      }
    }
    __syncthreads();                                 // all have read the state
    if (!STATE_ONLY && p.run && warp == 0) {
      Two v[2];
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int i = 2 * lane + j;
        float dot = 0.f;
        Two row = two(0.f);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          dot += dots[w][i];
          if (p.rev) row = row + two(rows_[w][i]);
        }
        s += dot;
        v[j] = two(dot);
        if (p.rev) v[j] = (v[j] + row) + -((two(cols_[0][i]) + two(cols_[1][i])) + (two(cols_[2][i]) + two(cols_[3][i])));
      }
      chunk_runs(p, tile, bh, i0, lane, v, s);
    }
    if (STATE_ONLY) total += (double)d.total.h + (double)d.total.l;
    const float keep = d.keep, keep_lo = d.keep_lo;
    for (int u = warp; u < dip / 16 * NW; u += WT / 32) {
      const int r0 = u / NW * 16, c0 = u % NW * (8 * NT);
      float acc[NT][4] = {};
      product<true, F32, 1, PQ, PV, 1, NT>(acc, sk + r0, d.out, sv + c0, CH, lane);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float *s = S + (r0 + gq + (e >> 1) * 8) * PV + c0 + n * 8 + tq * 2 + (e & 1);
          *s = fmaf(*s, keep, fmaf(*s, keep_lo, acc[n][e]));
        }
    }
    if (!STATE_ONLY && p.run && p.rev && chunk % kSnap == 0) {
      __syncthreads();
      snapshot(chunk, (float)exp2_two(log2_of(p, b, h, chunk * CH)));
    }
  }
  __syncthreads();
  if (STATE_ONLY) {
    for (int e = tid; e < p.di * DO; e += WT) {
      const int r = e / DO, c = e % DO;
      if (col0 + c < p.dout) p.seg[(((int64_t)bh * p.nseg + seg) * p.di + r) * p.dout + col0 + c] = S[r * PV + c];
    }
    if (tile == 0 && tid == 0) p.seg_g[(int64_t)bh * p.nseg + seg] = total;
  } else if (p.last && seg == p.nseg - 1) {
    const float f = p.last_decay ? (float)exp2_two(log2_of(p, b, h, 0)) : 1.f;
    for (int e = tid; e < p.di * DO; e += WT) {
      const int r = e / DO, c = e % DO;
      if (col0 + c < p.dout) p.last[b * p.last_bs + h * p.last_hs + r * p.last_is + (col0 + c) * p.last_os] = S[r * PV + c] * f;
    }
  }
  if (blockIdx.x == gridDim.x - 1) wait_for_last();
}

// ------------------------------------------------------------------------------------------------ bfloat16
//
// The same walk in chunks of 128 steps on the tensor cores' own accumulators (tcgen05 + TMEM).  A chunk is five products, each
// issued by one thread: scores q k^T (128 x 128), q with the state (128 x 64), scores with v, keys with decayed values (the
// state's sum of the chunk, a row of TMEM for each of its rows), and for the gradient of g the other scores x v^T.  256 threads do
// what lies between: a thread has one step (or row of the state) and half of the columns.  The scores are decayed,
// rounded and put back into TMEM where they were, as the left operand of the product with v; the state stays in the threads'
// registers in float32.  Two blocks fit an SM (256 columns of TMEM and about 100 KB of shared memory each), and one works
// while the other waits.
//
// All tiles are 128 rows of 64 columns in the 128-byte swizzle, and serve as K-major and as MN-major operands as they are.
// Terms of a float32 number are its bfloat16 rounding, that of the rest, and so on: two keep 2^-17 of it, three all of
// it.  Scores and the state that q meets are rounded once, as the result is (an error of 1.4 times the result's own rounding
// in all), the state in three terms where its dots with x go into the float32 gradient of g; decayed values, which add up in the state,
// are kept in two, or in three where the state is itself a result or goes into such a dot.  The small terms' products go into
// an accumulator first: the tensor core truncates when it adds.  float16 stays with the TF32 kernel: its states may exceed
// what it can hold.

constexpr int BC = 128;                     // steps of a chunk
constexpr int BT = 256;                     // threads
constexpr int BTILE = BC * 128;             // bytes: 128 rows of 64 columns
constexpr int kSnapB = kSnapSteps / BC;
constexpr uint32_t kWaitLimit = 1u << 24;

__device__ int g_linattn_status = 0;

// the next bfloat16 term of two numbers, which keep their rest
__device__ __forceinline__ uint32_t term(float &a, float &b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  const uint32_t w = *reinterpret_cast<const uint32_t *>(&v);
  a -= __uint_as_float(w << 16);
  b -= __uint_as_float(w & 0xffff0000u);
  return w;
}
__device__ __forceinline__ float low16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high16(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// byte offset of 16-byte piece c of row r in a swizzled tile
__device__ __forceinline__ uint32_t piece_at(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

// The operands as tensors of (size, heads or groups, length, batch), tiles of 64 x 128 steps; `tma` is 0 where an operand's strides or
// alignment do not allow it, and the blocks load all of them themselves.
struct Maps {
  CUtensorMap q, k, v, x, out;
  int tma, tma_out;
};
__device__ __forceinline__ void tma_4d(void *dst, const CUtensorMap *map, int c, int h, int t, int b, uint64_t *bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(c), "r"(h), "r"(t), "r"(b), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tma_st_4d(const CUtensorMap *map, const void *src, int c, int h, int t, int b) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(c), "r"(h),
               "r"(t), "r"(b), "r"(smem_u32(src))
               : "memory");
}
// 128 steps of W columns (64 a tile) from time t0 on, zero past the sequence and past its size
template <int W>
__device__ __noinline__ void load_tile(const Walk &p, const void *base, int64_t off, int64_t ls, int size, int col0, int t0, unsigned char *dst) {
  constexpr int PER = W / 8;                             // 16-byte pieces of a row
  const uint16_t *src = reinterpret_cast<const uint16_t *>(base) + off + col0;
  for (int e = threadIdx.x; e < BC * PER; e += BT) {
    const int r = e / PER, pc = e % PER, t = t0 + r, left = size - col0 - pc * 8;
    const uint16_t *s = src + (int64_t)t * ls + pc * 8;
    uint32_t x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = t < p.length && j < left ? s[j] : 0u;
    *reinterpret_cast<uint4 *>(dst + (pc >> 3) * BTILE + piece_at(r, pc & 7)) = make_uint4(x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16);
  }
}

// A chunk's decays by one warp, four steps a lane (see Decays), by the steps' order in time; G runs in the walk's order.  Between
// two blocks of 32 steps the decay is the product of two factors of at most one: from a step back to the start of its
// block (in the walk's order), and from there back to the earlier step (`back`, a row for each block that has earlier ones).
struct DecaysB {
  float hi[BC], lo[BC], in[BC], out[BC], back[3][BC];
  float keep, keep_lo;
  Two total;
};
__device__ __forceinline__ float between(const DecaysB &d, int r, int c) { return ex2a((d.hi[r] - d.hi[c]) + (d.lo[r] - d.lo[c])); }
__device__ __forceinline__ int in_time(const Walk &p, int i) { return p.rev ? BC - 1 - i : i; }
// the decays before a lane's four steps of the chunk from step i0 on, all four loads in flight at once
struct Four { float g[4]; };
__device__ __forceinline__ Four load_decays(const Walk &p, int b, int h, int i0, int lane) {
  Four f;
  const int64_t at = b * p.g_bs + h * p.g_hs;
  int t[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = i0 + 4 * lane + j;
    t[j] = p.rev ? p.chunks * BC - i : i;
  }
  if (p.g_dtype == B200_F32) {
    const float *g = reinterpret_cast<const float *>(p.g) + at;
#pragma unroll
    for (int j = 0; j < 4; ++j) f.g[j] = __ldg(g + (t[j] < p.length ? t[j] * p.g_ls : 0));
  } else {
    const __nv_bfloat16 *g = reinterpret_cast<const __nv_bfloat16 *>(p.g) + at;
#pragma unroll
    for (int j = 0; j < 4; ++j) f.g[j] = __bfloat162float(g[t[j] < p.length ? t[j] * p.g_ls : 0]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (t[j] >= p.length) f.g[j] = 0.f;
  return f;
}
__device__ __forceinline__ void chunk_decays_b(const Walk &p, const Four &f, int lane, DecaysB &d) {
  Two a[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) a[j] = to_log2(f.g[j]);
#pragma unroll
  for (int j = 1; j < 4; ++j) a[j] = a[j] + a[j - 1];
  const Two inc = inclusive(a[3], lane), end = from_lane(inc, 31);
  Two before = shfl_up2(inc, 1);
  if (lane == 0) before = two(0.f);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = in_time(p, 4 * lane + j);
    const Two G = before + a[j];
    d.hi[i] = G.h;
    d.lo[i] = G.l;
    d.in[i] = ex2a(G.h);
    d.out[i] = ex2a(minus(end, G)) * p.s_update;
  }
  if (lane == 0) keep_of(d, end);
  __syncwarp();
#pragma unroll
  for (int j = 1; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < j; ++i) {
      const int c = in_time(p, i * 32 + lane);
      d.back[j - 1][c] = between(d, in_time(p, 32 * j), c);
    }
}

// Sums over the 32 lanes of 16 numbers each: lane l (and l + 16) gets the sum of number l % 16.
__device__ __forceinline__ float sum_columns(float (&v)[16], int lane) {
#pragma unroll
  for (int n = 8; n >= 1; n >>= 1) {
    const bool up = lane & n;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, n);
    }
  }
  return v[0] + __shfl_xor_sync(0xffffffffu, v[0], 16);
}

// Whether one of eight bfloat16 is infinite or NaN: it times zero is NaN.
__device__ __forceinline__ bool not_finite(const uint32_t (&x)[4]) {
  __nv_bfloat162 t = __float2bfloat162_rn(0.f);
#pragma unroll
  for (int j = 0; j < 4; ++j) t = __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&x[j]), __float2bfloat162_rn(0.f), t);
  return (*reinterpret_cast<const uint32_t *>(&t) & 0x7fff7fffu) != 0u;
}

// MODE: only a segment's own state; results; results and dots with x, forwards; the same backwards
enum { OWN_STATE = 0, RESULTS = 1, DOTS = 2, DOTS_REV = 3 };

// shared memory: q | the state's terms, whose place the values' terms take once both have met; k, v, x
__host__ __device__ constexpr int terms_bytes(int di, int ts, int tu) {
  return (di / 64 * BTILE + ts * di * 128) > tu * BTILE ? di / 64 * BTILE + ts * di * 128 : tu * BTILE;
}

template <int DI, int MODE> __global__ void __launch_bounds__(BT, DI == 128 && MODE >= DOTS ? 1 : 2) linattn_walk_tc_kernel(const Walk p, const __grid_constant__ Maps maps, const int tu) {
  constexpr bool STATE_ONLY = MODE == OWN_STATE, grad = MODE >= DOTS, cross = MODE == DOTS_REV;
  constexpr int ts = grad ? 3 : 1, QB = DI / 64 * BTILE;
  extern __shared__ __align__(1024) unsigned char raw[];
  unsigned char *sq = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  unsigned char *ss = sq + QB, *su = sq;
  unsigned char *sk = sq + (STATE_ONLY ? tu * BTILE : terms_bytes(DI, ts, tu)), *sv = sk + QB, *sx = sv + BTILE;
  __shared__ DecaysB dd[2];
  __shared__ float dots[2][BC], rows_[2][BC], cols_[4][BC];
  __shared__ uint64_t bar, bar_d, loaded_qk, loaded_v;
  __shared__ uint32_t tmem_base;
  __shared__ int fail, odd[2], odd_from[2][DO];               // odd: a value of the chunk is infinite or NaN, from which step on in each column
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int tile = blockIdx.x % p.tiles, bh = blockIdx.x / p.tiles % (p.batch * p.heads), seg = blockIdx.x / p.tiles / (p.batch * p.heads);
  const int b = bh / p.heads, h = bh % p.heads, col0 = tile * DO;
  const int i_begin = seg * p.seg_chunks * BC, i_end = min(p.chunks, (seg + 1) * p.seg_chunks) * BC;
  const int snaps = (p.chunks + kSnapB - 1) / kSnapB;
  // this thread's TMEM lane (a step of the chunk, a row of the state) and half of the columns
  const int wr = warp & 3, half = warp >> 2, r = wr * 32 + lane, c0 = half * 32;
  if (tid < DO) {
    odd[0] = 0;
    odd_from[0][tid] = BC;
  }
  if (tid == 0) {
    mbar_init(&bar, 1);
    mbar_init(&bar_d, 1);
    mbar_init(&loaded_qk, 1);
    mbar_init(&loaded_v, 1);
    fail = 0;
    mbar_fence_init();
  }
  let_next_start();
  __syncwarp();
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)), "r"(256) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const auto time0 = [&](int i0) { return p.rev ? (p.chunks - 1) * BC - i0 : i0; };      // of the chunk's first step in time
  // Two of the warps without scores (their blocks lie after the steps themselves): one forms the next chunk's decays while all
  // wait for the first products, the other issues copies and products.  A third sums up the last chunk's dots meanwhile.
  const int decay_warp = p.rev ? 3 : 4, issue_warp = p.rev ? 2 : 5, sum_warp = p.rev ? 7 : 0;
  const bool issuer = warp == issue_warp && lane == 0;
  const int hq = h / p.q_div, hk = h / p.k_div, hv = h / p.v_div, hx = h / p.x_div;
  const auto copy_qk = [&](int i0) {                     // by the issuer
    const int t0 = time0(i0);
    mbar_expect_tx(&loaded_qk, (STATE_ONLY ? 1 : 2) * QB);
#pragma unroll
    for (int j = 0; j < DI / 64; ++j) {
      if (!STATE_ONLY) tma_4d(sq + j * BTILE, &maps.q, j * 64, hq, t0, b, &loaded_qk);
      tma_4d(sk + j * BTILE, &maps.k, j * 64, hk, t0, b, &loaded_qk);
    }
  };
  const auto copy_v = [&](int i0) {
    mbar_expect_tx(&loaded_v, (grad ? 2 : 1) * BTILE);
    tma_4d(sv, &maps.v, col0, hv, time0(i0), b, &loaded_v);
    if (grad) tma_4d(sx, &maps.x, col0, hx, time0(i0), b, &loaded_v);
  };
  const auto load_all = [&](int i0) {                    // by all threads, where the operands cannot be copied
    const int t0 = time0(i0);
    if (!STATE_ONLY) load_tile<DI>(p, p.q, b * p.q_bs + hq * p.q_hs, p.q_ls, p.di, 0, t0, sq);
    load_tile<DI>(p, p.k, b * p.k_bs + hk * p.k_hs, p.k_ls, p.di, 0, t0, sk);
    load_tile<64>(p, p.v, b * p.v_bs + hv * p.v_hs, p.v_ls, p.dout, col0, t0, sv);
    if (grad) load_tile<64>(p, p.x, b * p.x_bs + hx * p.x_hs, p.x_ls, p.dout, col0, t0, sx);
  };
  // This thread's part of the state: a row and NS columns.  With 64 rows TMEM's upper 64 lanes hold them once more, and the
  // warps there take half of the columns.
  constexpr int NS = DI == 64 ? 16 : 32;
  const int rs = r & (DI - 1), cs = half * 32 + (DI == 64 ? (wr >> 1) * 16 : 0);
  float S[NS];
  const bool has_row = rs < p.di;
  const auto each = [&](auto f) {
    if (has_row)
#pragma unroll
      for (int j = 0; j < NS; ++j)
        if (col0 + cs + j < p.dout) f(col0 + cs + j, S[j]);
  };
  const auto snapshot = [&](int s, float f) {
    float *at = p.snap + (((int64_t)bh * snaps + s) * p.di + rs) * p.dout;
    if (p.dout % 4 == 0 && has_row && col0 + cs + NS <= p.dout) {
#pragma unroll
      for (int j = 0; j < NS; j += 4) *reinterpret_cast<float4 *>(at + col0 + cs + j) = make_float4(S[j] * f, S[j + 1] * f, S[j + 2] * f, S[j + 3] * f);
    } else {
      each([&](int c, float &x) { at[c] = x * f; });
    }
  };
  const auto write_terms = [&]() {
#pragma unroll
    for (int j = 0; j < NS / 8; ++j) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = S[j * 8 + e];
#pragma unroll
      for (int t = 0; t < ts; ++t)
        *reinterpret_cast<uint4 *>(ss + t * DI * 128 + piece_at(rs, cs / 8 + j)) = make_uint4(term(x[0], x[1]), term(x[2], x[3]), term(x[4], x[5]), term(x[6], x[7]));
    }
  };
#pragma unroll
  for (int j = 0; j < NS; ++j) S[j] = 0.f;
  if (!STATE_ONLY) {
    if (p.nseg > 1) each([&](int c, float &x) { x = p.seg[(((int64_t)bh * p.nseg + seg) * p.di + rs) * p.dout + c]; });
    else if (p.s0) each([&](int c, float &x) { x = p.s0[b * p.s0_bs + h * p.s0_hs + rs * p.s0_is + c * p.s0_os]; });
    write_terms();
  }
  if (warp == 7) chunk_decays_b(p, load_decays(p, b, h, i_begin, lane), lane, dd[0]);
  fence_proxy_async();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (!maps.tma) load_all(i_begin);
  else if (issuer) {
    copy_qk(i_begin);
    copy_v(i_begin);
  }
  const uint32_t tm = tmem_base, tm_own = tm + ((uint32_t)(wr * 32) << 16);
  const uint32_t tP = 0, tO = 128, tD = 192;             // columns: scores, result, the state's sum (x v^T takes the place of the last two for a while)
  constexpr uint32_t kScores = idesc_f16(1, false, false, 128, 128), kState = idesc_f16(1, false, true, 128, 64), kUpdate = idesc_f16(1, true, true, 128, 64);
  const auto kmajor = [](int i) { return (uint64_t)(((i >> 2) * BTILE + (i & 3) * 32) / 16); };      // to the i-th 16 columns of a K-major operand
  uint32_t phase = 0;
  const auto wait_products = [&](uint64_t &on, uint32_t parity) {
    if (!mbar_wait(&on, parity, kWaitLimit)) *(volatile int *)&fail = 1;
    __syncwarp();
    tc_fence_after();
  };
  // the state's sum of the chunk; keys of 64 columns are both halves of the 128 rows
  const auto issue_update = [&]() {
    const uint64_t k = smem_desc(smem_u32(sk), DI == 64 ? 0 : BTILE, 1024, 2), u = smem_desc(smem_u32(su), 8192, 1024, 2);
#pragma unroll 1
    for (int t = tu - 1; t >= 0; --t)
#pragma unroll
      for (int i = 0; i < BC / 16; ++i) mma_f16(tm + tD, k + i * 128, u + t * (BTILE / 16) + i * 128, kUpdate, t < tu - 1 || i > 0);
  };
  const auto issue_scores = [&]() {
    const uint64_t q = smem_desc(smem_u32(sq), 16, 1024, 2), k = smem_desc(smem_u32(sk), 16, 1024, 2);
#pragma unroll
    for (int i = 0; i < DI / 16; ++i) mma_f16(tm + tP, q + kmajor(i), k + kmajor(i), kScores, i > 0);
  };
  Four next = {};                                        // the decay warp's: logarithms of the next chunk's decays
  if (warp == decay_warp && i_begin + BC < i_end) next = load_decays(p, b, h, i_begin + BC, lane);
  Two pairs[4] = {};                                     // the sum warp's: of the last chunk, four steps a lane
  float dot_sum = 0.f;
  bool scores_on = false;                                // the issuer's: this chunk's are on their way since the last one
  double total = 0.0;
  for (int i0 = i_begin, it = 0; i0 < i_end; i0 += BC, ++it) {
    const int chunk = p.rev ? p.chunks - 1 - i0 / BC : i0 / BC;
    const DecaysB &d = dd[it & 1];
    if (grad && !cross && chunk % kSnapB == 0) snapshot(chunk / kSnapB, 1.f);
    fence_proxy_async();
    tc_fence_before();
    if (__syncthreads_or(*(volatile int *)&fail)) break;     // the state's terms are written, accumulators read; a wait that ran out ends the walk for all
    if (!STATE_ONLY && tid < DO) {                       // the next chunk's
      odd[(it + 1) & 1] = 0;
      odd_from[(it + 1) & 1][tid] = BC;
    }
    if (issuer && maps.tma && !scores_on && !mbar_wait(&loaded_qk, it & 1, kWaitLimit)) *(volatile int *)&fail = 1;
    const auto meanwhile = [&]() {
      if (warp == decay_warp && i0 + BC < i_end) {
        chunk_decays_b(p, next, lane, dd[(it + 1) & 1]);
        if (i0 + 2 * BC < i_end) next = load_decays(p, b, h, i0 + 2 * BC, lane);
      }
      if (grad && warp == sum_warp && it > 0) chunk_runs(p, tile, bh, i0 - BC, lane, pairs, dot_sum);
    };
    if (STATE_ONLY) meanwhile();
    float O[32];
    if constexpr (!STATE_ONLY) {
      if (issuer) {
        tc_fence_after();
        const uint64_t q = smem_desc(smem_u32(sq), 16, 1024, 2), st = smem_desc(smem_u32(ss), 8192, 1024, 2);
        if (!scores_on) issue_scores();
        scores_on = false;
#pragma unroll
        for (int t = ts - 1; t >= 0; --t)
#pragma unroll
          for (int i = 0; i < DI / 16; ++i) mma_f16(tm + tO, q + kmajor(i), st + (t * DI * 128 + i * 2048) / 16, kState, t < ts - 1 || i > 0);
        mma_commit(&bar);
      }
      __syncwarp();
      meanwhile();
      wait_products(bar, phase);
      phase ^= 1;
      {
        tmem_ld32(tm_own + tO + c0, O);
        const float f = d.in[r] * p.s_inter;
#pragma unroll
        for (int j = 0; j < 32; ++j) O[j] *= f;
      }
      if (maps.tma && !mbar_wait(&loaded_v, it & 1, kWaitLimit)) *(volatile int *)&fail = 1;
      if (grad) {
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4 w = *reinterpret_cast<const uint4 *>(sx + piece_at(r, half * 4 + j));
          const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) dot = fmaf(O[j * 8 + 2 * e], low16(x[e]), fmaf(O[j * 8 + 2 * e + 1], high16(x[e]), dot));
        }
        dots[half][r] = dot;
      }
      if (cross) {
        tc_fence_before();
        __syncthreads();                                 // the result's columns are read
        if (issuer) {
          tc_fence_after();
          const uint64_t x = smem_desc(smem_u32(sx), 16, 1024, 2), v = smem_desc(smem_u32(sv), 16, 1024, 2);
#pragma unroll
          for (int i = 0; i < DO / 16; ++i) mma_f16(tm + tO, x + kmajor(i), v + kmajor(i), kScores, i > 0);
          mma_commit(&bar);
        }
        __syncwarp();
      }
    }
    if (STATE_ONLY && maps.tma && !mbar_wait(&loaded_v, it & 1, kWaitLimit)) *(volatile int *)&fail = 1;
    // values as the state takes them up, in terms: q and the state's terms have been read
#pragma unroll 1
    for (int i = 0; i < BC * 8 / BT; ++i) {
      const int e = i * BT + tid, row = e >> 3;
      const uint32_t at = piece_at(row, e & 7);
      const uint4 w = *reinterpret_cast<const uint4 *>(sv + at);
      const uint32_t x[4] = {w.x, w.y, w.z, w.w};
      const float f = d.out[row];
      float y[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[2 * j] = low16(x[j]) * f;
        y[2 * j + 1] = high16(x[j]) * f;
      }
      if (!STATE_ONLY && not_finite(x)) {
        // The zeros that stand for the scores of later steps would carry an infinite or NaN value to earlier results: the product
        // with the scores takes a zero for it, and the results from its step on become NaN in its column.
        if (cross && !mbar_wait(&bar, phase, kWaitLimit)) *(volatile int *)&fail = 1;      // x v^T has read it
        odd[it & 1] = 1;
        for (int j = 0; j < 8; ++j) {
          const uint32_t half_of = j & 1 ? x[j >> 1] >> 16 : x[j >> 1] & 0xffffu;
          if ((half_of & 0x7f80u) != 0x7f80u) continue;
          atomicMin(&odd_from[it & 1][(e & 7) * 8 + j], p.rev ? BC - 1 - row : row);
          *reinterpret_cast<uint16_t *>(sv + at + j * 2) = 0;
        }
      }
#pragma unroll
      for (int t = 0; t < 3; ++t)
        if (t < tu) *reinterpret_cast<uint4 *>(su + t * BTILE + at) = make_uint4(term(y[0], y[1]), term(y[2], y[3]), term(y[4], y[5]), term(y[6], y[7]));
    }
    if constexpr (!cross) {                              // the state's sum of the chunk, while scores are decayed
      fence_proxy_async();
      tc_fence_before();
      __syncthreads();
      if (issuer) {
        tc_fence_after();
        issue_update();
        mma_commit(&bar_d);
      }
      __syncwarp();
    }
    if constexpr (!STATE_ONLY) {
      if (cross) {
        wait_products(bar, phase);
        phase ^= 1;
      }
      // scores: decayed, zero after the step itself (in the walk's order)
      const int start = p.rev ? wr * 32 + 31 : wr * 32;
      const float hr = d.hi[r], lr = d.lo[r], f = between(d, r, start) * p.s_intra;
      const float *back = d.back[p.rev ? max(0, 2 - wr) : max(0, wr - 1)];
      float row = 0.f;
#pragma unroll 1
      for (int g = 0; g < 2; ++g) {                      // 32 columns at a time, 16 columns of TMEM as bfloat16
        const int cb = half * 2 + g;                     // block of 32 columns
        uint32_t packed[16];
        if (p.rev ? cb < wr : cb > wr) {
#pragma unroll
          for (int j = 0; j < 16; ++j) packed[j] = 0u;
          if (cross) cols_[wr][cb * 32 + lane] = 0.f;
        } else {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int c = cb * 32 + q * 16;
            float v[16], x2[16];
            __syncwarp();
            if constexpr (cross) tmem_ld16x2(tm_own + tP + c, tm_own + tO + c, v, x2);
            else tmem_ld16(tm_own + tP + c, v);
            if (cb != wr) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float4 w = *reinterpret_cast<const float4 *>(&back[c + 4 * j]);
                v[4 * j] *= f * w.x;
                v[4 * j + 1] *= f * w.y;
                v[4 * j + 2] *= f * w.z;
                v[4 * j + 3] *= f * w.w;
              }
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float4 hi = *reinterpret_cast<const float4 *>(&d.hi[c + 4 * j]), lo = *reinterpret_cast<const float4 *>(&d.lo[c + 4 * j]);
                const float x[4] = {(hr - hi.x) + (lr - lo.x), (hr - hi.y) + (lr - lo.y), (hr - hi.z) + (lr - lo.z), (hr - hi.w) + (lr - lo.w)};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const bool on = p.rev ? c + 4 * j + e >= r : c + 4 * j + e <= r;
                  const float w = ex2a(on ? x[e] : 0.f) * p.s_intra;
                  v[4 * j + e] = on ? v[4 * j + e] * w : 0.f;
                }
              }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const __nv_bfloat162 w = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
              packed[q * 8 + j] = *reinterpret_cast<const uint32_t *>(&w);
            }
            if (cross) {                                 // products of a pair's two scores, without the diagonal
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                v[j] = c + j == r ? 0.f : v[j] * x2[j];
                row += v[j];
              }
              const float col = sum_columns(v, lane);
              if (lane < 16) cols_[wr][c + lane] = col;
            }
          }
        }
        // the columns of 32 scores are free once read; their bfloat16 go into the first half of this half's 64 columns, which
        // the first of the two rounds has read
        __syncwarp();
        tmem_st16(tm_own + tP + half * 64 + g * 16, packed);
      }
      if (cross) rows_[half][r] = row;
      tmem_st_wait();
    }
    if (!cross && issuer) {                              // keys and q are free once the sum is there
      if (!mbar_wait(&bar_d, it & 1, kWaitLimit)) *(volatile int *)&fail = 1;
      if (maps.tma && i0 + BC < i_end) copy_qk(i0 + BC);
    }
    __syncwarp();
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();                                     // scores (and backwards the values' terms) are written
    if (!STATE_ONLY && issuer) {
      tc_fence_after();
      const uint64_t v = smem_desc(smem_u32(sv), 8192, 1024, 2);
#pragma unroll
      for (int i = 0; i < BC / 16; ++i) mma_f16_ta(tm + tO, tm + tP + (i >> 2) * 64 + (i & 3) * 8, v + i * 128, kState, i > 0);
      if (cross) issue_update();
      mma_commit(&bar);
    }
    if (grad && warp == sum_warp) {                      // before the next chunk's take their place
      dot_sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = in_time(p, 4 * lane + j);
        const float dot = dots[0][i] + dots[1][i];
        dot_sum += dot;
        pairs[j] = two(dot);
        if (cross) pairs[j] = (pairs[j] + (two(rows_[0][i]) + two(rows_[1][i]))) + -((two(cols_[0][i]) + two(cols_[1][i])) + (two(cols_[2][i]) + two(cols_[3][i])));
      }
    }
    __syncwarp();
    if (!cross) wait_products(bar_d, it & 1);
    if (!STATE_ONLY) {
      wait_products(bar, phase);
      phase ^= 1;
    }
    const bool more = i0 + BC < i_end, staged = !STATE_ONLY && maps.tma_out;
    if (more) {
      if (!maps.tma) {
        if (!staged) load_all(i0 + BC);                  // else once the results have left
      } else if (issuer) {
        if (cross) copy_qk(i0 + BC);
        if (!staged) copy_v(i0 + BC);
      }
      __syncwarp();
    }
    if constexpr (!STATE_ONLY) {
      float v[32];
      tmem_ld32(tm_own + tO + c0, v);
#pragma unroll
      for (int j = 0; j < 32; ++j) O[j] += v[j];
      if (odd[it & 1]) {
        const int i = p.rev ? BC - 1 - r : r;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (i >= odd_from[it & 1][c0 + j]) O[j] = __int_as_float(0x7fffffff);
      }
      const int t = time0(i0) + r, left = p.dout - col0 - c0;
      if (staged) {                                      // by way of shared memory, where v (and x) were
        if (p.out_f32) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<float4 *>(sv + half * BTILE + piece_at(r, j)) = make_float4(O[4 * j], O[4 * j + 1], O[4 * j + 2], O[4 * j + 3]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const __nv_bfloat162 x = __floats2bfloat162_rn(O[j * 8 + 2 * e], O[j * 8 + 2 * e + 1]);
              w[e] = *reinterpret_cast<const uint32_t *>(&x);
            }
            *reinterpret_cast<uint4 *>(sv + piece_at(r, half * 4 + j)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        fence_proxy_async();
        __syncthreads();
        if (issuer) {
          tma_st_4d(&maps.out, sv, col0, h, time0(i0), b);
          if (p.out_f32 && col0 + 32 < p.dout) tma_st_4d(&maps.out, sv + BTILE, col0 + 32, h, time0(i0), b);
          bulk_commit();
        }
        __syncwarp();
      } else if (t < p.length && left > 0) {
        const int64_t at = b * p.o_bs + t * p.o_ls + h * p.o_hs + col0 + c0;
        if (p.out_f32) {
          float *o = reinterpret_cast<float *>(p.out) + at;
          if (left >= 32 && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) reinterpret_cast<float4 *>(o)[j] = make_float4(O[4 * j], O[4 * j + 1], O[4 * j + 2], O[4 * j + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j < left) o[j] = O[j];
          }
        } else {
          __nv_bfloat16 *o = reinterpret_cast<__nv_bfloat16 *>(p.out) + at;
          if (left >= 32 && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const __nv_bfloat162 x = __floats2bfloat162_rn(O[j * 8 + 2 * e], O[j * 8 + 2 * e + 1]);
                w[e] = *reinterpret_cast<const uint32_t *>(&x);
              }
              reinterpret_cast<uint4 *>(o)[j] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j < left) o[j] = __float2bfloat16_rn(O[j]);
          }
        }
      }
    }
    {
      float v[NS];
      __syncwarp();                                      // lanes come from their own stores
      if constexpr (NS == 32) tmem_ld32(tm_own + tD + cs, v);
      else tmem_ld16(tm_own + tD + cs, v);
      const float keep = d.keep, keep_lo = d.keep_lo;
#pragma unroll
      for (int j = 0; j < NS; ++j) S[j] = fmaf(S[j], keep, fmaf(S[j], keep_lo, v[j]));
    }
    if (STATE_ONLY) total += (double)d.total.h + (double)d.total.l;
    if (cross && chunk % kSnapB == 0) snapshot(chunk / kSnapB, (float)exp2_two(log2_of(p, b, h, chunk * BC)));
    if (!STATE_ONLY) write_terms();
    if (staged && more) {
      if (issuer) {
        bulk_wait_read<0>();
        if (maps.tma) copy_v(i0 + BC);
        if (maps.tma && !cross && mbar_wait(&loaded_qk, (it + 1) & 1, 1)) {      // where they have arrived, the next scores start now
          tc_fence_after();
          issue_scores();
          scores_on = true;
        }
      }
      __syncwarp();
      if (!maps.tma) {
        __syncthreads();                                 // the results have left
        load_all(i0 + BC);
      }
    }
  }
  const bool ok = !__syncthreads_or(*(volatile int *)&fail);
  if (grad && warp == sum_warp && i_end > i_begin && ok) chunk_runs(p, tile, bh, i_end - BC, lane, pairs, dot_sum);
  if (!STATE_ONLY && issuer) bulk_wait<0>();
  if (!ok && issuer)
    for (int i = 0; i < 1 << 12; ++i) __nanosleep(256);  // copies and products in flight: a millisecond, many times what they take
  __syncwarp();
  if (STATE_ONLY && ok) {
    each([&](int c, float &x) { p.seg[(((int64_t)bh * p.nseg + seg) * p.di + rs) * p.dout + c] = x; });
    if (tile == 0 && tid == 0) p.seg_g[(int64_t)bh * p.nseg + seg] = total;
  } else if (!STATE_ONLY && ok && p.last && seg == p.nseg - 1) {
    const float f = p.last_decay ? (float)exp2_two(log2_of(p, b, h, 0)) : 1.f;
    each([&](int c, float &x) { p.last[b * p.last_bs + h * p.last_hs + rs * p.last_is + c * p.last_os] = x * f; });
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(256) : "memory");
  if (tid == 0 && fail) atomicExch(&g_linattn_status, 9);
  if (blockIdx.x == gridDim.x - 1) wait_for_last();
}

// Each segment's own state becomes the state before it.
__global__ void __launch_bounds__(256) linattn_join_kernel(const Walk p) {
  __shared__ float keep[kMaxSeg];
  const int64_t per = (int64_t)p.di * p.dout, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int bh = blockIdx.y, b = bh / p.heads, h = bh % p.heads;
  if (threadIdx.x < p.nseg - 1) keep[threadIdx.x] = (float)exp2(p.seg_g[(int64_t)bh * p.nseg + threadIdx.x]);
  __syncthreads();
  if (i >= per) return;
  float s = 0.f;
  if (p.s0) s = p.s0[b * p.s0_bs + h * p.s0_hs + i / p.dout * p.s0_is + i % p.dout * p.s0_os];
  float *at = p.seg + (int64_t)bh * p.nseg * per + i;
  for (int n0 = 0; n0 < p.nseg; n0 += 8) {              // eight segments' loads in flight
    float own[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) own[j] = n0 + j < p.nseg - 1 ? at[(n0 + j) * per] : 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (n0 + j < p.nseg) {
        at[(n0 + j) * per] = s;
        if (n0 + j < p.nseg - 1) s = fmaf(s, keep[n0 + j], own[j]);
      }
  }
}

// Gradients of operands that several heads share: the sum over the heads of a group.
template <typename T>
__global__ void __launch_bounds__(256) linattn_fold_kernel(const float *src, int64_t rows, int heads, int groups, int d, T *dst) {
  const int64_t n = rows * groups * d;
  const int per = heads / groups;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t rg = i / d;
    const int c = (int)(i - rg * d);
    const float *s = src + rg * per * d + c;
    float v = 0.f;
    for (int j = 0; j < per; ++j) v += s[(int64_t)j * d];
    dst[i] = T(v);
  }
}

// What the pairs of steps on both sides of a whole chunk give: every 512 steps all pairs across a border are the product of
// the two states there, and from border to border the sums of the chunk's dots are taken off and added on.
__global__ void __launch_bounds__(256) linattn_across_kernel(const float *snap_q, const float *snap_k, const float *sum_q, const float *sum_k, int tiles, int64_t per,
                                                            int chunks, int snap, int snaps, int bhs, double *across) {
  __shared__ double sh[8];
  const int bh = blockIdx.x / snaps, sn = blockIdx.x % snaps, tid = threadIdx.x;
  const float *a = snap_q + (int64_t)blockIdx.x * per, *c = snap_k + (int64_t)blockIdx.x * per;
  double s = 0.0;
  for (int64_t i = tid; i < per; i += 256) s += (double)a[i] * (double)c[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((tid & 31) == 0) sh[tid >> 5] = s;
  __syncthreads();
  if (tid == 0) {
    double x = 0.0;
    for (int i = 0; i < 8; ++i) x += sh[i];
    for (int n = sn * snap; n < min(chunks, (sn + 1) * snap); ++n) {
      double q = 0.0, k = 0.0;
      for (int t = 0; t < tiles; ++t) {
        q += (double)sum_q[((int64_t)t * bhs + bh) * chunks + n];
        k += (double)sum_k[((int64_t)t * bhs + bh) * chunks + n];
      }
      x -= q;
      across[(int64_t)bh * chunks + n] = x;
      x += k;
    }
  }
}

__device__ __forceinline__ double dg_at(const b200_linattn_args &p, const float *run_q, const float *run_k, int tiles, const double *across, int ch, int chunks, int bh, int t) {
  const int b = bh / p.heads, h = bh % p.heads;
  if (load_g(p.g, p.g_dtype, b * p.g_bs + t * p.g_ls + h * p.g_hs) == -INFINITY) return 0.0;      // a decay of nothing has no slope
  const int64_t plane = (int64_t)p.batch * p.heads * p.seqlen, i = (int64_t)bh * p.seqlen + t;
  double s = across[(int64_t)bh * chunks + t / ch];
  for (int n = 0; n < tiles; ++n) s += (double)run_q[n * plane + i] + (double)run_k[n * plane + i];
  return s;
}
// 32 steps x 8 heads a block, so that both layouts are read and written in runs
__global__ void __launch_bounds__(256) linattn_dg_kernel(const b200_linattn_args p, const float *run_q, const float *run_k, int tiles, const double *across, int ch, int chunks) {
  __shared__ float sh[8][33];
  const int b = blockIdx.z, t0 = blockIdx.x * 32, h0 = blockIdx.y * 8;
  {
    const int t = t0 + (threadIdx.x & 31), h = h0 + (threadIdx.x >> 5);
    sh[threadIdx.x >> 5][threadIdx.x & 31] = t < p.seqlen && h < p.heads ? (float)dg_at(p, run_q, run_k, tiles, across, ch, chunks, b * p.heads + h, t) : 0.f;
  }
  __syncthreads();
  const int t = t0 + (threadIdx.x >> 3), h = h0 + (threadIdx.x & 7);
  if (t < p.seqlen && h < p.heads) st_act(p.dg, p.g_dtype, ((int64_t)b * p.seqlen + t) * p.heads + h, sh[threadIdx.x & 7][threadIdx.x >> 3]);
}
// a decay for each head: the sum over a (batch, head), then over the batch
__global__ void __launch_bounds__(256) linattn_dg_sum_kernel(const b200_linattn_args p, const float *run_q, const float *run_k, int tiles, const double *across, int ch, int chunks,
                                                            double *per_head) {
  __shared__ double sh[8];
  double s = 0.0;
  for (int t = threadIdx.x; t < p.seqlen; t += 256) s += dg_at(p, run_q, run_k, tiles, across, ch, chunks, blockIdx.x, t);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int i = 0; i < 8; ++i) s += sh[i];
    per_head[blockIdx.x] = s;
  }
}
__global__ void linattn_dg_heads_kernel(const b200_linattn_args p, const double *per_head) {
  const int h = blockIdx.x * blockDim.x + threadIdx.x;
  if (h >= p.heads) return;
  double s = 0.0;
  for (int b = 0; b < p.batch; ++b) s += per_head[(int64_t)b * p.heads + h];
  st_act(p.dg, p.g_dtype, h, (float)s);
}

// ------------------------------------------------------------------------------------------------ one token

// A block takes a (batch entry, head): the state is read and written once, 16 bytes an access where its rows allow it, eight
// rows a thread in flight before the keys and queries are.  Threads along the state's rows of dv, and groups of them along dk
// whose sums are joined in shared memory.  Bound by HBM: 64 x 24 heads of 128 x 64 float32 (101 MB) 22.3 us, 0.69 of the copy rate with
// the launch; 14.8 us where the state is in L2.
template <typename TS, int VEC> struct Piece { typedef uint4 type; };
template <typename TS> struct Piece<TS, 1> { typedef TS type; };
template <typename TS, typename T, int VEC> __global__ void __launch_bounds__(128) linattn_step_kernel(const b200_linattn_step_args p) {
  __shared__ float sh[128 * VEC], sq[MAX_D], sk[MAX_D];
  const int b = blockIdx.x / p.heads, h = blockIdx.x % p.heads, grp = h / (p.heads / p.groups), tid = threadIdx.x;
  const T *v = reinterpret_cast<const T *>(p.v) + b * p.v_bs + h * p.v_hs;
  T *out = reinterpret_cast<T *>(p.out) + b * p.out_bs + h * p.out_hs;
  int64_t slot = b;
  if (p.state_batch_indices) {
    slot = p.state_batch_indices[b];
    if (slot < 0 || slot >= p.slots) {                    // no state: padding of the batch
      for (int c = tid; c < p.dv; c += 128) out[c] = T(0.f);
      return;
    }
  }
  const int across = (p.dv + VEC - 1) / VEC, along = 128 / across;           // threads along dv (at most 128) and along dk
  const int cx = tid % across, ry = tid / across, c0 = cx * VEC;
  typename Piece<TS, VEC>::type *S = reinterpret_cast<typename Piece<TS, VEC>::type *>(reinterpret_cast<TS *>(p.state) + slot * p.state_bs + h * p.state_hs + c0);
  const int64_t row = p.state_ks / VEC;
  // the state's rows are on their way before anything else is
  constexpr int AHEAD = 8;
  typename Piece<TS, VEC>::type e[AHEAD];
  const auto load = [&](int r0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int r = r0 + i * along;
      if (ry < along && r < p.dk) e[i] = S[r * row];
    }
  };
  load(ry);
  for (int i = tid; i < p.dk; i += 128) {
    sq[i] = (float)reinterpret_cast<const T *>(p.q)[b * p.q_bs + grp * p.q_gs + i] * p.scale;
    sk[i] = (float)reinterpret_cast<const T *>(p.k)[b * p.k_bs + grp * p.k_gs + i];
  }
  const float a = expf(load_g(p.g, p.g_dtype, b * p.g_bs + h * p.g_hs));
  __syncthreads();
  float acc[VEC], vv[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    acc[j] = 0.f;
    vv[j] = (float)v[c0 + j];
  }
  if (ry < along) {
    for (int r0 = ry; r0 < p.dk; r0 += AHEAD * along) {
      if (r0 > ry) load(r0);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int r = r0 + i * along;
        if (r >= p.dk) break;
        TS *x = reinterpret_cast<TS *>(&e[i]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float y = fmaf(a, (float)x[j], sk[r] * vv[j]);
          acc[j] = fmaf(sq[r], y, acc[j]);
          x[j] = TS(y);
        }
        S[r * row] = e[i];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) sh[tid * VEC + j] = acc[j];
  __syncthreads();
  for (int c = tid; c < p.dv; c += 128) {
    float s = 0.f;
    for (int r = 0; r < along; ++r) s += sh[(r * across) * VEC + c];
    out[c] = T(s);
  }
}

// ------------------------------------------------------------------------------------------------ host

int64_t up(int64_t n, int64_t unit) { return (n + unit - 1) / unit * unit; }

constexpr int walk_smem(int di, bool state_only, bool with_x) {
  return 4 * (CH * (di + 4) + CH * PV + di * PV + (state_only ? 0 : CH * (di + 4) + (with_x ? 2 : 1) * CH * PP));
}

// Segments: as many as make the walk shortest.  Counted in chunks that an SM goes through with as many blocks as fit it
// (`resident`; a last round that leaves the SMs one block each takes 0.6 of one), one more for a block's start; the first pass over
// the segments takes 0.7 of the second.  A prompt of 16384 steps x 16 heads of 128 x 128: 9 segments.
double rounds_of(int64_t blocks, int resident) {
  const int64_t sms = sm_count_current(), slots = sms * resident, left = blocks % slots;
  return (double)(blocks / slots) + (left == 0 ? 0.0 : left <= sms && resident > 1 ? 0.6 : 1.0);
}
int segments(int64_t blocks, int chunks, int resident, double &cost) {
  int best = 1;
  cost = 1e30;
  for (int n = 1; n <= kMaxSeg && n <= chunks; ++n) {
    const int per = (chunks + n - 1) / n;
    if ((int64_t)(n - 1) * per >= chunks) continue;
    const double c = rounds_of(blocks * n, resident) * (per + 1) * (n > 1 ? 1.7 : 1.0) + (n > 1 ? 1 : 0);
    if (c < cost * 0.97) { cost = c; best = n; }
  }
  return best;
}

double cut(Walk &w) {
  const int chunks = w.chunks;
  w.tiles = (w.dout + DO - 1) / DO;
  double cost;
  const int n = segments((int64_t)w.batch * w.heads * w.tiles, chunks, w.ch == BC || w.di <= 64 ? 2 : 1, cost);
  w.seg_chunks = (chunks + n - 1) / n;
  w.nseg = (chunks + w.seg_chunks - 1) / w.seg_chunks;
  return cost;
}
int64_t seg_bytes(int64_t bh, int nseg, int di, int dout) { return nseg > 1 ? up(4 * bh * nseg * di * dout, 256) + up(8 * bh * nseg, 256) : 0; }

// the launches of a walk: `own` and `all` are its kernels for a segment's own state and for the results
template <typename K, typename... More>
int launch_walk(Walk &w, K own, K all, int threads, int smem_own, int smem_all, unsigned char *work, cudaStream_t st, More... more) {
  const int64_t bh = (int64_t)w.batch * w.heads;
  cudaError_t e = cudaFuncSetAttribute(all, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_all);
  if (e == cudaSuccess && w.nseg > 1) e = cudaFuncSetAttribute(own, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_own);
  if (e != cudaSuccess) { set_error("cudaFuncSetAttribute: %s", cudaGetErrorString(e)); return (int)e; }
  if (w.nseg > 1) {
    w.seg = reinterpret_cast<float *>(work);
    w.seg_g = reinterpret_cast<double *>(work + up(4 * bh * w.nseg * w.di * w.dout, 256));
    own<<<(unsigned)(bh * w.tiles * (w.nseg - 1)), threads, smem_own, st>>>(w, more...);
    const int64_t per = (int64_t)w.di * w.dout;
    linattn_join_kernel<<<dim3((unsigned)((per + 255) / 256), (unsigned)bh), 256, 0, st>>>(w);
    if (int r = launch_status()) return r;
  }
  cudaLaunchAttribute beside = {};
  beside.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  beside.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(bh * w.tiles * w.nseg));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem_all;
  cfg.stream = st;
  cfg.attrs = &beside;
  cfg.numAttrs = w.beside && w.nseg == 1 ? 1 : 0;          // segments' states lie in the workspace that the walks share
  e = cudaLaunchKernelEx(&cfg, all, (const Walk)w, more...);
  if (e != cudaSuccess) { set_error("CUDA launch failed: %s", cudaGetErrorString(e)); return (int)e; }
  return launch_status();
}
template <typename T, int DI, int WT> int walk(Walk &w, unsigned char *work, cudaStream_t st) {
  return launch_walk(w, linattn_walk_kernel<T, DI, WT, true>, linattn_walk_kernel<T, DI, WT, false>, WT, walk_smem(DI, true, false),
                     walk_smem(DI, false, w.run != nullptr), work, st);
}
template <typename T> int walk(Walk &w, unsigned char *work, cudaStream_t st) {
  if (w.di > 64) return walk<T, 128, 512>(w, work, st);
  const int64_t blocks = (int64_t)w.batch * w.heads * w.tiles * w.nseg;
  return blocks > sm_count_current() ? walk<T, 64, 256>(w, work, st) : walk<T, 64, 512>(w, work, st);
}
bool map_of(CUtensorMap *m, const void *base, int size, int heads, int length, int batch, int64_t hs, int64_t ls, int64_t bs, bool f32 = false) {
  EncodeTiledFn enc = encoder();
  if (!enc || (reinterpret_cast<uintptr_t>(base) & 15)) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)size, (cuuint64_t)heads, (cuuint64_t)length, (cuuint64_t)batch};
  const int unit = f32 ? 4 : 2;
  int64_t st[3] = {heads > 1 ? hs : 8, length > 1 ? ls : 8, batch > 1 ? bs : 8};
  for (int64_t x : st)
    if (x <= 0 || x * unit % 16 || x >= (int64_t(1) << 37)) return false;
  const cuuint64_t strides[3] = {(cuuint64_t)st[0] * unit, (cuuint64_t)st[1] * unit, (cuuint64_t)st[2] * unit};
  const cuuint32_t box[4] = {(cuuint32_t)(128 / unit), 1, BC, 1}, one[4] = {1, 1, 1, 1};
  return enc(m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
template <int DI> int walk_tc(Walk &w, unsigned char *work, cudaStream_t st) {
  const int ts = w.run ? 3 : 1, tu = w.run || w.last ? 3 : 2, kv = DI / 64 * BTILE + BTILE + 1024;
  const int own = tu * BTILE + kv, all = terms_bytes(DI, ts, tu) + kv + (w.run ? BTILE : 0);
  const auto results = !w.run ? linattn_walk_tc_kernel<DI, RESULTS> : w.rev ? linattn_walk_tc_kernel<DI, DOTS_REV> : linattn_walk_tc_kernel<DI, DOTS>;
  Maps m;
  memset(&m, 0, sizeof(m));
  m.tma = map_of(&m.q, w.q, w.di, w.heads / w.q_div, w.length, w.batch, w.q_hs, w.q_ls, w.q_bs) &&
          map_of(&m.k, w.k, w.di, w.heads / w.k_div, w.length, w.batch, w.k_hs, w.k_ls, w.k_bs) &&
          map_of(&m.v, w.v, w.dout, w.heads / w.v_div, w.length, w.batch, w.v_hs, w.v_ls, w.v_bs) &&
          (!w.run || map_of(&m.x, w.x, w.dout, w.heads / w.x_div, w.length, w.batch, w.x_hs, w.x_ls, w.x_bs));
  // float32 results take the room of v and x
  m.tma_out = (!w.out_f32 || w.run) && map_of(&m.out, w.out, w.dout, w.heads, w.length, w.batch, w.o_hs, w.o_ls, w.o_bs, w.out_f32);
  return launch_walk(w, linattn_walk_tc_kernel<DI, OWN_STATE>, results, BT, own, all, work, st, m, tu);
}
int run_walk(int dtype, Walk &w, unsigned char *work, cudaStream_t st) {
  if (dtype == B200_F32) return walk<float>(w, work, st);
  if (dtype == B200_F16) return walk<__half>(w, work, st);
  return w.di <= 64 ? walk_tc<64>(w, work, st) : walk_tc<128>(w, work, st);
}

int check_linattn(const b200_linattn_args &a) {
  B200_REQUIRE(a.q && a.k && a.v && a.g, B200_ERR_NULL, "linattn: q, k, v and g must be non-null");
  B200_REQUIRE(a.batch > 0 && a.seqlen > 0 && a.heads > 0 && a.groups > 0 && a.dk > 0 && a.dv > 0, B200_ERR_SHAPE, "linattn: sizes must be positive");
  B200_REQUIRE(a.dk <= MAX_D && a.dv <= MAX_D, B200_ERR_SHAPE, "linattn: head sizes up to %d (got dk=%d dv=%d)", MAX_D, a.dk, a.dv);
  B200_REQUIRE(a.heads % a.groups == 0, B200_ERR_SHAPE, "linattn: heads (%d) must be a multiple of groups (%d)", a.heads, a.groups);
  B200_REQUIRE((int64_t)a.batch * a.heads <= 65535 && a.seqlen <= (1 << 30), B200_ERR_SHAPE, "linattn: batch * heads up to 65535 (got %d * %d)", a.batch, a.heads);
  B200_REQUIRE(a.dtype == B200_F32 || a.dtype == B200_F16 || a.dtype == B200_BF16, B200_ERR_DTYPE, "linattn: unknown dtype %d", a.dtype);
  B200_REQUIRE(a.g_dtype == B200_F32 || a.g_dtype == a.dtype, B200_ERR_DTYPE, "linattn: g is float32 or of the dtype of q, k, v");
  B200_REQUIRE((reinterpret_cast<uintptr_t>(a.work) & 255) == 0, B200_ERR_ALIGN, "linattn: work must be 256-byte aligned");
  return 0;
}

Walk base_walk(const b200_linattn_args &a) {
  Walk w;
  memset(&w, 0, sizeof(w));
  w.g = a.g; w.g_bs = a.g_bs; w.g_ls = a.g_ls; w.g_hs = a.g_hs; w.g_dtype = a.g_dtype;
  w.batch = a.batch; w.length = a.seqlen; w.heads = a.heads;
  w.ch = a.dtype == B200_BF16 ? BC : CH;
  w.chunks = (a.seqlen + w.ch - 1) / w.ch;
  w.q_div = w.k_div = w.v_div = w.x_div = 1;
  return w;
}
#define ROLE(slot, from)                                          \
  do {                                                            \
    w.slot = a.from;                                              \
    w.slot##_bs = a.from##_bs;                                    \
    w.slot##_ls = a.from##_ls;                                    \
    w.slot##_hs = a.from##_hs;                                    \
  } while (0)

// the walks: o, dq, dk, dv
Walk walk_o(const b200_linattn_args &a) {
  Walk w = base_walk(a);
  ROLE(q, q); ROLE(k, k); ROLE(v, v);
  w.q_div = w.k_div = a.heads / a.groups;
  w.di = a.dk; w.dout = a.dv;
  w.s_inter = w.s_intra = a.scale; w.s_update = 1.f;
  w.s0 = reinterpret_cast<const float *>(a.s0);
  w.s0_bs = a.s0_bs; w.s0_hs = a.s0_hs; w.s0_is = a.s0_ks; w.s0_os = 1;
  w.out = a.out; w.o_bs = a.out_bs; w.o_ls = a.out_ls; w.o_hs = a.out_hs;
  w.last = reinterpret_cast<float *>(a.last);
  w.last_bs = (int64_t)a.heads * a.dk * a.dv; w.last_hs = (int64_t)a.dk * a.dv; w.last_is = a.dv; w.last_os = 1;
  cut(w);
  return w;
}
Walk walk_dq(const b200_linattn_args &a) {
  Walk w = base_walk(a);
  ROLE(q, dout); ROLE(k, v); ROLE(v, k); ROLE(x, q);
  w.v_div = w.x_div = a.heads / a.groups;
  w.di = a.dv; w.dout = a.dk;
  w.s_inter = w.s_intra = a.scale; w.s_update = 1.f;
  w.s0 = reinterpret_cast<const float *>(a.s0);
  w.s0_bs = a.s0_bs; w.s0_hs = a.s0_hs; w.s0_is = 1; w.s0_os = a.s0_ks;
  return w;
}
Walk walk_dk(const b200_linattn_args &a) {
  Walk w = base_walk(a);
  ROLE(q, v); ROLE(k, dout); ROLE(v, q); ROLE(x, k);
  w.v_div = w.x_div = a.heads / a.groups;
  w.di = a.dv; w.dout = a.dk;
  w.rev = 1;
  w.s_inter = 1.f; w.s_intra = w.s_update = a.scale;
  w.s0 = reinterpret_cast<const float *>(a.dlast);
  w.s0_bs = (int64_t)a.heads * a.dk * a.dv; w.s0_hs = (int64_t)a.dk * a.dv; w.s0_is = 1; w.s0_os = a.dv;
  return w;
}
Walk walk_dv(const b200_linattn_args &a) {
  Walk w = base_walk(a);
  ROLE(q, k); ROLE(k, q); ROLE(v, dout);
  w.q_div = w.k_div = a.heads / a.groups;
  w.di = a.dk; w.dout = a.dv;
  w.rev = 1;
  w.s_inter = 1.f; w.s_intra = w.s_update = a.scale;
  w.s0 = reinterpret_cast<const float *>(a.dlast);
  w.s0_bs = (int64_t)a.heads * a.dk * a.dv; w.s0_hs = (int64_t)a.dk * a.dv; w.s0_is = a.dv; w.s0_os = 1;
  w.out = a.dv_out; w.o_bs = (int64_t)a.seqlen * a.heads * a.dv; w.o_ls = (int64_t)a.heads * a.dv; w.o_hs = a.dv;
  w.last = reinterpret_cast<float *>(a.ds0);
  w.last_bs = w.s0_bs; w.last_hs = w.s0_hs; w.last_is = a.dv; w.last_os = 1;
  w.last_decay = 1;
  return w;
}

// dq, dk and dv: whole sequences, which run beside one another, where by the count above that takes no longer than the
// segments of each, one walk after the other; a sequence of dk takes 1.4 times as long as the others.  9 x 2752 steps, 8 heads of
// 128 x 32, bfloat16, with the forward: 634 -> 587 us; 320 steps, 16 heads of 64 x 81, float32: 210 -> 195 us; where the count says
// segments, 3 x 777 steps, 6 heads of 48 x 77, float32: 308, whole sequences 361 us.
struct Walks { Walk dq, dk, dv; };
Walks backward_walks(const b200_linattn_args &a) {
  Walks ws = {walk_dq(a), walk_dk(a), walk_dv(a)};
  const int64_t bh = (int64_t)a.batch * a.heads;
  int64_t blocks = 0, most = 0;
  double apart = 0;
  for (Walk *w : {&ws.dq, &ws.dk, &ws.dv}) {
    apart += cut(*w);
    blocks += bh * w->tiles;
    most = std::max(most, bh * w->tiles);
  }
  const bool two = a.dtype == B200_BF16 || (a.dk <= 64 && a.dv <= 64 && most > sm_count_current());      // blocks on an SM
  if (std::max(rounds_of(blocks, two ? 2 : 1), 1.4 * rounds_of(1, two ? 2 : 1)) * (ws.dq.chunks + 1) <= apart)
    for (Walk *w : {&ws.dq, &ws.dk, &ws.dv}) {
      w->nseg = 1;
      w->seg_chunks = w->chunks;
    }
  return ws;
}

struct BwdPlan { int64_t seg, part, run, sum, snap, across, heads, total; };
BwdPlan bwd_plan(const b200_linattn_args &a) {
  BwdPlan q;
  const int64_t bh = (int64_t)a.batch * a.heads;
  const Walks ws = backward_walks(a);
  q.seg = 0;
  for (const Walk *w : {&ws.dq, &ws.dk, &ws.dv}) q.seg = std::max(q.seg, seg_bytes(bh, w->nseg, w->di, w->dout));
  const int64_t chunks = ws.dq.chunks;
  q.part = a.heads != a.groups ? up(4 * bh * a.seqlen * a.dk, 256) : 0;          // of each of dq and dk
  q.run = a.dg ? up(4 * bh * a.seqlen * ws.dq.tiles, 256) : 0;
  q.sum = a.dg ? up(4 * bh * chunks * ws.dq.tiles, 256) : 0;
  q.snap = a.dg ? up(4 * bh * ((a.seqlen + kSnapSteps - 1) / kSnapSteps) * a.dk * a.dv, 256) : 0;
  q.across = a.dg ? up(8 * bh * chunks, 256) : 0;
  q.heads = a.dg && a.g_heads ? up(8 * bh, 256) : 0;
  q.total = q.seg + 2 * (q.part + q.run + q.sum + q.snap) + q.across + q.heads;
  return q;
}

int fold(const b200_linattn_args &a, const float *src, void *dst, cudaStream_t st) {
  const int64_t rows = (int64_t)a.batch * a.seqlen, n = rows * a.groups * a.dk, most = (int64_t)sm_count_current() * 16;
  const unsigned grid = (unsigned)((n + 255) / 256 < most ? (n + 255) / 256 : most);
  if (a.dtype == B200_F32) linattn_fold_kernel<float><<<grid, 256, 0, st>>>(src, rows, a.heads, a.groups, a.dk, reinterpret_cast<float *>(dst));
  else if (a.dtype == B200_F16) linattn_fold_kernel<__half><<<grid, 256, 0, st>>>(src, rows, a.heads, a.groups, a.dk, reinterpret_cast<__half *>(dst));
  else linattn_fold_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(src, rows, a.heads, a.groups, a.dk, reinterpret_cast<__nv_bfloat16 *>(dst));
  return launch_status();
}

template <typename TS, typename T> int run_step(const b200_linattn_step_args &a, cudaStream_t st) {
  constexpr int V = 16 / sizeof(TS);
  const bool vec = a.dv % V == 0 && (reinterpret_cast<uintptr_t>(a.state) & 15) == 0 && a.state_bs % V == 0 && a.state_hs % V == 0 && a.state_ks % V == 0;
  const unsigned grid = (unsigned)((int64_t)a.batch * a.heads);
  if (vec) linattn_step_kernel<TS, T, V><<<grid, 128, 0, st>>>(a);
  else linattn_step_kernel<TS, T, 1><<<grid, 128, 0, st>>>(a);
  return launch_status();
}

}  // namespace

int linattn_status_read() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_linattn_status, sizeof(int)) != cudaSuccess) return -1;
  return v;
}

}  // namespace b200

using namespace b200;

extern "C" int64_t b200_linattn_fwd_work_bytes(const b200_linattn_args *args) {
  if (!args || check_linattn(*args)) return 0;
  const Walk w = walk_o(*args);
  return seg_bytes((int64_t)w.batch * w.heads, w.nseg, w.di, w.dout);
}

extern "C" int64_t b200_linattn_bwd_work_bytes(const b200_linattn_args *args) {
  if (!args || check_linattn(*args)) return 0;
  return bwd_plan(*args).total;
}

extern "C" int b200_linattn_fwd(const b200_linattn_args *args, void *stream) {
  B200_REQUIRE(args, B200_ERR_NULL, "linattn_fwd: null argument block");
  const b200_linattn_args &a = *args;
  if (int e = check_linattn(a)) return e;
  B200_REQUIRE(a.out, B200_ERR_NULL, "linattn_fwd: out must be non-null");
  const int64_t need = b200_linattn_fwd_work_bytes(args);
  B200_REQUIRE(a.work_bytes >= need && (a.work || !need), B200_ERR_TOO_LARGE, "linattn_fwd: work has %lld bytes, %lld are needed", (long long)a.work_bytes, (long long)need);
  Walk w = walk_o(a);
  return run_walk(a.dtype, w, reinterpret_cast<unsigned char *>(a.work), reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int b200_linattn_bwd(const b200_linattn_args *args, void *stream) {
  B200_REQUIRE(args, B200_ERR_NULL, "linattn_bwd: null argument block");
  const b200_linattn_args &a = *args;
  if (int e = check_linattn(a)) return e;
  B200_REQUIRE(a.dout && a.dq && a.dk_out && a.dv_out, B200_ERR_NULL, "linattn_bwd: dout, dq, dk_out and dv_out must be non-null");
  B200_REQUIRE(!a.dg || (int64_t)a.batch * a.heads * ((a.seqlen + kSnapSteps - 1) / kSnapSteps) < (int64_t(1) << 31), B200_ERR_SHAPE, "linattn_bwd: sizes too large");
  const BwdPlan q = bwd_plan(a);
  B200_REQUIRE(a.work_bytes >= q.total && (a.work || !q.total), B200_ERR_TOO_LARGE, "linattn_bwd: work has %lld bytes, %lld are needed", (long long)a.work_bytes,
               (long long)q.total);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  unsigned char *work = reinterpret_cast<unsigned char *>(a.work);
  unsigned char *at = work + q.seg;
  const auto take = [&](int64_t bytes) { unsigned char *r = at; at += bytes; return r; };
  float *part[2], *run[2], *sum[2], *snap[2];
  for (int i = 0; i < 2; ++i) {
    part[i] = reinterpret_cast<float *>(take(q.part));
    run[i] = reinterpret_cast<float *>(take(q.run));
    sum[i] = reinterpret_cast<float *>(take(q.sum));
    snap[i] = reinterpret_cast<float *>(take(q.snap));
  }
  double *across = reinterpret_cast<double *>(take(q.across)), *heads = reinterpret_cast<double *>(take(q.heads));
  const bool shared = a.heads != a.groups;
  Walks ws = backward_walks(a);
  int tiles = 0, chunks = 0;
  for (int i = 1; i >= 0; --i) {                          // from the longest blocks to the shortest
    Walk &w = i == 0 ? ws.dq : ws.dk;
    w.beside = i == 0;
    w.out = shared ? part[i] : i == 0 ? a.dq : a.dk_out;
    w.out_f32 = shared;
    w.o_bs = (int64_t)a.seqlen * a.heads * a.dk;
    w.o_ls = (int64_t)a.heads * a.dk;
    w.o_hs = a.dk;
    if (a.dg) {
      w.run = run[i];
      w.sum = sum[i];
      w.snap = snap[i];
    }
    tiles = w.tiles;
    chunks = w.chunks;
    if (int e = run_walk(a.dtype, w, work, st)) return e;
  }
  ws.dv.beside = 1;
  if (int e = run_walk(a.dtype, ws.dv, work, st)) return e;
  if (shared) {
    if (int e = fold(a, part[0], a.dq, st)) return e;
    if (int e = fold(a, part[1], a.dk_out, st)) return e;
  }
  if (a.dg) {
    const int bh = a.batch * a.heads, every = kSnapSteps / ws.dq.ch, snaps = (chunks + every - 1) / every;
    linattn_across_kernel<<<(unsigned)((int64_t)bh * snaps), 256, 0, st>>>(snap[0], snap[1], sum[0], sum[1], tiles, (int64_t)a.dk * a.dv, chunks, every, snaps, bh, across);
    if (a.g_heads) {
      linattn_dg_sum_kernel<<<(unsigned)bh, 256, 0, st>>>(a, run[0], run[1], tiles, across, ws.dq.ch, chunks, heads);
      linattn_dg_heads_kernel<<<(unsigned)((a.heads + 127) / 128), 128, 0, st>>>(a, heads);
    } else {
      linattn_dg_kernel<<<dim3((unsigned)((a.seqlen + 31) / 32), (unsigned)((a.heads + 7) / 8), (unsigned)a.batch), 256, 0, st>>>(a, run[0], run[1], tiles, across,
                                                                                                                             ws.dq.ch, chunks);
    }
  }
  return launch_status();
}

extern "C" int b200_linattn_step(const b200_linattn_step_args *args, void *stream) {
  B200_REQUIRE(args, B200_ERR_NULL, "linattn_step: null argument block");
  const b200_linattn_step_args &a = *args;
  B200_REQUIRE(a.state && a.q && a.k && a.v && a.g && a.out, B200_ERR_NULL, "linattn_step: state, q, k, v, g and out must be non-null");
  B200_REQUIRE(a.batch > 0 && a.heads > 0 && a.groups > 0 && a.dk > 0 && a.dv > 0 && a.heads % a.groups == 0, B200_ERR_SHAPE,
               "linattn_step: sizes must be positive, heads a multiple of groups");
  B200_REQUIRE(a.dk <= MAX_D && a.dv <= MAX_D, B200_ERR_SHAPE, "linattn_step: head sizes up to %d (got dk=%d dv=%d)", MAX_D, a.dk, a.dv);
  B200_REQUIRE((int64_t)a.batch * a.heads < (int64_t(1) << 31), B200_ERR_SHAPE, "linattn_step: batch * heads too large");
  B200_REQUIRE(a.dtype == B200_F32 || a.dtype == B200_F16 || a.dtype == B200_BF16, B200_ERR_DTYPE, "linattn_step: unknown dtype %d", a.dtype);
  B200_REQUIRE((a.state_dtype == B200_F32 || a.state_dtype == a.dtype) && (a.g_dtype == B200_F32 || a.g_dtype == a.dtype), B200_ERR_DTYPE,
               "linattn_step: the state and g are float32 or of the dtype of q, k, v");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a.dtype == B200_F32) return run_step<float, float>(a, st);
  if (a.dtype == B200_F16) return a.state_dtype == B200_F32 ? run_step<float, __half>(a, st) : run_step<__half, __half>(a, st);
  return a.state_dtype == B200_F32 ? run_step<float, __nv_bfloat16>(a, st) : run_step<__nv_bfloat16, __nv_bfloat16>(a, st);
}

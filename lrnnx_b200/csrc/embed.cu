// Embedding lookup with a scale, and its gradient by sorted tokens (b200_embed_fwd / b200_embed_bwd), sm_100a.
//
//     out[t] = scale W[ids[t]],        dW[v] = scale sum over t with ids[t] = v of dout[t]
//
// Forward: a copy of rows, 16 bytes a thread; bound by HBM, and by the launch for the few tokens of a decoding step.
// Backward: the (id, position) pairs are sorted by id, stably (least significant digit first, up to 9 bits a pass), so
// that rows of one id lie in the order of their positions: no atomics, the same bits every time.  One cluster of eight
// thread blocks sorts, with its digit counts in distributed shared memory; the other SMs clear the gradient meanwhile.
// Every 16 sorted pairs are a piece, whatever ids they hold, so a frequent token does not make one block slow: a thread
// block adds up the runs of equal ids in its piece in float32 and writes a run that lies inside it; what a run crossing
// borders has in a piece goes to the workspace and is joined by the piece where the run begins, in eight interleaved shares.  Where
// the borders fall within a run depends on the whole list of ids, and with them the order of its sums.  Each row is rounded
// once.  Ids outside [0, classes) and the padding id sort behind all others and are not summed.
//
// Measured (one B200, 16384 tokens as frequent as in text, 50280 x 768 bfloat16): lookup 9 us, sort and clearing 24 us (77 MB cleared;
// the sort alone takes 20, latency of its cluster barriers), sums 14 us, joins 14 us; 58 us in all where the bytes alone take 23.
// From Python the call takes 100 us, autograd's bookkeeping.
#include "common.cuh"
#include "dispatch.h"
#include <cstring>
#include <type_traits>

namespace b200 {
namespace {

constexpr int PIECE = 16;             // sorted pairs a piece
constexpr int SORT_T = 1024, SORT_WARPS = SORT_T / 32, CLUSTER = 8;
constexpr int MAX_BITS = 9, MAX_BINS = 1 << MAX_BITS;
constexpr int ROW_T = 128;

// VEC consecutive elements as floats, by one access of up to 16 bytes
template <int BYTES> struct Word;
template <> struct Word<2> { typedef uint16_t type; };
template <> struct Word<4> { typedef uint32_t type; };
template <> struct Word<8> { typedef uint2 type; };
template <> struct Word<16> { typedef uint4 type; };
template <typename T, int VEC> struct Row {
  typedef typename Word<VEC * sizeof(T)>::type W;
  static __device__ __forceinline__ W raw(const T *p) { return __ldg(reinterpret_cast<const W *>(p)); }
  static __device__ __forceinline__ void open(const W &w, float (&v)[VEC]) {
    const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = (float)e[i];
  }
  static __device__ __forceinline__ void store(T *p, const float (&v)[VEC]) {
    W w;
    T *e = reinterpret_cast<T *>(&w);
#pragma unroll
    for (int i = 0; i < VEC; ++i) e[i] = T(v[i]);
    *reinterpret_cast<W *>(p) = w;
  }
};

__device__ __forceinline__ int64_t id_at(const void *ids, int wide, int64_t t) {
  return wide ? reinterpret_cast<const int64_t *>(ids)[t] : reinterpret_cast<const int32_t *>(ids)[t];
}

// A warp takes up to FWD_PER accesses a lane of one row.
constexpr int FWD_PER = 4;
template <typename T, int VEC> __global__ void __launch_bounds__(256) embed_fwd_kernel(const b200_embed_args p, int parts) {
  const int lane = threadIdx.x & 31, per = p.features / VEC;
  const int64_t n = p.tokens * parts, step = (int64_t)gridDim.x * 8;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += step) {
    const int64_t t = parts == 1 ? i : i / parts;
    const int c0 = (int)(i - t * parts) * (FWD_PER * 32) + lane;
    const int64_t id = id_at(p.ids, p.ids_wide, t);
    T *out = reinterpret_cast<T *>(p.out) + t * p.out_rs;
    if (id >= 0 && id < p.classes) {
      const T *row = reinterpret_cast<const T *>(p.weight) + id * p.weight_rs;
      typename Row<T, VEC>::W w[FWD_PER];
#pragma unroll
      for (int j = 0; j < FWD_PER; ++j)
        if (c0 + j * 32 < per) w[j] = Row<T, VEC>::raw(row + (c0 + j * 32) * VEC);
#pragma unroll
      for (int j = 0; j < FWD_PER; ++j)
        if (c0 + j * 32 < per) {
          float v[VEC];
          Row<T, VEC>::open(w[j], v);
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[e] *= p.scale;
          Row<T, VEC>::store(out + (c0 + j * 32) * VEC, v);
        }
    } else {
      float v[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = __int_as_float(0x7fffffff);      // no such row: NaN
      for (int j = 0; j < FWD_PER; ++j)
        if (c0 + j * 32 < per) Row<T, VEC>::store(out + (c0 + j * 32) * VEC, v);
    }
  }
}

// ------------------------------------------------------------------------------------------------ sort

__device__ __forceinline__ uint32_t key_of(const b200_embed_args &p, int64_t t) {
  const int64_t id = id_at(p.ids, p.ids_wide, t);
  return id >= 0 && id < p.classes && id != p.padding_idx ? (uint32_t)id : (uint32_t)p.classes;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// a word of another block's shared memory, at the place of `p` in this one's
__device__ __forceinline__ uint32_t peer_word(const uint32_t *p, int rank) {
  uint32_t at, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

struct SortArgs {
  uint32_t *keys[2], *pos[2];
  int passes, bits;
};

// The first cluster sorts: each warp has a run of the pairs, counts the digits of 32 at a time by comparing lanes, and places
// them by the same comparison once it knows where each of its digits begins (pairs are read twice, and nothing is kept, so
// that any number of them will do).  The blocks of the other clusters clear the gradient.
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(SORT_T) embed_sort_kernel(const b200_embed_args p, const SortArgs q, int esz) {
  extern __shared__ uint32_t cnt[];                              // (warps, bins)
  __shared__ uint32_t total[MAX_BINS], base[MAX_BINS], ws[32];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, bins = 1 << q.bits;
  if (blockIdx.x >= CLUSTER) {
    const int64_t bytes = (int64_t)p.classes * p.features * esz, words = bytes / 16;
    uint4 *dw = reinterpret_cast<uint4 *>(p.dweight);            // as torch allocates: 16-byte aligned (checked)
    const int64_t step = (int64_t)(gridDim.x - CLUSTER) * SORT_T;
    const int64_t first = (int64_t)(blockIdx.x - CLUSTER) * SORT_T + tid;
    for (int64_t i = first; i < words; i += step) dw[i] = make_uint4(0, 0, 0, 0);
    for (int64_t i = words * 16 + first; i < bytes; i += step) reinterpret_cast<unsigned char *>(p.dweight)[i] = 0;
    return;
  }
  const int rank = blockIdx.x;
  const int64_t per = (p.tokens + CLUSTER * SORT_WARPS * 32 - 1) / (CLUSTER * SORT_WARPS * 32) * 32;     // pairs a warp
  const int64_t t0 = ((int64_t)rank * SORT_WARPS + w) * per, t1 = min(p.tokens, t0 + per);
  for (int pass = 0; pass < q.passes; ++pass) {
    const uint32_t *keys = pass ? q.keys[(pass - 1) & 1] : nullptr, *pos = pass ? q.pos[(pass - 1) & 1] : nullptr;
    uint32_t *keys_out = q.keys[pass & 1], *pos_out = q.pos[pass & 1];
    const int shift = pass * q.bits;
    uint32_t *mine = cnt + w * bins;
    for (int i = lane; i < bins; i += 32) mine[i] = 0;
    __syncwarp();
    const auto key_at = [&](int64_t t) { return t < t1 ? (keys ? __ldcg(keys + t) : key_of(p, t)) : 0u; };
    for (int64_t i = t0; i < t1; i += 32) {
      const int64_t t = i + lane;
      const uint32_t d = t < t1 ? (key_at(t) >> shift) & (bins - 1) : 0xffffffffu;
      const uint32_t peers = __match_any_sync(0xffffffffu, d);
      if (t < t1 && (peers >> lane) == 1u) mine[d] += __popc(peers);      // the last of the equal lanes
      __syncwarp();
    }
    __syncthreads();
    if (tid < bins) {
      uint32_t s = 0;
#pragma unroll 8
      for (int j = 0; j < SORT_WARPS; ++j) {
        const uint32_t c = cnt[j * bins + tid];
        cnt[j * bins + tid] = s;
        s += c;
      }
      total[tid] = s;
    }
    cluster_sync();
    uint32_t before = 0, all = 0;
    if (tid < bins) {
#pragma unroll
      for (int j = 0; j < CLUSTER; ++j) {
        const uint32_t c = peer_word(&total[tid], j);
        before += j < rank ? c : 0;
        all += c;
      }
    }
    uint32_t inc = all;                                          // exclusive sums over the bins
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) ws[w] = inc;
    __syncthreads();
    uint32_t lower = lane < w ? ws[lane] : 0;                    // of the warps before
    lower = __reduce_add_sync(0xffffffffu, lower);
    if (tid < bins) base[tid] = lower + inc - all + before;
    cluster_sync();                                              // counts have been read
    for (int64_t i = t0; i < t1; i += 32) {
      const int64_t t = i + lane;
      const uint32_t key = key_at(t);
      const uint32_t d = t < t1 ? (key >> shift) & (bins - 1) : 0xffffffffu;
      const uint32_t peers = __match_any_sync(0xffffffffu, d);
      if (t < t1) {
        const uint32_t o = base[d] + mine[d] + __popc(peers & ((1u << lane) - 1));
        keys_out[o] = key;
        pos_out[o] = pos ? __ldcg(pos + t) : (uint32_t)t;
      }
      __syncwarp();
      if (t < t1 && (peers >> lane) == 1u) mine[d] += __popc(peers);
      __syncwarp();
    }
    if (pass + 1 < q.passes) cluster_sync();                     // places are written, and visible to the cluster
  }
}

// ------------------------------------------------------------------------------------------------ sums

// One piece, ROW_T * VEC columns.  head[piece]: sum of the run that came in from the piece before; tail[piece]: sum of the run that
// begins here and goes on.  A run that covers the whole piece is a head.
template <typename T, int VEC>
__global__ void __launch_bounds__(ROW_T) embed_sum_kernel(const b200_embed_args p, const uint32_t *keys, const uint32_t *pos, float *head, float *tail) {
  __shared__ uint32_t k[PIECE + 2], at[PIECE];
  const int64_t s0 = (int64_t)blockIdx.x * PIECE;
  const int n = (int)min((int64_t)PIECE, p.tokens - s0);
  if (threadIdx.x < PIECE + 2) {
    const int64_t i = s0 + threadIdx.x - 1;
    k[threadIdx.x] = i >= 0 && i < p.tokens ? keys[i] : 0xffffffffu;
    if (threadIdx.x >= 1 && threadIdx.x <= PIECE) at[threadIdx.x - 1] = i < p.tokens ? pos[i] : 0;
  }
  __syncthreads();
  const int c = (blockIdx.y * ROW_T + threadIdx.x) * VEC;
  if (c >= p.features) return;
  const T *dout = reinterpret_cast<const T *>(p.dout) + c;
  T *dw = reinterpret_cast<T *>(p.dweight) + c;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
  bool came_in = k[0] == k[1];
  typename Row<T, VEC>::W w[PIECE];                            // all rows of the piece in flight
#pragma unroll
  for (int i = 0; i < PIECE; ++i)
    if (i < n && k[i + 1] < (uint32_t)p.classes) w[i] = Row<T, VEC>::raw(dout + (int64_t)at[i] * p.dout_rs);
#pragma unroll
  for (int i = 0; i < PIECE; ++i) {
    if (i >= n) break;
    const uint32_t key = k[i + 1];
    if (key >= (uint32_t)p.classes) return;                    // these sort behind all others
    float v[VEC];
    Row<T, VEC>::open(w[i], v);
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] += v[j];
    const bool ends = k[i + 2] != key;
    if (!ends && i + 1 < n) continue;
    if (ends && !came_in) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] *= p.scale;
      Row<T, VEC>::store(dw + (int64_t)key * p.dweight_rs, acc);
    } else {
      float *o = (came_in ? head : tail) + (int64_t)blockIdx.x * p.features + c;
#pragma unroll
      for (int j = 0; j < VEC; ++j) o[j] = acc[j];
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    came_in = false;
  }
}

// The runs that cross borders: the piece where one begins adds up its parts, eight interleaved shares of them.
constexpr int JOIN_C = 128;                 // columns a block
template <typename T>
__global__ void __launch_bounds__(256) embed_join_kernel(const b200_embed_args p, const uint32_t *keys, const float *head, const float *tail, int pieces) {
  __shared__ float sh[8][JOIN_C];
  __shared__ int ends;
  const int piece = blockIdx.x;
  const int64_t last = (int64_t)piece * PIECE + PIECE - 1;              // of this piece
  if (last + 1 >= p.tokens) return;
  const uint32_t key = keys[last];
  if (key >= (uint32_t)p.classes || keys[last + 1] != key) return;      // nothing goes on
  const int64_t first = (int64_t)piece * PIECE;
  if (first > 0 && keys[first - 1] == key && keys[first] == key) return;      // it began earlier
  // the piece that the run ends in: the last whose entry border still has the key
  if (threadIdx.x == 0) {
    int lo = piece + 1, hi = pieces - 1;                                // keys are sorted
    if (lo < hi && keys[(int64_t)(lo + 1) * PIECE] != key) hi = lo;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (keys[(int64_t)mid * PIECE] == key) lo = mid;
      else hi = mid - 1;
    }
    ends = lo;
  }
  __syncthreads();
  const int to = ends, lane = threadIdx.x & 31, w = threadIdx.x >> 5, c0 = blockIdx.y * JOIN_C;
  float s[JOIN_C / 32];
#pragma unroll
  for (int j = 0; j < JOIN_C / 32; ++j) {
    const int c = c0 + j * 32 + lane;
    s[j] = w == 0 && c < p.features ? tail[(int64_t)piece * p.features + c] : 0.f;
  }
#pragma unroll 4
  for (int i = piece + 1 + w; i <= to; i += 8)
#pragma unroll
    for (int j = 0; j < JOIN_C / 32; ++j) {
      const int c = c0 + j * 32 + lane;
      if (c < p.features) s[j] += head[(int64_t)i * p.features + c];
    }
#pragma unroll
  for (int j = 0; j < JOIN_C / 32; ++j) sh[w][j * 32 + lane] = s[j];
  __syncthreads();
  const int c = c0 + threadIdx.x;
  if (threadIdx.x < JOIN_C && c < p.features) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) x += sh[i][threadIdx.x];
    reinterpret_cast<T *>(p.dweight)[(int64_t)key * p.dweight_rs + c] = T(x * p.scale);
  }
}

// ------------------------------------------------------------------------------------------------ host

int64_t up(int64_t n, int64_t unit) { return (n + unit - 1) / unit * unit; }

struct Sort { int passes, bits; int64_t pieces; };

Sort sort_of(const b200_embed_args &a) {
  Sort s;
  int width = 1;
  while ((int64_t(1) << width) <= a.classes) ++width;           // keys reach classes
  s.passes = (width + MAX_BITS - 1) / MAX_BITS;
  s.bits = (width + s.passes - 1) / s.passes;
  s.pieces = (a.tokens + PIECE - 1) / PIECE;
  return s;
}

int check_embed(const b200_embed_args &a, bool bwd) {
  B200_REQUIRE(a.ids && (bwd ? a.dout && a.dweight : a.weight && a.out), B200_ERR_NULL, "embed: null operand");
  B200_REQUIRE(a.tokens > 0 && a.classes > 0 && a.features > 0 && a.tokens < (int64_t(1) << 30) && a.classes < (1 << 30), B200_ERR_SHAPE,
               "embed: sizes must be positive and tokens below 2^30 (tokens %lld, classes %d, features %d)", (long long)a.tokens, a.classes, a.features);
  B200_REQUIRE(a.dtype == B200_F32 || a.dtype == B200_F16 || a.dtype == B200_BF16, B200_ERR_DTYPE, "embed: unknown dtype %d", a.dtype);
  return 0;
}

// The widest access, in elements, that rows of two tensors allow.
template <typename T> int widest(int features, const void *p, int64_t p_rs, const void *q, int64_t q_rs) {
  const uint64_t all = (uint64_t)features * sizeof(T) | reinterpret_cast<uintptr_t>(p) | (uint64_t)p_rs * sizeof(T) | reinterpret_cast<uintptr_t>(q) | (uint64_t)q_rs * sizeof(T);
  int bytes = 16;
  while (bytes > (int)sizeof(T) && all % bytes) bytes >>= 1;
  return bytes / (int)sizeof(T);
}
// f of that width as a constant
template <typename T, typename F> void with_width(int vec, F f) {
  if (vec == 1) f(std::integral_constant<int, 1>());
  else if (vec == 2) f(std::integral_constant<int, 2>());
  else if (vec == 4) f(std::integral_constant<int, 4>());
  else if constexpr (sizeof(T) == 2) f(std::integral_constant<int, 8>());
}

template <typename T> int run_fwd(const b200_embed_args &a, cudaStream_t st) {
  const int vec = widest<T>(a.features, a.weight, a.weight_rs, a.out, a.out_rs);
  const int parts = (a.features / vec + FWD_PER * 32 - 1) / (FWD_PER * 32);
  const int64_t blocks = (a.tokens * parts + 7) / 8, most = int64_t(1) << 20;
  with_width<T>(vec, [&](auto v) { embed_fwd_kernel<T, decltype(v)::value><<<(unsigned)(blocks < most ? blocks : most), 256, 0, st>>>(a, parts); });
  return launch_status();
}

template <typename T> int run_sums(const b200_embed_args &a, const Sort &s, const uint32_t *keys, const uint32_t *pos, float *head, float *tail, cudaStream_t st) {
  const int vec = widest<T>(a.features, a.dout, a.dout_rs, a.dweight, a.dweight_rs);
  const dim3 grid((unsigned)s.pieces, (unsigned)((a.features / vec + ROW_T - 1) / ROW_T));
  with_width<T>(vec, [&](auto v) { embed_sum_kernel<T, decltype(v)::value><<<grid, ROW_T, 0, st>>>(a, keys, pos, head, tail); });
  if (int e = launch_status()) return e;
  if (s.pieces > 1) embed_join_kernel<T><<<dim3((unsigned)s.pieces, (unsigned)((a.features + JOIN_C - 1) / JOIN_C)), 256, 0, st>>>(a, keys, head, tail, (int)s.pieces);
  return launch_status();
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_embed_fwd(const b200_embed_args *args, void *stream) {
  B200_REQUIRE(args, B200_ERR_NULL, "embed_fwd: null argument block");
  if (int e = check_embed(*args, false)) return e;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (args->dtype == B200_F32) return run_fwd<float>(*args, st);
  return args->dtype == B200_F16 ? run_fwd<__half>(*args, st) : run_fwd<__nv_bfloat16>(*args, st);
}

extern "C" int64_t b200_embed_bwd_work_bytes(const b200_embed_args *args) {
  if (!args || check_embed(*args, true)) return 0;
  const Sort s = sort_of(*args);
  return 4 * up(4 * args->tokens, 256) + 2 * up(4 * s.pieces * args->features, 256);
}

extern "C" int b200_embed_bwd(const b200_embed_args *args, void *stream) {
  B200_REQUIRE(args, B200_ERR_NULL, "embed_bwd: null argument block");
  const b200_embed_args &a = *args;
  if (int e = check_embed(a, true)) return e;
  B200_REQUIRE(a.work, B200_ERR_NULL, "embed_bwd: work must be non-null");
  B200_REQUIRE((reinterpret_cast<uintptr_t>(a.work) & 255) == 0, B200_ERR_ALIGN, "embed_bwd: work must be 256-byte aligned");
  B200_REQUIRE(a.work_bytes >= b200_embed_bwd_work_bytes(args), B200_ERR_TOO_LARGE, "embed_bwd: work has %lld bytes, %lld are needed", (long long)a.work_bytes,
               (long long)b200_embed_bwd_work_bytes(args));
  B200_REQUIRE(a.dweight_rs == a.features, B200_ERR_SHAPE, "embed_bwd: dweight must be dense");
  B200_REQUIRE((reinterpret_cast<uintptr_t>(a.dweight) & 15) == 0, B200_ERR_ALIGN, "embed_bwd: dweight must be 16-byte aligned");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const Sort s = sort_of(a);
  unsigned char *w = reinterpret_cast<unsigned char *>(a.work);
  const int64_t arr = up(4 * a.tokens, 256);
  SortArgs q;
  for (int i = 0; i < 2; ++i) {
    q.keys[i] = reinterpret_cast<uint32_t *>(w + i * arr);
    q.pos[i] = reinterpret_cast<uint32_t *>(w + (2 + i) * arr);
  }
  q.passes = s.passes;
  q.bits = s.bits;
  float *head = reinterpret_cast<float *>(w + 4 * arr);
  float *tail = head + up(4 * s.pieces * a.features, 256) / 4;
  const int smem = 4 * SORT_WARPS << s.bits, esz = act_size(a.dtype);
  cudaError_t ce = cudaFuncSetAttribute(embed_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (ce != cudaSuccess) { set_error("cudaFuncSetAttribute: %s", cudaGetErrorString(ce)); return (int)ce; }
  // a cluster to sort, and clusters that clear: about one a GPC's worth of SMs, fewer where there is little to clear
  int64_t clear = ((int64_t)a.classes * a.features * esz / 16 + SORT_T * CLUSTER - 1) / (SORT_T * CLUSTER), most = sm_count_current() / CLUSTER - 1;
  clear = clear < most ? clear : most;
  embed_sort_kernel<<<(unsigned)(CLUSTER * (1 + (clear > 0 ? clear : 1))), SORT_T, smem, st>>>(a, q, esz);
  if (int e = launch_status()) return e;
  const uint32_t *k = q.keys[(s.passes - 1) & 1], *at = q.pos[(s.passes - 1) & 1];
  if (a.dtype == B200_F32) return run_sums<float>(a, s, k, at, head, tail, st);
  return a.dtype == B200_F16 ? run_sums<__half>(a, s, k, at, head, tail, st) : run_sums<__nv_bfloat16>(a, s, k, at, head, tail, st);
}

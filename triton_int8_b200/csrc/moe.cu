// Tokens to their experts and back: a stable counting sort by expert with the rows copied in its order, the weighted sum of a
// token's rows, and the gradients of both.  Nothing here computes much: every kernel is bound by the bytes of the rows, or by
// launch latency for a few tokens.
//
// A token t has k choices ids[t, 0..k); choice i = t * k + j.  Expert e has c_e choices and the rows
// [offsets[e], offsets[e] + c_e) in the order of i, padded to offsets[e + 1], a multiple of `align` further on.  pos[i] is the row
// of a choice (-1: the id is no expert's), src its inverse (-1: a row of no choice, which is zero).
#include <cuda_fp16.h>

#include "common.cuh"

namespace i8l {
namespace {

constexpr int MAX_EXPERTS = 1024, MAX_CHOICES = 64;
constexpr int THREADS = 256;

// ------------------------------------------------------------------------------------------ types
// One access of a row: 16 bytes, or an element where rows or pointers are not 16-byte aligned.
template <typename T, bool WIDE> struct Piece;
template <typename T> struct Piece<T, true> { using type = uint4; static constexpr int N = 16 / sizeof(T); };
template <typename T> struct Piece<T, false> { using type = T; static constexpr int N = 1; };

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);   // round to nearest even, the one rounding of a result
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, bool WIDE>
__device__ __forceinline__ void unpack(const typename Piece<T, WIDE>::type& p, float* v) {
  const T* e = reinterpret_cast<const T*>(&p);
#pragma unroll
  for (int i = 0; i < Piece<T, WIDE>::N; ++i) v[i] = to_float(e[i]);
}
template <typename T, bool WIDE>
__device__ __forceinline__ typename Piece<T, WIDE>::type pack(const float* v) {
  typename Piece<T, WIDE>::type p;
  T* e = reinterpret_cast<T*>(&p);
#pragma unroll
  for (int i = 0; i < Piece<T, WIDE>::N; ++i) e[i] = from_float<T>(v[i]);
  return p;
}

__device__ __forceinline__ int64_t load_id(const void* ids, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
}
__device__ __forceinline__ int expert_of(const void* ids, int wide, int64_t i, int experts) {
  const int64_t e = load_id(ids, wide, i);
  return e >= 0 && e < experts ? (int)e : -1;
}
__device__ __forceinline__ int padded_to(int n, int align) { return (n + align - 1) / align * align; }

// ------------------------------------------------------------------------------------------ the sort
struct SortArgs {
  const void* x;
  const void* ids;
  void* rows;
  int32_t *offsets, *pos, *src;
  int32_t* hist;        // [blocks, experts]: choices of each expert in each chunk
  int64_t tokens, pieces;   // pieces of a row
  int n, k, experts, align, n_rows, ids64;
  int chunk, blocks;    // choices of a block in the counting and placing kernels
  int lanes;            // threads of a token in the copying kernels, a power of two
};

// Exclusive scan of the padded counts into offsets[0 .. experts], by the first warp.
__device__ __forceinline__ void scan_offsets(const int* count, int* offsets, int experts, int align) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int carry = 0;
    for (int e0 = 0; e0 < experts; e0 += 32) {
      const int mine = e0 + lane < experts ? padded_to(count[e0 + lane], align) : 0;
      int up = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, up, d);
        if (lane >= d) up += v;
      }
      if (e0 + lane < experts) offsets[e0 + lane] = carry + up - mine;
      carry += __shfl_sync(0xffffffffu, up, 31);
    }
    if (lane == 0) offsets[experts] = carry;
  }
}

// Copies the row of token t to the rows of its choices, `lanes` threads a token.
template <typename P>
__device__ __forceinline__ void copy_row(const SortArgs& a, int64_t t, int l, const int32_t* pos) {
  const P* from = static_cast<const P*>(a.x) + t * a.pieces;
  for (int64_t c0 = l; c0 < a.pieces; c0 += 4 * a.lanes) {
    P v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (c0 + u * a.lanes < a.pieces) v[u] = from[c0 + u * a.lanes];
    for (int j = 0; j < a.k; ++j) {
      const int r = pos[j];
      if (r < 0) continue;
      P* to = static_cast<P*>(a.rows) + (int64_t)r * a.pieces;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (c0 + u * a.lanes < a.pieces) to[c0 + u * a.lanes] = v[u];
    }
  }
}
template <typename P>
__device__ __forceinline__ void clear_row(void* rows, int64_t pieces, int64_t r, int lane) {
  P zero;
  memset(&zero, 0, sizeof(P));
  P* to = static_cast<P*>(rows) + r * pieces;
  for (int64_t c = lane; c < pieces; c += 32) to[c] = zero;
}

// Few choices: one launch.  Every block counts all of them for itself (they fit its shared memory) and copies the rows of its
// tokens; the rows of no choice are spread over all warps.
constexpr int SMALL_SORT = 1024;
template <typename P>
__global__ void __launch_bounds__(THREADS) sort_small_kernel(const SortArgs a) {
  __shared__ int16_t expert[SMALL_SORT];
  __shared__ int count[MAX_EXPERTS], offsets[MAX_EXPERTS + 1];
  __shared__ int32_t pos[THREADS / 32][MAX_CHOICES];   // of the block's tokens: at most one a warp
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int e = tid; e < a.experts; e += THREADS) count[e] = 0;
  __syncthreads();
  for (int i = tid; i < a.n; i += THREADS) {
    const int e = expert_of(a.ids, a.ids64, i, a.experts);
    expert[i] = (int16_t)e;
    if (e >= 0) atomicAdd(&count[e], 1);   // integers: the order of the additions does not show
  }
  __syncthreads();
  scan_offsets(count, offsets, a.experts, a.align);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = tid; e <= a.experts; e += THREADS) a.offsets[e] = offsets[e];
  // The row of a choice: its expert's first one, and the choices of that expert in front of it.
  const int per_block = THREADS / a.lanes;
  const int64_t t0 = (int64_t)blockIdx.x * per_block;
  for (int w = warp; w < per_block * a.k; w += THREADS / 32) {
    const int64_t t = t0 + w / a.k;
    if (t >= a.tokens) break;
    const int i = (int)t * a.k + w % a.k, e = expert[i];
    int before = 0;
    if (e >= 0)
      for (int q = lane; q < i; q += 32) before += expert[q] == e;
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0) {
      const int r = e < 0 ? -1 : offsets[e] + before;
      pos[w / a.k][w % a.k] = r;
      a.pos[i] = r;
      if (r >= 0) a.src[r] = i;
    }
  }
  __syncthreads();
  const int64_t t = t0 + tid / a.lanes;
  if (t < a.tokens) copy_row<P>(a, t, tid & (a.lanes - 1), pos[tid / a.lanes]);
  for (int64_t r = (int64_t)blockIdx.x * (THREADS / 32) + warp; r < a.n_rows; r += (int64_t)gridDim.x * (THREADS / 32)) {
    int lo = 0, hi = a.experts;   // the expert whose rows r is among: offsets[lo] <= r < offsets[hi], or lo = experts
    if (r >= offsets[a.experts]) lo = a.experts;
    else
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (offsets[mid] <= r) lo = mid;
        else hi = mid;
      }
    if (lo < a.experts && r - offsets[lo] < count[lo]) continue;
    if (lane == 0) a.src[r] = -1;
    clear_row<P>(a.rows, a.pieces, r, lane);
  }
}

// Many choices: count them per chunk, place them, copy the rows.  The chunk of a block is split into runs of its warps; a warp
// goes through its run 32 choices at a time, equal ones found with match.any, so that places follow the order of the choices.
__global__ void __launch_bounds__(THREADS) sort_count_kernel(const SortArgs a) {
  __shared__ int count[MAX_EXPERTS];
  chain_wait();
  chain_trigger();
  for (int e = threadIdx.x; e < a.experts; e += THREADS) count[e] = 0;
  __syncthreads();
  const int first = blockIdx.x * a.chunk, last = min(first + a.chunk, a.n);
  for (int i = first + threadIdx.x; i < last; i += THREADS) {
    const int e = expert_of(a.ids, a.ids64, i, a.experts);
    if (e >= 0) atomicAdd(&count[e], 1);
  }
  for (int64_t r = (int64_t)blockIdx.x * THREADS + threadIdx.x; r < a.n_rows; r += (int64_t)gridDim.x * THREADS) a.src[r] = -1;   // until it is placed
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += THREADS) a.hist[(int64_t)blockIdx.x * a.experts + e] = count[e];
}

__global__ void __launch_bounds__(THREADS) sort_place_kernel(const SortArgs a) {
  __shared__ int total[MAX_EXPERTS], before[MAX_EXPERTS], offsets[MAX_EXPERTS + 1];
  extern __shared__ int next[];   // [warps, experts]: the row of a warp's next choice of an expert
  constexpr int WARPS = THREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int e = tid; e < a.experts; e += THREADS) total[e] = before[e] = 0;
  for (int e = tid; e < WARPS * a.experts; e += THREADS) next[e] = 0;
  chain_wait();
  chain_trigger();
  __syncthreads();
  for (int i = tid; i < a.blocks * a.experts; i += THREADS) {
    const int b = i / a.experts, e = i - b * a.experts, c = a.hist[i];
    if (c) {
      atomicAdd(&total[e], c);
      if (b < (int)blockIdx.x) atomicAdd(&before[e], c);
    }
  }
  const int run = (a.chunk + WARPS - 1) / WARPS;
  const int end = min((int)(blockIdx.x + 1) * a.chunk, a.n), first = min((int)blockIdx.x * a.chunk + warp * run, end), last = min(first + run, end);
  int* mine = next + warp * a.experts;
  for (int i0 = first; i0 < last; i0 += 32) {
    const int e = i0 + lane < last ? expert_of(a.ids, a.ids64, i0 + lane, a.experts) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  scan_offsets(total, offsets, a.experts, a.align);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = tid; e <= a.experts; e += THREADS) a.offsets[e] = offsets[e];
  for (int e = tid; e < a.experts; e += THREADS) {
    int at = offsets[e] + before[e];
    for (int w = 0; w < WARPS; ++w) {
      const int c = next[w * a.experts + e];
      next[w * a.experts + e] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int i0 = first; i0 < last; i0 += 32) {
    const int i = i0 + lane, e = i < last ? expert_of(a.ids, a.ids64, i, a.experts) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int r = e >= 0 ? mine[e] + __popc(same & ((1u << lane) - 1)) : -1;
    __syncwarp();
    if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
    if (i < last) {
      a.pos[i] = r;
      if (r >= 0) a.src[r] = i;
    }
    __syncwarp();
  }
}

template <typename P>
__global__ void __launch_bounds__(THREADS) sort_copy_kernel(const SortArgs a) {
  chain_wait();
  const int64_t t = (int64_t)blockIdx.x * (THREADS / a.lanes) + threadIdx.x / a.lanes;
  if (t < a.tokens) copy_row<P>(a, t, threadIdx.x & (a.lanes - 1), a.pos + t * a.k);
  const int lane = threadIdx.x & 31;
  for (int64_t r = (int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5); r < a.n_rows; r += (int64_t)gridDim.x * (THREADS / 32))
    if (a.src[r] < 0) clear_row<P>(a.rows, a.pieces, r, lane);
}

// ------------------------------------------------------------------------------------------ the way back
struct CombineArgs {
  const void *rows, *weights;   // weights null: ones
  const int32_t *pos, *src;
  const void* dy;
  void *y, *drows, *dweights;
  int64_t tokens, pieces, n_rows;
  int k, lanes;
};

template <typename W> __device__ __forceinline__ float weight_of(const void* w, int64_t i) { return w ? to_float(static_cast<const W*>(w)[i]) : 1.f; }
// The row of a choice, or -1; what is out of range counts as dropped, so that no access leaves the rows.
__device__ __forceinline__ int row_of(const CombineArgs& a, int64_t i) {
  const int r = a.pos[i];
  return r >= 0 && r < a.n_rows ? r : -1;
}

// y[t] = sum over j of w[t, j] * rows[pos[t, j]], in the order of j, in 32 bits and rounded once.  Choices four at a time, so that
// their loads are in flight together.
template <typename T, typename W, bool WIDE>
__global__ void __launch_bounds__(THREADS) combine_kernel(const CombineArgs a) {
  using P = typename Piece<T, WIDE>::type;
  constexpr int N = Piece<T, WIDE>::N;
  const int64_t t = (int64_t)blockIdx.x * (THREADS / a.lanes) + threadIdx.x / a.lanes;
  if (t >= a.tokens) return;
  for (int64_t c = threadIdx.x & (a.lanes - 1); c < a.pieces; c += a.lanes) {
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    for (int j0 = 0; j0 < a.k; j0 += 4) {
      P v[4];
      float w[4];
      int r[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) r[u] = j0 + u < a.k ? row_of(a, t * a.k + j0 + u) : -1;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (r[u] >= 0) {
          v[u] = static_cast<const P*>(a.rows)[(int64_t)r[u] * a.pieces + c];
          w[u] = weight_of<W>(a.weights, t * a.k + j0 + u);
        }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (r[u] >= 0) {
          float f[N];
          unpack<T, WIDE>(v[u], f);
#pragma unroll
          for (int i = 0; i < N; ++i) acc[i] = fmaf(w[u], f[i], acc[i]);
        }
    }
    static_cast<P*>(a.y)[t * a.pieces + c] = pack<T, WIDE>(acc);
  }
}

// drows[pos[t, j]] = w[t, j] * dy[t], rows of no choice zero; dw[t, j] = the sum of dy[t] * rows[pos[t, j]], added in an order that
// depends on the sizes only.  A row is written by the choice that src names, so that rows are written once whatever pos holds.
template <typename T, typename W, bool WIDE>
__global__ void __launch_bounds__(THREADS) combine_backward_kernel(const CombineArgs a) {
  using P = typename Piece<T, WIDE>::type;
  constexpr int N = Piece<T, WIDE>::N;
  __shared__ float part[THREADS / 32][MAX_CHOICES];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * (THREADS / a.lanes) + threadIdx.x / a.lanes;
  if (t < a.tokens) {   // the same for all threads of a warp
    const P* dy = static_cast<const P*>(a.dy) + t * a.pieces;
    for (int j = 0; j < a.k; ++j) {
      const int64_t i = t * a.k + j;
      const int r = row_of(a, i);
      float dot = 0.f;
      if (r >= 0) {
        const float w = weight_of<W>(a.weights, i);
        const bool owner = a.drows && a.src[r] == (int32_t)i;
        const P* row = static_cast<const P*>(a.rows) + (int64_t)r * a.pieces;
        P* drow = static_cast<P*>(a.drows) + (int64_t)r * a.pieces;
        for (int64_t c = threadIdx.x & (a.lanes - 1); c < a.pieces; c += a.lanes) {
          float g[N], f[N];
          unpack<T, WIDE>(dy[c], g);
          if (a.dweights) {
            unpack<T, WIDE>(row[c], f);
#pragma unroll
            for (int q = 0; q < N; ++q) dot = fmaf(g[q], f[q], dot);
          }
          if (owner) {
#pragma unroll
            for (int q = 0; q < N; ++q) g[q] *= w;
            drow[c] = pack<T, WIDE>(g);
          }
        }
      }
      if (a.dweights) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (lane == 0) part[warp][j] = dot;
      }
    }
  }
  if (a.dweights) {
    __syncthreads();
    const int warps = a.lanes / 32, per_block = THREADS / a.lanes;
    for (int q = threadIdx.x; q < per_block * a.k; q += THREADS) {
      const int g = q / a.k, j = q - g * a.k;
      const int64_t at = (int64_t)blockIdx.x * per_block + g;
      if (at >= a.tokens) break;
      float sum = 0.f;
      for (int w = 0; w < warps; ++w) sum += part[g * warps + w][j];
      static_cast<W*>(a.dweights)[at * a.k + j] = from_float<W>(sum);
    }
  }
  if (a.drows)
    for (int64_t r = (int64_t)blockIdx.x * (THREADS / 32) + warp; r < a.n_rows; r += (int64_t)gridDim.x * (THREADS / 32))
      if (a.src[r] < 0) clear_row<P>(a.drows, a.pieces, r, lane);
}

// ------------------------------------------------------------------------------------------ host
// Threads of a token: a warp's worth at least (dot products are added up within warps), at most the block, four pieces each in between.
int lanes_for(int64_t pieces) {
  int lanes = 32;
  while (lanes < THREADS && lanes * 4 < pieces) lanes *= 2;
  return lanes;
}
int elem_size(int dtype) { return dtype == I8L_DTYPE_F32 ? 4 : 2; }

int check_rows(const char* name, int64_t tokens, int64_t cols, int64_t rows, int k, int dtype, int wdtype = I8L_DTYPE_F32) {
  if (dtype != I8L_DTYPE_BF16 && dtype != I8L_DTYPE_F16 && dtype != I8L_DTYPE_F32) return fail(I8L_ERR_ARG, "%s: unknown dtype %d", name, dtype);
  if (wdtype != I8L_DTYPE_F32 && wdtype != dtype) return fail(I8L_ERR_ARG, "%s: weights are fp32 or of the rows' type", name);
  if (k < 1 || k > MAX_CHOICES) return fail(I8L_ERR_SHAPE, "%s: %d choices a token, 1 to %d are possible", name, k, MAX_CHOICES);
  if (tokens < 0 || cols < 1 || rows < 0 || tokens > (1ll << 30) / k || rows >= (1ll << 31) || cols >= (1ll << 31))
    return fail(I8L_ERR_SHAPE, "%s: tokens=%lld cols=%lld rows=%lld out of range", name, (long long)tokens, (long long)cols, (long long)rows);
  return I8L_OK;
}
bool aligned_to(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <typename T, typename W>
int launch_combine(CombineArgs a, bool backward, bool wide, cudaStream_t st) {
  const unsigned grid = (unsigned)((a.tokens + THREADS / a.lanes - 1) / (THREADS / a.lanes));
  if (backward) {
    const unsigned blocks = grid ? grid : 1;   // without tokens there still are rows to clear
    if (wide) combine_backward_kernel<T, W, true><<<blocks, THREADS, 0, st>>>(a);
    else combine_backward_kernel<T, W, false><<<blocks, THREADS, 0, st>>>(a);
  } else {
    if (wide) combine_kernel<T, W, true><<<grid, THREADS, 0, st>>>(a);
    else combine_kernel<T, W, false><<<grid, THREADS, 0, st>>>(a);
  }
  I8L_CUDA_OK(cudaGetLastError());
  return I8L_OK;
}
template <typename T>
int launch_combine(const CombineArgs& a, int wdtype, int dtype, bool backward, bool wide, cudaStream_t st) {
  return wdtype == I8L_DTYPE_F32 ? launch_combine<T, float>(a, backward, wide, st) : launch_combine<T, T>(a, backward, wide, st);
}
int run_combine(CombineArgs a, int64_t cols, int dtype, int wdtype, bool backward, bool wide, cudaStream_t st) {
  a.pieces = wide ? cols * elem_size(dtype) / 16 : cols;
  a.lanes = lanes_for(a.pieces);
  if (dtype == I8L_DTYPE_F32) return launch_combine<float, float>(a, backward, wide, st);
  if (dtype == I8L_DTYPE_F16) return launch_combine<__half>(a, wdtype, dtype, backward, wide, st);
  return launch_combine<__nv_bfloat16>(a, wdtype, dtype, backward, wide, st);
}

}  // namespace
}  // namespace i8l

using namespace i8l;

extern "C" int64_t i8l_sort_workspace(int64_t tokens, int k, int experts) {
  if (tokens < 0 || k < 1 || experts < 1 || tokens * k <= SMALL_SORT) return 0;
  const int64_t chunk = experts * 4 > 1024 ? experts * 4 : 1024;
  return (tokens * k + chunk - 1) / chunk * experts * (int64_t)sizeof(int32_t);
}

extern "C" int i8l_sort_tokens(const void* x, const void* ids, int ids64, int64_t tokens, int64_t cols, int k, int experts, int64_t align,
                               int dtype, int64_t rows, void* out, int32_t* offsets, int32_t* pos, int32_t* src, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  if (int e = check_rows("i8l_sort_tokens", tokens, cols, rows, k, dtype)) return e;
  if (experts < 1 || experts > MAX_EXPERTS) return fail(I8L_ERR_SHAPE, "i8l_sort_tokens: %d experts, 1 to %d are possible", experts, MAX_EXPERTS);
  const int64_t n = tokens * k;
  if (align < 1 || align > 65536) return fail(I8L_ERR_SHAPE, "i8l_sort_tokens: align=%lld, 1 to 65536 are possible", (long long)align);
  const int64_t need = (n + (experts < n ? experts : n) * (align - 1) + align - 1) / align * align;
  if (rows < need) return fail(I8L_ERR_SHAPE, "i8l_sort_tokens: %lld rows, %lld are needed", (long long)rows, (long long)need);
  if (!offsets || (tokens && (!x || !ids || !pos)) || (rows && (!out || !src))) return fail(I8L_ERR_ARG, "i8l_sort_tokens: null pointer");
  const int size = elem_size(dtype);
  if (!aligned_to(x, size) || !aligned_to(out, size) || !aligned_to(ids, ids64 ? 8 : 4))
    return fail(I8L_ERR_ALIGN, "i8l_sort_tokens: pointers are aligned to their elements");
  if (workspace_bytes < i8l_sort_workspace(tokens, k, experts) || (i8l_sort_workspace(tokens, k, experts) && !workspace))
    return fail(I8L_ERR_ARG, "i8l_sort_tokens: workspace of %lld bytes is too small", (long long)workspace_bytes);
  if (int e = check_arch()) return e;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = cols * size % 16 == 0 && aligned16(x) && aligned16(out);
  SortArgs a{};
  a.x = x; a.ids = ids; a.rows = out; a.offsets = offsets; a.pos = pos; a.src = src;
  a.hist = static_cast<int32_t*>(workspace);
  a.tokens = tokens; a.pieces = wide ? cols * size / 16 : cols;
  a.n = (int)n; a.k = k; a.experts = experts; a.align = (int)align; a.n_rows = (int)rows; a.ids64 = ids64 ? 1 : 0;
  a.lanes = lanes_for(a.pieces);
  const unsigned copies = (unsigned)((tokens + THREADS / a.lanes - 1) / (THREADS / a.lanes));
  const unsigned grid = copies ? copies : 1;
  if (n <= SMALL_SORT) {
    if (wide) sort_small_kernel<uint4><<<grid, THREADS, 0, st>>>(a);
    else if (size == 4) sort_small_kernel<uint32_t><<<grid, THREADS, 0, st>>>(a);
    else sort_small_kernel<uint16_t><<<grid, THREADS, 0, st>>>(a);
    I8L_CUDA_OK(cudaGetLastError());
    return I8L_OK;
  }
  a.chunk = experts * 4 > 1024 ? experts * 4 : 1024;
  a.blocks = (int)((n + a.chunk - 1) / a.chunk);
  const LaunchChain chain(st);
  (void)chain_first();
  I8L_CUDA_OK(launch(sort_count_kernel, dim3(a.blocks), THREADS, 0, st, a));
  I8L_CUDA_OK(launch(sort_place_kernel, dim3(a.blocks), THREADS, THREADS / 32 * experts * sizeof(int), st, a));
  I8L_CUDA_OK(wide        ? launch(sort_copy_kernel<uint4>, dim3(grid), THREADS, 0, st, a)
              : size == 4 ? launch(sort_copy_kernel<uint32_t>, dim3(grid), THREADS, 0, st, a)
                          : launch(sort_copy_kernel<uint16_t>, dim3(grid), THREADS, 0, st, a));
  return I8L_OK;
}

extern "C" int i8l_combine(const void* rows, const void* weights, const int32_t* pos, int64_t n_rows, int64_t tokens, int64_t cols, int k,
                           int dtype, int wdtype, void* y, void* stream) {
  if (int e = check_rows("i8l_combine", tokens, cols, n_rows, k, dtype, wdtype)) return e;
  if (!tokens) return I8L_OK;
  if (!pos || !y || (n_rows && !rows)) return fail(I8L_ERR_ARG, "i8l_combine: null pointer");
  const int size = elem_size(dtype);
  if (!aligned_to(rows, size) || !aligned_to(y, size) || !aligned_to(weights, wdtype == I8L_DTYPE_F32 ? 4 : 2) || !aligned_to(pos, 4))
    return fail(I8L_ERR_ALIGN, "i8l_combine: pointers are aligned to their elements");
  if (int e = check_arch()) return e;
  CombineArgs a{};
  a.rows = rows; a.weights = weights; a.pos = pos; a.y = y;
  a.tokens = tokens; a.n_rows = n_rows; a.k = k;
  const bool wide = cols * size % 16 == 0 && aligned16(rows) && aligned16(y);
  return run_combine(a, cols, dtype, wdtype, false, wide, static_cast<cudaStream_t>(stream));
}

extern "C" int i8l_combine_backward(const void* rows, const void* weights, const int32_t* pos, const int32_t* src, const void* dy,
                                    int64_t n_rows, int64_t tokens, int64_t cols, int k, int dtype, int wdtype, void* drows, void* dweights,
                                    void* stream) {
  if (int e = check_rows("i8l_combine_backward", tokens, cols, n_rows, k, dtype, wdtype)) return e;
  if ((!tokens || !dweights) && (!n_rows || !drows)) return I8L_OK;
  if ((tokens && (!pos || !dy || !weights)) || (n_rows && (!rows || (drows && !src)))) return fail(I8L_ERR_ARG, "i8l_combine_backward: null pointer");
  const int size = elem_size(dtype);
  const int wsize = wdtype == I8L_DTYPE_F32 ? 4 : 2;
  if (!aligned_to(rows, size) || !aligned_to(dy, size) || !aligned_to(drows, size) || !aligned_to(weights, wsize) || !aligned_to(dweights, wsize))
    return fail(I8L_ERR_ALIGN, "i8l_combine_backward: pointers are aligned to their elements");
  if (int e = check_arch()) return e;
  CombineArgs a{};
  a.rows = rows; a.weights = weights; a.pos = pos; a.src = src; a.dy = dy; a.drows = drows; a.dweights = dweights;
  a.tokens = tokens; a.n_rows = n_rows; a.k = k;
  const bool wide = cols * size % 16 == 0 && aligned16(rows) && aligned16(dy) && aligned16(drows);
  return run_combine(a, cols, dtype, wdtype, true, wide, static_cast<cudaStream_t>(stream));
}

// Tokens to their experts and back: a stable counting sort by expert with the rows copied in its order, the weighted sum of a
// token's rows, and the gradients of both.  Nothing here computes much: every kernel is bound by the bytes of the rows, or by
// launch latency for a few tokens.
//
// A token t has k choices ids[t, 0..k); choice i = t * k + j.  Expert e has c_e choices and the rows
// [offsets[e], offsets[e] + c_e) in the order of i, padded to offsets[e + 1], a multiple of `align` further on.  pos[i] is the row
// of a choice (-1: the id is no expert's), src its inverse (-1: a row of no choice, which is zero).
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"

namespace i8l {
namespace {

constexpr int MAX_EXPERTS = 1024, MAX_CHOICES = 64;
constexpr int THREADS = 256, MIN_LANES = 8;   // of a block; of a token

// ------------------------------------------------------------------------------------------ rows, 16 bytes at a time
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);   // round to nearest even, the one rounding of a result
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T> constexpr int PER_PIECE = 16 / sizeof(T);
template <typename T> __device__ __forceinline__ void unpack(const uint4& p, float* v) {
  const T* e = reinterpret_cast<const T*>(&p);
#pragma unroll
  for (int i = 0; i < PER_PIECE<T>; ++i) v[i] = to_float(e[i]);
}
template <typename T> __device__ __forceinline__ uint4 pack(const float* v) {
  uint4 p;
  T* e = reinterpret_cast<T*>(&p);
#pragma unroll
  for (int i = 0; i < PER_PIECE<T>; ++i) e[i] = from_float<T>(v[i]);
  return p;
}

// Rows that are no multiple of 16 bytes, or do not start on one ("odd"), still move 16 bytes at a time: whole aligned pieces of the row
// that is written, each put together from the two aligned pieces that it lies across in the row that is read, and the elements at
// the ends one by one.  Both of those pieces hold bytes of the piece that is wanted, so nothing is read that the row has no part in
// (memory comes in whole ones).
struct Cut {          // of a row that is written
  int head, pieces;   // bytes in front of its whole pieces, their number
};
__device__ __forceinline__ Cut cut_of(const void* row, int bytes) {
  const int head = (int)(-reinterpret_cast<uintptr_t>(row) & 15);
  return head < bytes ? Cut{head, (bytes - head) / 16} : Cut{bytes, 0};
}
// Element i of those at the ends, or a negative number: their bytes in the row.
template <typename T> __device__ __forceinline__ int end_element(const Cut& c, int bytes, int i) {
  const int heads = c.head / (int)sizeof(T);
  const int at = i < heads ? i * (int)sizeof(T) : c.head + 16 * c.pieces + (i - heads) * (int)sizeof(T);
  return at < bytes ? at : -1;
}
template <typename T> constexpr int MOST_ENDS = 2 * (PER_PIECE<T> - 1);   // elements at both ends
struct Across {       // a row that is read at the pieces of another one
  const uint4* piece;   // the aligned one in which the first wanted piece begins
  int off;              // where in it
};
__device__ __forceinline__ Across across(const char* row, const Cut& c) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(row + c.head);
  return Across{reinterpret_cast<const uint4*>(p & ~(uintptr_t)15), (int)(p & 15)};
}
struct Pair {
  uint4 lo, hi;
};
__device__ __forceinline__ Pair load_pair(const Across& r, int q) {
  Pair v;
  v.lo = r.piece[q];
  if (r.off) v.hi = r.piece[q + 1];
  return v;
}
// off is the same for a whole row: the branches are uniform.
__device__ __forceinline__ uint4 joined(const Pair& v, int off) {
  const int bits = (off & 3) * 8;
  const uint4 &a = v.lo, &b = v.hi;
  if (!off) return a;
  switch (off >> 2) {
    case 0: return make_uint4(__funnelshift_r(a.x, a.y, bits), __funnelshift_r(a.y, a.z, bits), __funnelshift_r(a.z, a.w, bits), __funnelshift_r(a.w, b.x, bits));
    case 1: return make_uint4(__funnelshift_r(a.y, a.z, bits), __funnelshift_r(a.z, a.w, bits), __funnelshift_r(a.w, b.x, bits), __funnelshift_r(b.x, b.y, bits));
    case 2: return make_uint4(__funnelshift_r(a.z, a.w, bits), __funnelshift_r(a.w, b.x, bits), __funnelshift_r(b.x, b.y, bits), __funnelshift_r(b.y, b.z, bits));
    default: return make_uint4(__funnelshift_r(a.w, b.x, bits), __funnelshift_r(b.x, b.y, bits), __funnelshift_r(b.y, b.z, bits), __funnelshift_r(b.z, b.w, bits));
  }
}
// An odd row, from another one or from nothing, by threads l, l + lanes, ...
template <typename T> __device__ __forceinline__ void copy_odd(char* to, const char* from, int bytes, int l, int lanes) {
  const Cut c = cut_of(to, bytes);
  for (int i = l; i < MOST_ENDS<T>; i += lanes) {
    const int at = end_element<T>(c, bytes, i);
    if (at >= 0) *reinterpret_cast<T*>(to + at) = from ? *reinterpret_cast<const T*>(from + at) : T{};
  }
  uint4* out = reinterpret_cast<uint4*>(to + c.head);
  if (!from) {
    for (int q = l; q < c.pieces; q += lanes) out[q] = make_uint4(0, 0, 0, 0);
    return;
  }
  const Across r = across(from, c);
  for (int q = l; q < c.pieces; q += lanes) out[q] = joined(load_pair(r, q), r.off);
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
  int64_t tokens;
  int bytes;   // of a row
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

// Copies the row of token t to the rows of its choices, `lanes` threads a token, four pieces in flight each.
template <typename T, bool ODD>
__device__ __forceinline__ void copy_row(const SortArgs& a, int64_t t, int l, const int32_t* pos) {
  constexpr int U = 4;
  const char* from = static_cast<const char*>(a.x) + t * a.bytes;
  char* const rows = static_cast<char*>(a.rows);
  if (ODD) {
    for (int j = 0; j < a.k; ++j)
      if (pos[j] >= 0) copy_odd<T>(rows + (int64_t)pos[j] * a.bytes, from, a.bytes, l, a.lanes);
    return;
  }
  const int pieces = a.bytes / 16;
  for (int c0 = l; c0 < pieces; c0 += U * a.lanes) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * a.lanes < pieces) v[u] = reinterpret_cast<const uint4*>(from)[c0 + u * a.lanes];
    for (int j = 0; j < a.k; ++j) {
      const int r = pos[j];
      if (r < 0) continue;
      uint4* to = reinterpret_cast<uint4*>(rows + (int64_t)r * a.bytes);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + u * a.lanes < pieces) to[c0 + u * a.lanes] = v[u];
    }
  }
}

// Few choices: one launch.  Every block counts all of them for itself (they fit its shared memory) and copies the rows of its
// tokens; the rows of no choice are spread over all warps.
constexpr int SMALL_SORT = 1024;
template <typename T, bool ODD>
__global__ void __launch_bounds__(THREADS) sort_small_kernel(const SortArgs a) {
  __shared__ int16_t expert[SMALL_SORT];
  __shared__ int count[MAX_EXPERTS], offsets[MAX_EXPERTS + 1];
  __shared__ int32_t pos[THREADS / MIN_LANES][MAX_CHOICES];   // of the block's tokens
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int e = tid; e < a.experts; e += THREADS) count[e] = 0;
  __syncthreads();
  for (int i = tid; i < a.n; i += THREADS) {
    const int e = expert_of(a.ids, a.ids64, i, a.experts);
    expert[i] = (int16_t)e;
    if (e >= 0) atomicAdd(&count[e], 1);
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
  if (t < a.tokens) copy_row<T, ODD>(a, t, tid & (a.lanes - 1), pos[tid / a.lanes]);
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
    copy_odd<T>(static_cast<char*>(a.rows) + r * a.bytes, nullptr, a.bytes, lane, 32);
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
  // All blocks' counts added up: a thread takes every `stride`th block's of one expert, so that its loads are in flight together.
  int wide = 32;
  while (wide < a.experts && wide < THREADS) wide *= 2;
  const int stride = THREADS / wide;
  for (int e = tid & (wide - 1); e < a.experts; e += wide) {
    int all = 0, front = 0;
#pragma unroll 4
    for (int b = tid / wide; b < a.blocks; b += stride) {
      const int c = a.hist[(int64_t)b * a.experts + e];
      all += c;
      front += b < (int)blockIdx.x ? c : 0;
    }
    if (all) atomicAdd(&total[e], all);   // integers: the order of the additions does not show
    if (front) atomicAdd(&before[e], front);
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

// A token's row is read once and written to each of its places.
__global__ void __launch_bounds__(THREADS) sort_copy_kernel(const SortArgs a) {
  chain_wait();
  const int64_t t = (int64_t)blockIdx.x * (THREADS / a.lanes) + threadIdx.x / a.lanes;
  if (t < a.tokens) copy_row<uint32_t, false>(a, t, threadIdx.x & (a.lanes - 1), a.pos + t * a.k);
  const int lane = threadIdx.x & 31;
  for (int64_t r = (int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5); r < a.n_rows; r += (int64_t)gridDim.x * (THREADS / 32))
    if (a.src[r] < 0) copy_odd<uint32_t>(static_cast<char*>(a.rows) + r * a.bytes, nullptr, a.bytes, lane, 32);
}
// Odd rows are put together for each place anyway: row by row, those of no choice among them, all of them alike much work.  Blocks go
// on to further rows and know where from before they get there, and there are many of them: 13554 x 780 fp16 with 6 choices 53 us (four
// pieces a lane and half the blocks 60).
template <typename T>
__global__ void __launch_bounds__(THREADS, 8) sort_copy_odd_kernel(const SortArgs a) {
  chain_wait();
  const int64_t step = (int64_t)gridDim.x * (THREADS / a.lanes);
  int64_t r = (int64_t)blockIdx.x * (THREADS / a.lanes) + threadIdx.x / a.lanes;
  int i = r < a.n_rows ? a.src[r] : -1;
  for (; r < a.n_rows; r += step) {
    const int next = r + step < a.n_rows ? a.src[r + step] : -1;
    copy_odd<T>(static_cast<char*>(a.rows) + r * a.bytes, i < 0 ? nullptr : static_cast<const char*>(a.x) + (int64_t)(i / a.k) * a.bytes, a.bytes,
                threadIdx.x & (a.lanes - 1), a.lanes);
    i = next;
  }
}

// ------------------------------------------------------------------------------------------ the way back
struct CombineArgs {
  const void *rows, *weights;   // weights null: ones
  const int32_t *pos, *src;
  const void* dy;
  void *y, *drows, *dweights;
  int64_t tokens, n_rows;
  int bytes, k, lanes;   // bytes of a row
};

template <typename W> __device__ __forceinline__ float weight_of(const void* w, int64_t i) { return w ? to_float(static_cast<const W*>(w)[i]) : 1.f; }
// The row of a choice, or -1; what is out of range counts as dropped, so that no access leaves the rows.
__device__ __forceinline__ int row_of(const CombineArgs& a, int64_t i) {
  const int r = a.pos[i];
  return r >= 0 && r < a.n_rows ? r : -1;
}
__device__ __forceinline__ const char* row_at(const void* rows, int64_t r, int bytes) { return static_cast<const char*>(rows) + r * bytes; }
__device__ __forceinline__ char* row_at(void* rows, int64_t r, int bytes) { return static_cast<char*>(rows) + r * bytes; }

// y[t] = sum over j of w[t, j] * rows[pos[t, j]], in the order of j, in 32 bits and rounded once.  J choices at a time and U
// pieces of their rows, so that J * U loads are in flight together; odd rows, of which a piece is two loads and more registers, one at a
// time in more warps (9460 x 658 bf16 with 8 choices 37 us, two choices at a time 48).
template <typename T, typename W, bool ODD, int J, int U>
__global__ void __launch_bounds__(THREADS, ODD ? 6 : 1) combine_kernel(const CombineArgs a) {
  constexpr int N = PER_PIECE<T>;
  const int64_t t = (int64_t)blockIdx.x * (THREADS / a.lanes) + threadIdx.x / a.lanes;
  const int l = threadIdx.x & (a.lanes - 1);
  if (t >= a.tokens) return;
  char* y = row_at(a.y, t, a.bytes);
  const Cut cut = ODD ? cut_of(y, a.bytes) : Cut{0, a.bytes / 16};
  uint4* out = reinterpret_cast<uint4*>(y + cut.head);
  for (int q0 = l; q0 < cut.pieces; q0 += U * a.lanes) {
    float acc[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) acc[u][i] = 0.f;
    int later_r[J];
    float later_w[J];
    auto choices = [&](int j0) {   // loaded while the rows of those in front are on their way
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const bool some = j0 + j < a.k;
        later_r[j] = some ? row_of(a, t * a.k + j0 + j) : -1;
        later_w[j] = some ? weight_of<W>(a.weights, t * a.k + j0 + j) : 0.f;
      }
    };
    choices(0);
    for (int j0 = 0; j0 < a.k; j0 += J) {
      Pair v[J][U];
      Across from[J];
      float w[J];
      int r[J];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        r[j] = later_r[j];
        w[j] = later_w[j];
      }
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (r[j] < 0) continue;
        const char* row = row_at(a.rows, r[j], a.bytes);
        from[j] = ODD ? across(row, cut) : Across{reinterpret_cast<const uint4*>(row), 0};
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (q0 + u * a.lanes < cut.pieces) v[j][u] = load_pair(from[j], q0 + u * a.lanes);
      }
      choices(j0 + J);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (r[j] < 0) continue;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float f[N];
          unpack<T>(joined(v[j][u], ODD ? from[j].off : 0), f);
#pragma unroll
          for (int i = 0; i < N; ++i) acc[u][i] = fmaf(w[j], f[i], acc[u][i]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (q0 + u * a.lanes < cut.pieces) out[q0 + u * a.lanes] = pack<T>(acc[u]);
  }
  if (ODD)
    for (int i = l; i < MOST_ENDS<T>; i += a.lanes) {
      const int at = end_element<T>(cut, a.bytes, i);
      if (at < 0) continue;
      float sum = 0.f;
      for (int j = 0; j < a.k; ++j) {
        const int r = row_of(a, t * a.k + j);
        if (r >= 0) sum = fmaf(weight_of<W>(a.weights, t * a.k + j), to_float(*reinterpret_cast<const T*>(row_at(a.rows, r, a.bytes) + at)), sum);
      }
      *reinterpret_cast<T*>(y + at) = from_float<T>(sum);
    }
}

// drows[pos[t, j]] = w[t, j] * dy[t], rows of no choice zero; dw[t, j] = the sum of dy[t] * rows[pos[t, j]], added in an order that
// depends on the sizes only.  A row is written by the choice that src names, so that rows are written once whatever pos holds.  J choices at
// a time share the loads of dy.
template <typename T, typename W, int J, int U>
__global__ void __launch_bounds__(THREADS) combine_backward_kernel(const CombineArgs a) {
  constexpr int N = PER_PIECE<T>;
  __shared__ float part[THREADS / 32][MAX_CHOICES];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = threadIdx.x & (a.lanes - 1);
  const int64_t t = (int64_t)blockIdx.x * (THREADS / a.lanes) + threadIdx.x / a.lanes;
  const bool live = t < a.tokens;
  const char* dy = row_at(a.dy, t, a.bytes);
  for (int j0 = 0; j0 < a.k; j0 += J) {
    float w[J], dot[J];
    const char* from[J];   // the choice's row, null: nothing to read, or to write
    char* to[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int64_t i = t * a.k + j0 + j;
      const int r = live && j0 + j < a.k ? row_of(a, i) : -1;
      w[j] = r >= 0 ? weight_of<W>(a.weights, i) : 0.f;
      from[j] = r >= 0 && a.dweights ? row_at(a.rows, r, a.bytes) : nullptr;
      to[j] = r >= 0 && a.drows && a.src[r] == (int32_t)i ? row_at(a.drows, r, a.bytes) : nullptr;
      dot[j] = 0.f;
    }
    const int pieces = live ? a.bytes / 16 : 0;
    for (int q0 = l; q0 < pieces; q0 += U * a.lanes) {
      uint4 g[U], v[J][U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (q0 + u * a.lanes < pieces) g[u] = reinterpret_cast<const uint4*>(dy)[q0 + u * a.lanes];
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (from[j] && q0 + u * a.lanes < pieces) v[j][u] = reinterpret_cast<const uint4*>(from[j])[q0 + u * a.lanes];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (q0 + u * a.lanes >= pieces) break;
        float d[N];
        unpack<T>(g[u], d);
#pragma unroll
        for (int j = 0; j < J; ++j) {
          if (from[j]) {
            float f[N];
            unpack<T>(v[j][u], f);
#pragma unroll
            for (int q = 0; q < N; ++q) dot[j] = fmaf(d[q], f[q], dot[j]);
          }
          if (to[j]) {
            float f[N];
#pragma unroll
            for (int q = 0; q < N; ++q) f[q] = d[q] * w[j];
            reinterpret_cast<uint4*>(to[j])[q0 + u * a.lanes] = pack<T>(f);
          }
        }
      }
    }
    if (a.dweights) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        for (int o = (a.lanes < 32 ? a.lanes : 32) / 2; o > 0; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
        if (j0 + j >= a.k) continue;
        if (a.lanes >= 32) {
          if (lane == 0) part[warp][j0 + j] = dot[j];
        } else if (l == 0 && live)
          static_cast<W*>(a.dweights)[t * a.k + j0 + j] = from_float<W>(dot[j]);
      }
    }
  }
  if (a.dweights && a.lanes >= 32) {
    __syncthreads();
    const int warps = a.lanes / 32, per_block = THREADS / a.lanes;
    for (int q = threadIdx.x; q < per_block * a.k; q += THREADS) {
      const int g = q / a.k, j = q - g * a.k;
      const int64_t at = (int64_t)blockIdx.x * per_block + g;
      if (at >= a.tokens) break;
      float sum = 0.f;
      for (int i = 0; i < warps; ++i) sum += part[g * warps + i][j];
      static_cast<W*>(a.dweights)[at * a.k + j] = from_float<W>(sum);
    }
  }
  if (a.drows)
    for (int64_t r = (int64_t)blockIdx.x * (THREADS / 32) + warp; r < a.n_rows; r += (int64_t)gridDim.x * (THREADS / 32))
      if (a.src[r] < 0) copy_odd<T>(row_at(a.drows, r, a.bytes), nullptr, a.bytes, lane, 32);
}

// Odd rows, a warp each: the choice that src names has its whole dot product there and its gradient's row to write.  Pieces are those of
// the row that is written, so dy is put together anew for each of them.  Latency bounds it, so many warps beat many loads a warp: 9460 x
// 658 bf16 with 8 choices 56 us (two pieces a lane and three blocks an SM 69, choice by choice of a token 165).
template <typename T, typename W>
__global__ void __launch_bounds__(THREADS, 5) combine_backward_odd_kernel(const CombineArgs a) {
  constexpr int N = PER_PIECE<T>, U = 1;
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * (THREADS / 32), me = (int64_t)(threadIdx.x >> 5) * gridDim.x + blockIdx.x, choices = a.tokens * a.k;
  int next = me < a.n_rows ? a.src[me] : -1;
  for (int64_t r = me; r < a.n_rows; r += warps) {
    const int i = next;
    next = r + warps < a.n_rows ? a.src[r + warps] : -1;
    char* to = a.drows ? row_at(a.drows, r, a.bytes) : nullptr;
    if (i < 0 || i >= choices) {
      if (to) copy_odd<T>(to, nullptr, a.bytes, lane, 32);
      continue;
    }
    const float w = weight_of<W>(a.weights, i);
    const char *dy = row_at(a.dy, i / a.k, a.bytes), *row = row_at(a.rows, r, a.bytes);
    const Cut cut = cut_of(to ? to : row, a.bytes);
    const Across g_from = across(dy, cut), v_from = across(row, cut);
    float dot = 0.f;
    if (lane < MOST_ENDS<T>) {
      const int at = end_element<T>(cut, a.bytes, lane);
      if (at >= 0) {
        const float d = to_float(*reinterpret_cast<const T*>(dy + at));
        if (a.dweights) dot = d * to_float(*reinterpret_cast<const T*>(row + at));
        if (to) *reinterpret_cast<T*>(to + at) = from_float<T>(d * w);
      }
    }
    for (int q0 = lane; q0 < cut.pieces; q0 += U * 32) {
      Pair g[U], v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (q0 + u * 32 < cut.pieces) {
          g[u] = load_pair(g_from, q0 + u * 32);
          if (a.dweights) v[u] = load_pair(v_from, q0 + u * 32);
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (q0 + u * 32 >= cut.pieces) break;
        float d[N];
        unpack<T>(joined(g[u], g_from.off), d);
        if (a.dweights) {
          float f[N];
          unpack<T>(joined(v[u], v_from.off), f);
#pragma unroll
          for (int q = 0; q < N; ++q) dot = fmaf(d[q], f[q], dot);
        }
        if (to) {
#pragma unroll
          for (int q = 0; q < N; ++q) d[q] *= w;
          reinterpret_cast<uint4*>(to + cut.head)[q0 + u * 32] = pack<T>(d);
        }
      }
    }
    if (a.dweights) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      if (lane == 0) static_cast<W*>(a.dweights)[i] = from_float<W>(dot);
    }
  }
  if (a.dweights)   // choices without a row
    for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < choices; i += (int64_t)gridDim.x * THREADS) {
      const int r = row_of(a, i);
      if (r < 0 || a.src[r] != (int32_t)i) static_cast<W*>(a.dweights)[i] = from_float<W>(0.f);
    }
}

// The same two for many tokens with rows of whole 16 bytes.  What bounds them is how many bytes are in flight: with loads into registers
// 14 warps of an SM waited for 64 KB at most, and for their positions first.  Here every lane copies its pieces asynchronously into a
// ring of its own in shared memory, two stages of two choices' (and dy's) pieces, and reads back what it copied itself, so nobody waits
// for anybody else.  The positions of a token are loaded while the one before it is copied; a warp goes through whole tokens.
// 16384 x 4096 bf16, 2 choices: 82 -> 65 us (6.2 TB/s) and 149 -> 120 (5.7).  8 warps and twice the stages 73 and 129, half the
// pieces and twice the stages 65 and 125.
constexpr int RING_THREADS = 512, RING_STAGES = 2, RING_PIECES = 4, RING_J = 2, RING_SEG = 32 * RING_PIECES;   // a stage holds a segment of each row
constexpr int RING_MAX_CHOICES = 32;   // one a lane
template <bool BACKWARD> constexpr int RING_ROWS = RING_J + (BACKWARD ? 1 : 0);
template <bool BACKWARD> constexpr int RING_SMEM = RING_THREADS / 32 * RING_STAGES * RING_ROWS<BACKWARD> * RING_SEG * 16;

__device__ __forceinline__ void copy_async(uint32_t to, const uint4* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ uint4 load_shared(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

template <typename T, typename W, bool BACKWARD>
__global__ void __launch_bounds__(RING_THREADS) combine_ring_kernel(const CombineArgs a) {
  constexpr int N = PER_PIECE<T>, ROWS = RING_ROWS<BACKWARD>, STAGE = ROWS * RING_SEG * 16;
  extern __shared__ __align__(16) uint8_t ring_raw[];
  const int lane = threadIdx.x & 31;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(ring_raw) + (threadIdx.x >> 5) * RING_STAGES * STAGE + lane * 16;
  const int64_t warps = (int64_t)gridDim.x * (RING_THREADS / 32), me = (int64_t)(threadIdx.x >> 5) * gridDim.x + blockIdx.x;
  const int64_t pieces = a.bytes / 16;
  const int segments = (int)((pieces + RING_SEG - 1) / RING_SEG);
  const bool dots = BACKWARD && a.dweights;

  // Where a walk over the warp's stages is.
  struct Walk {
    int64_t token;
    int segment, choice;   // the first choice of the stage
  };
  auto step = [&](Walk& w) {   // whether it enters another token
    w.choice += RING_J;
    if (w.choice < a.k) return false;
    w.choice = 0;
    if (++w.segment < segments) return false;
    w.segment = 0;
    w.token += warps;
    return true;
  };
  // The lane's choice of a token: its row, or -1.
  auto choice_of = [&](int64_t token) { return token < a.tokens && lane < a.k ? row_of(a, token * a.k + lane) : -1; };

  Walk issue{me, 0, 0}, use{me, 0, 0};
  int issue_row = choice_of(me), next_row = choice_of(me + warps), slot = 0;
  auto issue_stage = [&]() {
    if (issue.token < a.tokens) {
      const uint32_t to = ring + slot * STAGE;
      const int64_t c0 = (int64_t)issue.segment * RING_SEG + lane;
      if (BACKWARD && issue.choice == 0) {
#pragma unroll
        for (int p = 0; p < RING_PIECES; ++p)
          if (c0 + p * 32 < pieces) copy_async(to + (RING_J * RING_PIECES + p) * 512, static_cast<const uint4*>(a.dy) + issue.token * pieces + c0 + p * 32);
      }
      if (!BACKWARD || dots) {
#pragma unroll
        for (int j = 0; j < RING_J; ++j) {
          const int r = __shfl_sync(0xffffffffu, issue_row, (issue.choice + j) & 31);
          if (issue.choice + j < a.k && r >= 0) {
#pragma unroll
            for (int p = 0; p < RING_PIECES; ++p)
              if (c0 + p * 32 < pieces) copy_async(to + (j * RING_PIECES + p) * 512, static_cast<const uint4*>(a.rows) + (int64_t)r * pieces + c0 + p * 32);
          }
        }
      }
      if (step(issue)) {
        issue_row = next_row;
        next_row = choice_of(issue.token + warps);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");   // a group a stage, also where there is nothing to copy
    slot = slot + 1 == RING_STAGES ? 0 : slot + 1;
  };

  // What the lane's choice of the token in use needs: row, weight, and the choice that may write the row.
  auto weight_at = [&](int64_t token) { return token < a.tokens && lane < a.k ? weight_of<W>(a.weights, token * a.k + lane) : 0.f; };
  auto owner_of = [&](int row) { return BACKWARD && a.drows && row >= 0 ? a.src[row] : -1; };
  int row = choice_of(me), later_row = choice_of(me + warps), owner = owner_of(row), later_owner = owner_of(later_row);
  float weight = weight_at(me), later_weight = weight_at(me + warps), dot = 0.f;   // dot: of the lane's choice

  for (int i = 0; i < RING_STAGES - 1; ++i) issue_stage();
  uint4 g[RING_PIECES];
  float acc[RING_PIECES][N];
  for (int at = 0; use.token < a.tokens; at = at + 1 == RING_STAGES ? 0 : at + 1) {
    issue_stage();
    asm volatile("cp.async.wait_group %0;" ::"n"(RING_STAGES - 1) : "memory");
    const uint32_t from = ring + at * STAGE;
    const int64_t c0 = (int64_t)use.segment * RING_SEG + lane;
    if (use.choice == 0) {
#pragma unroll
      for (int p = 0; p < RING_PIECES; ++p) {
        if (BACKWARD) g[p] = load_shared(from + (RING_J * RING_PIECES + p) * 512);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[p][i] = 0.f;
      }
    }
#pragma unroll
    for (int j = 0; j < RING_J; ++j) {
      const int c = use.choice + j, r = __shfl_sync(0xffffffffu, row, c & 31);
      const float w = __shfl_sync(0xffffffffu, weight, c & 31);
      const bool mine = BACKWARD && __shfl_sync(0xffffffffu, owner, c & 31) == (int32_t)(use.token * a.k + c);
      if (c >= a.k || r < 0) continue;
      float sum = 0.f;
#pragma unroll
      for (int p = 0; p < RING_PIECES; ++p) {
        if (c0 + p * 32 >= pieces) break;
        float f[N];
        if (!BACKWARD) {
          unpack<T>(load_shared(from + (j * RING_PIECES + p) * 512), f);
#pragma unroll
          for (int i = 0; i < N; ++i) acc[p][i] = fmaf(w, f[i], acc[p][i]);
        } else {
          float d[N];
          unpack<T>(g[p], d);
          if (dots) {
            unpack<T>(load_shared(from + (j * RING_PIECES + p) * 512), f);
#pragma unroll
            for (int i = 0; i < N; ++i) sum = fmaf(d[i], f[i], sum);
          }
          if (mine) {
#pragma unroll
            for (int i = 0; i < N; ++i) d[i] *= w;
            static_cast<uint4*>(a.drows)[(int64_t)r * pieces + c0 + p * 32] = pack<T>(d);
          }
        }
      }
      if (dots) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == c) dot += sum;
      }
    }
    const Walk done = use;
    if (!BACKWARD && use.choice + RING_J >= a.k) {
#pragma unroll
      for (int p = 0; p < RING_PIECES; ++p)
        if (c0 + p * 32 < pieces) static_cast<uint4*>(a.y)[use.token * pieces + c0 + p * 32] = pack<T>(acc[p]);
    }
    if (step(use)) {
      if (dots && lane < a.k) static_cast<W*>(a.dweights)[done.token * a.k + lane] = from_float<W>(dot);
      dot = 0.f;
      row = later_row;
      weight = later_weight;
      owner = later_owner;
      later_row = choice_of(use.token + warps);
      later_weight = weight_at(use.token + warps);
      later_owner = owner_of(later_row);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (BACKWARD && a.drows)
    for (int64_t r = me; r < a.n_rows; r += warps)
      if (a.src[r] < 0) copy_odd<T>(row_at(a.drows, r, a.bytes), nullptr, a.bytes, lane, 32);
}

// ------------------------------------------------------------------------------------------ host
// The ring wants a token or more for most of its 2368 warps, and rows that fill a warp's pieces: forward, 2 choices of bf16,
// 1024 x 4096 5.6 us against 5.1, 2048 x 4096 9.4 against 12.1; backward 512 x 4096 7.3 against 4.5, 1024 x 4096 8.9 against 9.2,
// 1037 x 2176 fp32 8.8 against 12.3.
bool ring_fits(const CombineArgs& a, bool backward) {
  return a.k <= RING_MAX_CHOICES && a.bytes > 512 && a.tokens >= (backward ? 1024 : 2048);
}
// Threads of a token: one a piece for short rows and where there are few tokens to fill the SMs with, else what has four pieces each
// in flight, up to the block.
int lanes_for(int64_t bytes, int64_t tokens) {
  const int64_t few = 2048ll * sm_count();
  int lanes = MIN_LANES;
  while (lanes < THREADS && lanes * 16 < bytes && (lanes < 32 || lanes * 64 < bytes || tokens * lanes < few)) lanes *= 2;
  return lanes;
}
// Blocks for all tokens, and for the rows of no choice, of which there may be many more (padding behind a few tokens): a warp a row.
unsigned blocks_for(int64_t tokens, int lanes, int64_t rows) {
  const int64_t copies = (tokens + THREADS / lanes - 1) / (THREADS / lanes), resident = 4ll * sm_count();
  int64_t clears = (rows + THREADS / 32 - 1) / (THREADS / 32);
  if (clears > resident) clears = resident;
  const int64_t blocks = copies > clears ? copies : clears;
  return (unsigned)(blocks ? blocks : 1);
}
// Choices of a block that counts and places them: one a thread, more where all blocks' counts, which every block adds up, would be
// over 16384.
int64_t sort_chunk(int64_t n, int64_t experts) {
  int64_t chunk = THREADS;
  while ((n + chunk - 1) / chunk * experts > 16384) chunk *= 2;
  return chunk;
}
int elem_size(int dtype) { return dtype == I8L_DTYPE_F32 ? 4 : 2; }

int check_rows(const char* name, int64_t tokens, int64_t cols, int64_t rows, int k, int dtype, int wdtype = I8L_DTYPE_F32) {
  if (dtype != I8L_DTYPE_BF16 && dtype != I8L_DTYPE_F16 && dtype != I8L_DTYPE_F32) return fail(I8L_ERR_ARG, "%s: unknown dtype %d", name, dtype);
  if (wdtype != I8L_DTYPE_F32 && wdtype != dtype) return fail(I8L_ERR_ARG, "%s: weights are fp32 or of the rows' type", name);
  if (k < 1 || k > MAX_CHOICES) return fail(I8L_ERR_SHAPE, "%s: %d choices a token, 1 to %d are possible", name, k, MAX_CHOICES);
  if (tokens < 0 || cols < 1 || rows < 0 || tokens > (1ll << 30) / k || rows >= (1ll << 31) || cols > (1ll << 28))
    return fail(I8L_ERR_SHAPE, "%s: tokens=%lld cols=%lld rows=%lld out of range", name, (long long)tokens, (long long)cols, (long long)rows);
  return I8L_OK;
}
bool aligned_to(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <typename T, typename W, bool BACKWARD>
int launch_ring(const CombineArgs& a, cudaStream_t st) {
  static std::atomic<int> allowed[MAX_SMEM_DEVICES];
  auto kernel = combine_ring_kernel<T, W, BACKWARD>;
  I8L_CUDA_OK(allow_smem(kernel, allowed, RING_SMEM<BACKWARD>));
  kernel<<<sm_count(), RING_THREADS, RING_SMEM<BACKWARD>, st>>>(a);
  I8L_CUDA_OK(cudaGetLastError());
  return I8L_OK;
}
template <typename T, typename W>
int launch_combine(const CombineArgs& a, bool backward, bool odd, cudaStream_t st) {
  if (!odd && ring_fits(a, backward)) return backward ? launch_ring<T, W, true>(a, st) : launch_ring<T, W, false>(a, st);
  const unsigned grid = blocks_for(a.tokens, a.lanes, backward && a.drows ? a.n_rows : 0);
  const bool one = a.bytes <= 16 * a.lanes;    // a piece a thread: fewer registers, more blocks on an SM
  if (backward) {
    if (odd) combine_backward_odd_kernel<T, W><<<10 * sm_count(), THREADS, 0, st>>>(a);
    else if (one) combine_backward_kernel<T, W, 2, 1><<<grid, THREADS, 0, st>>>(a);
    else if (a.k <= 2) combine_backward_kernel<T, W, 2, 2><<<grid, THREADS, 0, st>>>(a);
    else combine_backward_kernel<T, W, 4, 2><<<grid, THREADS, 0, st>>>(a);
  } else {
    if (odd) combine_kernel<T, W, true, 1, 1><<<grid, THREADS, 0, st>>>(a);
    else if (one) combine_kernel<T, W, false, 4, 1><<<grid, THREADS, 0, st>>>(a);
    else if (a.k <= 2) combine_kernel<T, W, false, 2, 4><<<grid, THREADS, 0, st>>>(a);
    else combine_kernel<T, W, false, 4, 2><<<grid, THREADS, 0, st>>>(a);
  }
  I8L_CUDA_OK(cudaGetLastError());
  return I8L_OK;
}
template <typename T>
int launch_combine(const CombineArgs& a, int wdtype, bool backward, bool odd, cudaStream_t st) {
  return wdtype == I8L_DTYPE_F32 ? launch_combine<T, float>(a, backward, odd, st) : launch_combine<T, T>(a, backward, odd, st);
}
int run_combine(CombineArgs a, int64_t cols, int dtype, int wdtype, bool backward, cudaStream_t st) {
  a.bytes = (int)(cols * elem_size(dtype));
  a.lanes = lanes_for(a.bytes, a.tokens);
  const bool odd = a.bytes % 16 || !aligned16(a.rows) || !aligned16(a.y) || !aligned16(a.dy) || !aligned16(a.drows);
  if (dtype == I8L_DTYPE_F32) return launch_combine<float, float>(a, backward, odd, st);
  if (dtype == I8L_DTYPE_F16) return launch_combine<__half>(a, wdtype, backward, odd, st);
  return launch_combine<__nv_bfloat16>(a, wdtype, backward, odd, st);
}

}  // namespace
}  // namespace i8l

using namespace i8l;

extern "C" int64_t i8l_sort_workspace(int64_t tokens, int k, int experts) {
  if (tokens < 0 || k < 1 || k > MAX_CHOICES || tokens > (1ll << 30) / k || experts < 1 || experts > MAX_EXPERTS) return 0;   // refused
  if (tokens * k <= SMALL_SORT) return 0;
  const int64_t chunk = sort_chunk(tokens * k, experts);
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
  if (!aligned_to(x, size) || !aligned_to(out, size) || !aligned_to(ids, ids64 ? 8 : 4) || !aligned_to(offsets, 4) || !aligned_to(pos, 4) ||
      !aligned_to(src, 4) || !aligned_to(workspace, 4))
    return fail(I8L_ERR_ALIGN, "i8l_sort_tokens: pointers are aligned to their elements");
  if (workspace_bytes < i8l_sort_workspace(tokens, k, experts) || (i8l_sort_workspace(tokens, k, experts) && !workspace))
    return fail(I8L_ERR_ARG, "i8l_sort_tokens: workspace of %lld bytes is too small", (long long)workspace_bytes);
  if (int e = check_arch()) return e;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool odd = cols * size % 16 || !aligned16(x) || !aligned16(out);
  SortArgs a{};
  a.x = x; a.ids = ids; a.rows = out; a.offsets = offsets; a.pos = pos; a.src = src;
  a.hist = static_cast<int32_t*>(workspace);
  a.tokens = tokens; a.bytes = (int)(cols * size);
  a.n = (int)n; a.k = k; a.experts = experts; a.align = (int)align; a.n_rows = (int)rows; a.ids64 = ids64 ? 1 : 0;
  a.lanes = lanes_for(a.bytes, tokens);
  const unsigned grid = blocks_for(tokens, a.lanes, rows);
  if (n <= SMALL_SORT) {
    if (!odd) sort_small_kernel<uint32_t, false><<<grid, THREADS, 0, st>>>(a);
    else if (size == 4) sort_small_kernel<uint32_t, true><<<grid, THREADS, 0, st>>>(a);
    else sort_small_kernel<uint16_t, true><<<grid, THREADS, 0, st>>>(a);
    I8L_CUDA_OK(cudaGetLastError());
    return I8L_OK;
  }
  a.chunk = (int)sort_chunk(n, experts);
  a.blocks = (int)((n + a.chunk - 1) / a.chunk);
  const LaunchChain chain(st);
  (void)chain_first();
  I8L_CUDA_OK(launch(sort_count_kernel, dim3(a.blocks), THREADS, 0, st, a));
  I8L_CUDA_OK(launch(sort_place_kernel, dim3(a.blocks), THREADS, THREADS / 32 * experts * sizeof(int), st, a));
  if (odd) a.lanes = lanes_for(a.bytes, rows);
  const int64_t row_blocks = (rows + THREADS / a.lanes - 1) / (THREADS / a.lanes), resident = 16 * sm_count();
  const dim3 by_row((unsigned)(row_blocks < resident ? row_blocks : resident));
  I8L_CUDA_OK(!odd        ? launch(sort_copy_kernel, dim3(grid), THREADS, 0, st, a)
              : size == 4 ? launch(sort_copy_odd_kernel<uint32_t>, by_row, THREADS, 0, st, a)
                          : launch(sort_copy_odd_kernel<uint16_t>, by_row, THREADS, 0, st, a));
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
  return run_combine(a, cols, dtype, wdtype, false, static_cast<cudaStream_t>(stream));
}

extern "C" int i8l_combine_backward(const void* rows, const void* weights, const int32_t* pos, const int32_t* src, const void* dy,
                                    int64_t n_rows, int64_t tokens, int64_t cols, int k, int dtype, int wdtype, void* drows, void* dweights,
                                    void* stream) {
  if (int e = check_rows("i8l_combine_backward", tokens, cols, n_rows, k, dtype, wdtype)) return e;
  if ((!tokens || !dweights) && (!n_rows || !drows)) return I8L_OK;
  if ((tokens && (!pos || !dy || !weights)) || (n_rows && (!rows || !src))) return fail(I8L_ERR_ARG, "i8l_combine_backward: null pointer");
  const int size = elem_size(dtype);
  const int wsize = wdtype == I8L_DTYPE_F32 ? 4 : 2;
  if (!aligned_to(rows, size) || !aligned_to(dy, size) || !aligned_to(drows, size) || !aligned_to(weights, wsize) || !aligned_to(dweights, wsize) ||
      !aligned_to(pos, 4) || !aligned_to(src, 4))
    return fail(I8L_ERR_ALIGN, "i8l_combine_backward: pointers are aligned to their elements");
  if (int e = check_arch()) return e;
  CombineArgs a{};
  a.rows = rows; a.weights = weights; a.pos = pos; a.src = src; a.dy = dy; a.drows = drows; a.dweights = dweights;
  a.tokens = tokens; a.n_rows = n_rows; a.k = k;
  return run_combine(a, cols, dtype, wdtype, true, static_cast<cudaStream_t>(stream));
}

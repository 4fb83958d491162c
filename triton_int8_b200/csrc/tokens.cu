// The INT8 product for serving: bf16 rows x int8 weights that were quantized once, for any number of rows, one weight matrix an
// expert (i8l_token_linear).  Row scales and channel scales are those of the double_channel variant, so that the sum over K is
// exact in int32 and an output needs one product by each scale.
#include "common.cuh"
#include "ptx.cuh"

namespace i8l {
namespace {

constexpr int MAX_EXPERTS = 1024;
constexpr int64_t MAX_K = 131072;   // 127 * 128 * K < 2^31

struct TokenArgs {
  const __nv_bfloat16* x;
  const int8_t* wq;
  const float* ws;
  const int32_t* offsets;   // null: one matrix for all rows
  const __nv_bfloat16* bias;
  void* y;
  int64_t rows, N, K;
  int experts, out_f32;
};

// Rows of expert e, inside [0, rows) whatever the offsets hold.
__device__ __forceinline__ void segment(const TokenArgs& a, int e, int64_t& begin, int64_t& end) {
  if (!a.offsets) {
    begin = 0;
    end = a.rows;
    return;
  }
  const int64_t b = a.offsets[e], n = a.offsets[e + 1];
  begin = b < 0 ? 0 : (b < a.rows ? b : a.rows);
  end = n < begin ? begin : (n < a.rows ? n : a.rows);
}

__device__ __forceinline__ uint4 load_weights(const int8_t* p) {   // read once: no place in L1
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// ------------------------------------------------------------------------------------------ few rows
// One launch: a block takes 32 channels of one expert, quantizes up to MT of its rows into shared memory and multiplies them with the
// channels' weights by dp4a, a warp four channels at a time, so that a piece of x read from shared memory serves four loads of
// weights.  Bound by the weights' bytes.
constexpr int FEW_THREADS = 256, FEW_WARP_COLS = 4, FEW_COLS = FEW_THREADS / 32 * FEW_WARP_COLS;

template <int MT>
__global__ void __launch_bounds__(FEW_THREADS) few_rows_kernel(const TokenArgs a) {
  extern __shared__ __align__(16) int8_t xq[];   // [MT, K]
  __shared__ float xs[MT], red[FEW_THREADS / 32];
  __shared__ int s_expert;
  constexpr int LANES = FEW_THREADS / MT;        // threads that quantize a row
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int K = (int)a.K;
  int64_t begin, end;
  int e = 0;
  if (a.offsets) {   // the blockIdx.y-th expert that has rows
    if (warp == 0) {
      int found = -1, left = blockIdx.y;
      for (int e0 = 0; e0 < a.experts && found < 0; e0 += 32) {
        bool some = false;
        if (e0 + lane < a.experts) {
          segment(a, e0 + lane, begin, end);
          some = end > begin;
        }
        const unsigned set = __ballot_sync(0xffffffffu, some);
        if (left < __popc(set)) found = e0 + (int)__fns(set, 0, left + 1);
        else left -= __popc(set);
      }
      if (lane == 0) s_expert = found;
    }
    __syncthreads();
    e = s_expert;
  }
  const int64_t n0 = (int64_t)blockIdx.x * FEW_COLS + warp * FEW_WARP_COLS;
  if (a.offsets && blockIdx.y == 0) {   // rows of no expert
    int64_t b, n, last_b, last_n;
    segment(a, 0, b, n);
    segment(a, a.experts - 1, last_b, last_n);
    const int64_t dead = b + (a.rows - last_n);
    for (int64_t i = tid; i < dead * FEW_COLS; i += FEW_THREADS) {
      const int64_t r = i / FEW_COLS, c = (int64_t)blockIdx.x * FEW_COLS + i % FEW_COLS;
      const int64_t at = (r < b ? r : last_n + r - b) * a.N + c;
      if (c < a.N) {
        if (a.out_f32) static_cast<float*>(a.y)[at] = 0.f;
        else static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(0.f);
      }
    }
  }
  if (e < 0) return;
  segment(a, e, begin, end);
  const int8_t* w = a.wq + ((int64_t)e * a.N + n0) * a.K;
  for (int64_t r0 = begin; r0 < end; r0 += MT) {
    // the rows in int8, a scale each
    {
      const int t = tid / LANES, l = tid & (LANES - 1);
      const bool live = r0 + t < end;
      const uint4* row = reinterpret_cast<const uint4*>(a.x + (r0 + t) * a.K);
      float m = 0.f;
      if (live)
        for (int c = l; c < K / 8; c += LANES) {
          float v[8];
          unpack8(row[c], v);
#pragma unroll
          for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      __syncthreads();   // also: the rows in front of these have been multiplied
      if (lane == 0) red[warp] = m;
      __syncthreads();
      m = red[t * (LANES / 32)];
#pragma unroll
      for (int i = 1; i < LANES / 32; ++i) m = fmaxf(m, red[t * (LANES / 32) + i]);
      float s, stored;
      make_scale<I8L_QMODE_ROWRCP>(m, s, stored);
      if (l == 0) xs[t] = stored;
      uint2* q = reinterpret_cast<uint2*>(xq + (int64_t)t * K);
      for (int c = l; c < K / 8; c += LANES) q[c] = live ? quant_piece<I8L_QMODE_ROWRCP>(row[c], s) : make_uint2(0, 0);
      __syncthreads();
    }
    if (n0 >= a.N) continue;
    int acc[FEW_WARP_COLS][MT];
#pragma unroll
    for (int j = 0; j < FEW_WARP_COLS; ++j)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[j][t] = 0;
#pragma unroll 2
    for (int k = lane * 16; k < K; k += 512) {
      uint4 u[FEW_WARP_COLS];
#pragma unroll
      for (int j = 0; j < FEW_WARP_COLS; ++j) u[j] = load_weights(w + (int64_t)j * K + k);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const uint4 v = *reinterpret_cast<const uint4*>(xq + (int64_t)t * K + k);
#pragma unroll
        for (int j = 0; j < FEW_WARP_COLS; ++j) {
          acc[j][t] = __dp4a((int)u[j].x, (int)v.x, acc[j][t]);
          acc[j][t] = __dp4a((int)u[j].y, (int)v.y, acc[j][t]);
          acc[j][t] = __dp4a((int)u[j].z, (int)v.z, acc[j][t]);
          acc[j][t] = __dp4a((int)u[j].w, (int)v.w, acc[j][t]);
        }
      }
    }
    int mine = 0;   // lane j * MT + t has the sum of channel j and row t
#pragma unroll
    for (int j = 0; j < FEW_WARP_COLS; ++j)
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const int sum = __reduce_add_sync(0xffffffffu, acc[j][t]);
        if (lane == j * MT + t) mine = sum;
      }
    const int j = lane / MT, t = lane % MT;
    if (j < FEW_WARP_COLS && r0 + t < end) {
      const int64_t n = n0 + j, c = (int64_t)e * a.N + n, at = (r0 + t) * a.N + n;
      float v = __fmul_rn(__fmul_rn(__int2float_rn(mine), xs[t]), a.ws[c]);
      if (a.bias) v = __fadd_rn(v, __bfloat162float(a.bias[c]));
      if (a.out_f32) static_cast<float*>(a.y)[at] = v;
      else static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(v);
    }
  }
}

constexpr int FEW_SMEM = 160 * 1024;
template <int MT> int launch_few(const TokenArgs& a, cudaStream_t st) {
  const size_t smem = (size_t)(MT * a.K);
  if (smem > 48 * 1024) I8L_CUDA_OK(cudaFuncSetAttribute(few_rows_kernel<MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const int64_t segments = a.offsets ? (a.experts < a.rows ? a.experts : a.rows) : 1;
  few_rows_kernel<MT><<<dim3((unsigned)((a.N + FEW_COLS - 1) / FEW_COLS), (unsigned)segments), FEW_THREADS, smem, st>>>(a);
  I8L_CUDA_OK(cudaGetLastError());
  return I8L_OK;
}

}  // namespace
}  // namespace i8l

using namespace i8l;

extern "C" int64_t i8l_token_linear_workspace(int64_t rows, int64_t K) {
  if (rows <= 0 || K <= 0 || rows >= (1ll << 31) || K > MAX_K) return 0;
  return (rows * K + 255) / 256 * 256 + (4 * rows + 255) / 256 * 256;
}

extern "C" int i8l_token_linear(const void* x, const int8_t* w_q, const float* w_scale, const int32_t* offsets, const void* bias, void* y,
                                int64_t rows, int experts, int64_t N, int64_t K, int flags, void* workspace, int64_t workspace_bytes,
                                int32_t* status, void* stream) {
  if (rows < 0 || rows >= (1ll << 31) || N < 8 || N % 8 || K < 16 || K % 16 || K > MAX_K || N >= (1ll << 31))
    return fail(I8L_ERR_SHAPE, "i8l_token_linear: rows=%lld N=%lld K=%lld: N a multiple of 8, K of 16 and at most %lld", (long long)rows,
                (long long)N, (long long)K, (long long)MAX_K);
  if (experts < 1 || experts > MAX_EXPERTS || (!offsets && experts != 1) || experts * N >= (1ll << 31))
    return fail(I8L_ERR_SHAPE, "i8l_token_linear: %d experts, 1 to %d are possible, and one without offsets", experts, MAX_EXPERTS);
  if (flags & ~I8L_GEMM_OUT_F32) return fail(I8L_ERR_ARG, "i8l_token_linear: unknown flags %d", flags);
  if (!w_q || !w_scale || (rows && (!x || !y || !workspace))) return fail(I8L_ERR_ARG, "i8l_token_linear: null pointer");
  if (!aligned16(x) || !aligned16(w_q) || !aligned16(y) || !aligned16(bias) || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return fail(I8L_ERR_ALIGN, "i8l_token_linear: x, w_q, y and bias must be 16-byte aligned, the workspace 256-byte");
  if (workspace_bytes < i8l_token_linear_workspace(rows, K))
    return fail(I8L_ERR_ARG, "i8l_token_linear: workspace of %lld bytes is too small", (long long)workspace_bytes);
  if (!rows) return I8L_OK;
  if (int e = check_arch()) return e;
  TokenArgs a{};
  a.x = static_cast<const __nv_bfloat16*>(x); a.wq = w_q; a.ws = w_scale; a.offsets = offsets;
  a.bias = static_cast<const __nv_bfloat16*>(bias); a.y = y;
  a.rows = rows; a.N = N; a.K = K; a.experts = experts; a.out_f32 = (flags & I8L_GEMM_OUT_F32) ? 1 : 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  (void)status;
  if (rows == 1 || K > FEW_SMEM / 2) return launch_few<1>(a, st);
  if (rows == 2 || K > FEW_SMEM / 4) return launch_few<2>(a, st);
  if (rows <= 4 || K > FEW_SMEM / 8) return launch_few<4>(a, st);
  return launch_few<8>(a, st);
}

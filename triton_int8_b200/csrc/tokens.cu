// The INT8 product for serving: bf16 rows x int8 weights that were quantized once, for any number of rows, one weight matrix an
// expert (i8l_token_linear).  Row scales and channel scales are those of the double_channel variant, so that the sum over K is
// exact in int32 and an output needs one product by each scale.
#include <atomic>
#include <cstddef>

#include "common.cuh"
#include "ptx.cuh"

namespace i8l {
namespace {

constexpr int MAX_EXPERTS = 1024;
constexpr int64_t MAX_K = 131072;      // 127 * 128 * K < 2^31
constexpr int64_t MAX_ROWS = 1 << 30;   // row and tile numbers are int

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
// Up to eight rows in one launch, bound by the weights' bytes.  Two kernels share the frame: every block quantizes the rows into its shared
// memory and then goes through channels of the experts that have rows, resident blocks over all of them, with loads from memory
// straight into registers, the next batch in flight while one is multiplied and the next channels on their way into L2; the first
// batch goes out ahead of the quantization.  (Set-up and drain of tcgen05 take longer than these products.)
constexpr int FEW_THREADS = 256, FEW_WARPS = FEW_THREADS / 32, FEW_ROWS = 8;
struct FewSegment {
  int expert, row, rows;
};
struct FewShared {
  float scale[FEW_ROWS], red[FEW_WARPS];
  FewSegment seg[FEW_ROWS];
  int segments;
};

// The experts that have rows, at most as many as rows.
__device__ __forceinline__ void few_segments(const TokenArgs& a, FewShared& sh) {
  const int lane = threadIdx.x & 31;
  if (!a.offsets) {
    if (threadIdx.x == 0) {
      sh.seg[0] = FewSegment{0, 0, (int)a.rows};
      sh.segments = 1;
    }
  } else if (threadIdx.x < 32) {
    int count = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      int64_t begin = 0, end = 0;
      if (e0 + lane < a.experts) segment(a, e0 + lane, begin, end);
      const unsigned set = __ballot_sync(0xffffffffu, end > begin);
      const int at = count + __popc(set & ((1u << lane) - 1));
      if (end > begin && at < FEW_ROWS) sh.seg[at] = FewSegment{e0 + lane, (int)begin, (int)(end - begin)};
      count += __popc(set);
    }
    if (lane == 0) sh.segments = count < FEW_ROWS ? count : FEW_ROWS;   // more only where offsets decrease
  }
  __syncthreads();
}
// All rows in int8, `stride` bytes apart, zeros behind K, and a scale each; as many threads a row as there are for a power of two rows.
__device__ __forceinline__ void few_quantize(const TokenArgs& a, FewShared& sh, int8_t* xq, int stride) {
  const int rows = (int)a.rows, pieces = (int)a.K / 8, lanes = rows == 1 ? 256 : rows == 2 ? 128 : rows <= 4 ? 64 : 32;
  const int t = threadIdx.x / lanes, l = threadIdx.x & (lanes - 1);
  const bool live = t < rows;
  const uint4* row = reinterpret_cast<const uint4*>(a.x + t * a.K);
  float m = 0.f;
  if (live)
#pragma unroll 4
    for (int c = l; c < pieces; c += lanes) {
      float v[8];
      unpack8(row[c], v);
#pragma unroll
      for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) sh.red[threadIdx.x >> 5] = m;
  __syncthreads();
  for (int i = 0; i < lanes / 32; ++i) m = fmaxf(m, sh.red[t * (lanes / 32) + i]);
  float s, stored;
  make_scale<I8L_QMODE_ROWRCP>(m, s, stored);
  if (live && l == 0) sh.scale[t] = stored;
  uint2* q = reinterpret_cast<uint2*>(xq + t * stride);
  if (live)
#pragma unroll 4
    for (int c = l; c < stride / 8; c += lanes) q[c] = c < pieces ? quant_piece<I8L_QMODE_ROWRCP>(row[c], s) : make_uint2(0, 0);
  __syncthreads();
}
__device__ __forceinline__ void few_store(const TokenArgs& a, const FewShared& sh, const FewSegment& seg, int r, int64_t n, int sum) {
  const int64_t c = (int64_t)seg.expert * a.N + n, at = (int64_t)(seg.row + r) * a.N + n;
  float v = __fmul_rn(__fmul_rn(__int2float_rn(sum), sh.scale[seg.row + r]), a.ws[c]);
  if (a.bias) v = __fadd_rn(v, __bfloat162float(a.bias[c]));
  if (a.out_f32) static_cast<float*>(a.y)[at] = v;
  else static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ void few_clear(const TokenArgs& a, const FewShared& sh) {   // rows of no expert
  const int64_t pieces = a.N * (a.out_f32 ? 4 : 2) / 16;
  for (int64_t r = 0; a.offsets && r < a.rows; ++r) {
    bool some = false;
    for (int i = 0; i < sh.segments; ++i) some |= r >= sh.seg[i].row && r < sh.seg[i].row + sh.seg[i].rows;
    if (some) continue;
    for (int64_t c = (int64_t)blockIdx.x * FEW_THREADS + threadIdx.x; c < pieces; c += (int64_t)gridDim.x * FEW_THREADS)
      static_cast<uint4*>(a.y)[r * pieces + c] = make_uint4(0, 0, 0, 0);
  }
}
// Where a warp is: channels from n on of segment `seg`, of K from `k` on.
struct FewPlace {
  int seg, k;
  int64_t n;
};
__device__ __forceinline__ void few_settle(FewPlace& p, int segments, int64_t channels) {   // into the segment that n belongs to
  while (p.seg < segments && p.n >= channels) {
    p.n -= channels;
    ++p.seg;
  }
}
__device__ __forceinline__ void fetch_l2(const TokenArgs& a, const FewShared& sh, const FewPlace& p, int channels) {   // by one thread
  const int64_t some = a.N - p.n < channels ? a.N - p.n : channels;
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a.wq + ((int64_t)sh.seg[p.seg].expert * a.N + p.n) * a.K), "r"((uint32_t)(some * a.K))
               : "memory");
}

// Up to four rows: a warp takes two channels at a time over all of K, 512 bytes of each a load, and multiplies by dp4a; a batch is 2 KB of
// each.  Weights from memory, 11008x4096: one row 11.7 us, two 12.1, four x 10240x4096 14.1; 4096x4096 6.3, 6.6, 7.8; one token x 2 of 8
// experts of 11008x4096 19.2 (14 of bytes).  Weights in L2 8.1, 8.7 and 11.2, 4.6, 5.0 and 6.6.  The fetch into L2 ahead took one, two and four rows x
// 11008x4096 from 11.5, 12.1 and 13.8 to 9.3, 9.8 and 12.2 where part of the weights were there.
constexpr int DP_CHANNELS = 2, DP_STEPS = 4, DP_BATCH = DP_STEPS * 512;
struct DpBatch {
  uint4 w[DP_CHANNELS][DP_STEPS];
};
template <int MT, int CT>
__device__ __forceinline__ void dp_multiply(int (&acc)[DP_CHANNELS][MT], const DpBatch& w, const int8_t* rows, int count, int K, int limit, int k0) {
  int at[CT];   // of a row: CT may be above their number, and what is multiplied with the first one once more is not used
#pragma unroll
  for (int t = 0; t < CT; ++t) at[t] = t < count ? t * K : 0;
#pragma unroll
  for (int s = 0; s < DP_STEPS; ++s) {
    const int k = k0 + s * 512;
    if (k >= limit) break;
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      const uint4 v = *reinterpret_cast<const uint4*>(rows + at[t] + k);
#pragma unroll
      for (int j = 0; j < DP_CHANNELS; ++j) {
        acc[j][t] = __dp4a((int)w.w[j][s].x, (int)v.x, acc[j][t]);
        acc[j][t] = __dp4a((int)w.w[j][s].y, (int)v.y, acc[j][t]);
        acc[j][t] = __dp4a((int)w.w[j][s].z, (int)v.z, acc[j][t]);
        acc[j][t] = __dp4a((int)w.w[j][s].w, (int)v.w, acc[j][t]);
      }
    }
  }
}

template <int MT>
__global__ void __launch_bounds__(FEW_THREADS, 2) few_dp_kernel(const TokenArgs a) {
  extern __shared__ __align__(16) int8_t xq[];   // [MT, K]
  __shared__ FewShared sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, K = (int)a.K;
  chain_wait();   // launched ahead of its predecessor's end, as the first kernels of the other calls are
  chain_trigger();
  few_segments(a, sh);
  const int segments = sh.segments;
  const int64_t step = (int64_t)gridDim.x * FEW_WARPS * DP_CHANNELS;
  auto load = [&](DpBatch& b, const FewPlace& p) {
    if (p.seg >= segments) return;
    const int8_t* w = a.wq + ((int64_t)sh.seg[p.seg].expert * a.N + p.n) * a.K + lane * 16;
#pragma unroll
    for (int s = 0; s < DP_STEPS; ++s)
#pragma unroll
      for (int j = 0; j < DP_CHANNELS; ++j)   // N is a multiple of 8: both channels or none
        if (p.k + s * 512 + lane * 16 < K) b.w[j][s] = load_weights(w + (int64_t)j * K + p.k + s * 512);
  };
  auto after = [&](FewPlace p) {
    p.n += step;
    few_settle(p, segments, a.N);
    return p;
  };
  FewPlace now{0, 0, ((int64_t)warp * gridDim.x + blockIdx.x) * DP_CHANNELS};
  few_settle(now, segments, a.N);
  DpBatch even, odd;
  load(even, now);
  FewPlace fetched = now;
  if (lane == 0 && fetched.seg < segments) fetch_l2(a, sh, fetched, DP_CHANNELS);   // the rest of these, and the next
  fetched = after(fetched);
  if (lane == 0 && fetched.seg < segments) fetch_l2(a, sh, fetched, DP_CHANNELS);
  few_quantize(a, sh, xq, K);

  int acc[DP_CHANNELS][MT];
#pragma unroll
  for (int j = 0; j < DP_CHANNELS; ++j)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[j][t] = 0;
  auto work = [&](const DpBatch& mine, DpBatch& ahead) {
    FewPlace next = now;
    next.k += DP_BATCH;
    const bool last = next.k >= K;
    if (last) {
      next = after(now);
      next.k = 0;
      fetched = after(fetched);
      if (lane == 0 && fetched.seg < segments) fetch_l2(a, sh, fetched, DP_CHANNELS);
    }
    load(ahead, next);
    const FewSegment seg = sh.seg[now.seg];
    const int8_t* rows = xq + seg.row * K + lane * 16;
    const int limit = K - lane * 16;   // of k, so that the lane's 16 bytes are inside the row
    if (MT == 1 || seg.rows == 1) dp_multiply<MT, 1>(acc, mine, rows, seg.rows, K, limit, now.k);
    else if (MT == 2 || seg.rows == 2) dp_multiply<MT, MT < 2 ? MT : 2>(acc, mine, rows, seg.rows, K, limit, now.k);
    else dp_multiply<MT, MT>(acc, mine, rows, seg.rows, K, limit, now.k);
    if (last) {
      int sum = 0;   // lane j * MT + t has that of channel j and row t
#pragma unroll
      for (int j = 0; j < DP_CHANNELS; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const int all = __reduce_add_sync(0xffffffffu, acc[j][t]);
          if (lane == j * MT + t) sum = all;
          acc[j][t] = 0;
        }
      if (lane < DP_CHANNELS * MT && lane % MT < seg.rows) few_store(a, sh, seg, lane % MT, now.n + lane / MT, sum);
    }
    now = next;
  };
  while (now.seg < segments) {
    work(even, odd);
    if (now.seg >= segments) break;
    work(odd, even);
  }
  few_clear(a, sh);
}

// Five to eight rows, which dp4a is too slow for: a block takes 16 channels at a time, its warps split K into pieces of 128 and multiply by
// mma.sync m16n8k32, channels times rows.  The order of K inside a product does not matter, so a lane's 16 contiguous bytes serve
// as its fragments as they are, for weights and rows alike.  8 rows, weights from memory, x 4096x4096 10.2 us, 6144x4096 12.4, 1024x1024 3.6; in
// L2 8.6 and 10.2.  There dp4a took 9.8 for 4096x4096; one row 5.7 against 4.4 (lines of four rows a load and the sum over the warps cost
// more).
constexpr int MMA_CHANNELS = 16, MMA_K = 128, MMA_PIECES = 2;
struct MmaBatch {
  uint4 w[MMA_PIECES][2][2];   // piece of K, channel g or g + 8, half of the piece
};
__device__ __forceinline__ void mma_16x8x32(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__global__ void __launch_bounds__(FEW_THREADS, 2) few_mma_kernel(const TokenArgs a, int row_bytes) {
  extern __shared__ __align__(16) int8_t xq[];   // [rows, row_bytes]: K rounded up to whole pieces
  __shared__ FewShared sh;
  __shared__ __align__(16) int part[2][FEW_WARPS][MMA_CHANNELS * FEW_ROWS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = (int)a.K, stride = FEW_WARPS * MMA_K;   // of a warp's pieces
  const int g = lane >> 2, byte = (lane & 3) * 16;   // the lane's channel (and g + 8) or row, its bytes of half a piece
  chain_wait();
  chain_trigger();
  few_segments(a, sh);
  const int segments = sh.segments;
  const int64_t step = (int64_t)gridDim.x * MMA_CHANNELS, width = (a.N + MMA_CHANNELS - 1) / MMA_CHANNELS * MMA_CHANNELS;
  auto load = [&](MmaBatch& b, const FewPlace& p) {
    if (p.seg >= segments) return;
    const int8_t* w = a.wq + ((int64_t)sh.seg[p.seg].expert * a.N + p.n + g) * a.K;
#pragma unroll
    for (int i = 0; i < MMA_PIECES; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int k = p.k + warp * MMA_K + i * stride + c * 64 + byte;
          b.w[i][h][c] = k < K && p.n + g + h * 8 < a.N ? load_weights(w + h * 8 * a.K + k) : make_uint4(0, 0, 0, 0);
        }
  };
  auto after = [&](FewPlace p) {
    p.n += step;
    few_settle(p, segments, width);
    return p;
  };
  FewPlace now{0, 0, (int64_t)blockIdx.x * MMA_CHANNELS};   // the same for all warps of the block
  few_settle(now, segments, width);
  MmaBatch even, odd;
  load(even, now);
  FewPlace fetched = now;
  if (tid == 0 && fetched.seg < segments) fetch_l2(a, sh, fetched, MMA_CHANNELS);   // the rest of these, and the next
  fetched = after(fetched);
  if (tid == 0 && fetched.seg < segments) fetch_l2(a, sh, fetched, MMA_CHANNELS);
  few_quantize(a, sh, xq, row_bytes);

  int acc[4] = {0, 0, 0, 0}, turn = 0;
  auto work = [&](const MmaBatch& mine, MmaBatch& ahead) {
    FewPlace next = now;
    next.k += MMA_PIECES * stride;
    const bool last = next.k >= row_bytes;
    if (last) {
      next = after(now);
      next.k = 0;
      fetched = after(fetched);
      if (tid == 0 && fetched.seg < segments) fetch_l2(a, sh, fetched, MMA_CHANNELS);
    }
    load(ahead, next);
    const FewSegment seg = sh.seg[now.seg];
    const int8_t* row = xq + (seg.row + (g < seg.rows ? g : 0)) * row_bytes + byte;   // rows past the segment's: some row, not used
#pragma unroll
    for (int i = 0; i < MMA_PIECES; ++i) {
      const int k = now.k + warp * MMA_K + i * stride;
      if (k >= row_bytes) break;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint4 x = *reinterpret_cast<const uint4*>(row + k + c * 64), &u = mine.w[i][0][c], &v = mine.w[i][1][c];
        mma_16x8x32(acc, u.x, v.x, u.y, v.y, x.x, x.y);
        mma_16x8x32(acc, u.z, v.z, u.w, v.w, x.z, x.w);
      }
    }
    if (last) {   // the warps' sums are added up; the other buffer is that of the channels before, whose readers may still be at it
      *reinterpret_cast<int4*>(&part[turn][warp][lane * 4]) = make_int4(acc[0], acc[1], acc[2], acc[3]);
      acc[0] = acc[1] = acc[2] = acc[3] = 0;
      __syncthreads();
      if (tid < MMA_CHANNELS * FEW_ROWS) {
        int sum = 0;
#pragma unroll
        for (int w = 0; w < FEW_WARPS; ++w) sum += part[turn][w][tid];
        // as mma.sync leaves them: lane l has channels l / 4 (and + 8 in the upper two), rows 2 * (l % 4) and the next one
        const int from = tid >> 2, r = (from & 3) * 2 + (tid & 1);
        const int64_t n = now.n + (from >> 2) + (tid & 2) * 4;
        if (r < seg.rows && n < a.N) few_store(a, sh, seg, r, n, sum);
      }
      turn ^= 1;
    }
    now = next;
  };
  while (now.seg < segments) {
    work(even, odd);
    if (now.seg >= segments) break;
    work(odd, even);
  }
  few_clear(a, sh);
}

// ------------------------------------------------------------------------------------------ many rows
// The tensor cores with the operands exchanged: 128 output channels are the rows of an MMA and up to TOK tokens its columns, whose
// number is the instruction's N and may be any multiple of 16.  A segment of 17 rows costs 32 columns that way, where tokens as
// MMA rows would cost 128, and the weights, which bound the product until a segment has some hundred rows, are read once.
//
// Persistent, a CTA per SM, 640 threads: warp 0 brings K blocks of 128 bytes by TMA (128 weight rows and the tokens of the tile) into a
// ring, warp 1 issues tcgen05.mma kind::i8 into one of several accumulators in tensor memory, warps 4 to 19 take a finished one
// out: a lane is a channel there, a register a token, so a bf16 tile is turned in shared memory, two tokens a word, and leaves 16 bytes a
// lane.  Warps 2 and 3 clear the rows of no expert, the others too when their tiles are done.  Tiles come from the offsets in device memory: nothing waits for the host.
// All waits are bounded, as in gemm.cu: on expiry every role leaves, the status word says so.
constexpr int GRP_THREADS = 640, GRP_EPI_WARPS = 16, CHANNELS = 128, KBYTES = 128;
constexpr int A_BYTES = CHANNELS * KBYTES;
constexpr int BOXES = 5;   // maps of 16, 32, 64, 128 and 256 tokens
constexpr int EPI_TOKENS = 16, EPI_BYTES = EPI_TOKENS * 32 * 2;   // tokens that a warp takes out at a time, x 32 channels in bf16
constexpr int CLEAR_WARPS = 2 + GRP_EPI_WARPS;
constexpr int RASTER = 16;                    // token tiles whose rows should stay in L2 while the channels are gone through

struct __align__(16) Segment {
  int row, rows;   // of an expert
  int share;       // tokens of each of its tiles
  int first;       // number of its first tile
};
template <int TOK, int SPLIT> struct Grp {
  static constexpr int STAGES = TOK == 256 ? 4 : TOK == 128 ? 6 : SPLIT > 1 ? 7 : 8, BUFS = 512 / TOK < 4 ? 512 / TOK : 4, COLUMNS = BUFS * TOK;
  static constexpr int B_BYTES = TOK * KBYTES;
  static constexpr int RING = STAGES * (A_BYTES + B_BYTES);
  static constexpr int TABLE = RING + (SPLIT > 1 ? TOK * CHANNELS * 4 : GRP_EPI_WARPS * EPI_BYTES);   // then experts + 1 segments
  static int smem(int experts) { return TABLE + (experts + 1) * (int)sizeof(Segment) + 1024; }
};

struct GroupArgs {
  TokenArgs t;
  const float* xs;
  int32_t *status, *mirror;
  uint32_t max_polls;
  int n_tiles, withhold;
  int most;   // tiles there can be
  int cap;    // tokens of a tile at most, in sixteens: TOK or fewer
  uint32_t by_cap;   // 2^32 / cap rounded up
  int64_t x_stride;
};
struct __align__(16) GroupCtl {
  uint64_t full[8], empty[8], tfull[4], tempty[4], done, ready, freed;
  int abort_flag;
  uint32_t tmem_base, by[RASTER + 1];
  __align__(16) float scale[GRP_EPI_WARPS][EPI_TOKENS];   // of the tokens that a warp takes out, read four at a time
};
static_assert(offsetof(GroupCtl, scale) % 16 == 0, "vector reads");
struct TokenMaps {
  CUtensorMap box[BOXES];   // of 16 << i tokens
};
struct Tile {
  int expert, channel;
  int64_t row;
  int rows, columns;   // tokens, and those rounded up to the MMA's N
};

// Instruction descriptor of kind::i8: D s32, A and B s8, K-major, M = 128.
__device__ __forceinline__ uint32_t mma_desc(int n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(CHANNELS >> 4) << 24); }

// The tokens of a tile come in one or two boxes: one of the next power of two where that is at most a quarter more, else the power of
// two below and one for the rest.
struct Boxes {
  int first, second;   // numbers of maps, second < 0: none
  __device__ __forceinline__ int tokens() const { return (16 << first) + (second < 0 ? 0 : 16 << second); }
};
__device__ __forceinline__ Boxes boxes_of(int columns) {
  const int up = columns <= 16 ? 0 : 32 - __clz((columns - 1) >> 4);   // 16 << up >= columns
  if ((16 << up) * 4 <= columns * 5) return Boxes{up, -1};
  const int rest = columns - (16 << (up - 1));
  return Boxes{up - 1, rest <= 16 ? 0 : 32 - __clz((rest - 1) >> 4)};
}

__device__ __forceinline__ int tiles_of(int rows, const GroupArgs& p) { return (int)__umulhi((uint32_t)(((rows + 15) >> 4) + p.cap - 1), p.by_cap); }

// Divisions by numbers that are not known at compile time cost a tile some 500 cycles, which every role goes through: the quotient
// that the rows of a segment need is in the table, more than one group of token tiles makes a tile long enough, and the last one is a
// multiplication.  by[w]: 2^32 / w rounded up, exact for numbers below 2^28 (16 * channels / 128) and w up to 16.
template <int TOK>
__device__ __forceinline__ Tile tile_of(int t, const GroupArgs& p, const Segment* seg, const uint32_t* by) {
  int lo = 0, hi = p.t.experts;   // seg[lo].first <= t < seg[hi].first; experts without rows have no tiles and are stepped over
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (seg[mid].first <= t) lo = mid;
    else hi = mid;
  }
  const Segment s = seg[lo];
  const int tiles = tiles_of(s.rows, p), local = t - s.first, per_group = RASTER * p.n_tiles;
  const int group = tiles <= RASTER ? 0 : local / per_group, g0 = group * RASTER;
  const int width = tiles - g0 < RASTER ? tiles - g0 : RASTER, at = local - group * per_group;
  const int n = width == 1 ? at : (int)__umulhi((uint32_t)at, by[width]), m = g0 + at - n * width;
  Tile r;
  r.expert = lo;
  r.channel = n * CHANNELS;
  r.row = s.row + (int64_t)m * s.share;
  r.rows = s.rows - m * s.share < s.share ? s.rows - m * s.share : s.share;
  r.columns = (r.rows + 15) & ~15;
  return r;
}

// Waits for arrivals from the cluster's CTAs: what they wrote before them is visible behind it.  Bounded like the others; once the flag is
// set it gives up after one poll.
__device__ __forceinline__ void wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag, uint32_t max_polls) {
  for (uint32_t i = 0; i < max_polls; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok || *abort_flag) return;
  }
  *abort_flag = 1;
}
__device__ __forceinline__ void store_remote(uint32_t at, int v) { asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ int4 load_remote(uint32_t at) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

// SPLIT > 1: the CTAs of a cluster share a tile, each takes its part of K; the int32 sums meet in shared memory (integers: their order does
// not show), and each CTA finishes its share of the tokens.
template <int TOK, int SPLIT>
__global__ void __launch_bounds__(GRP_THREADS, 1)
group_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ TokenMaps map_x, const GroupArgs p) {
  using G = Grp<TOK, SPLIT>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ GroupCtl ctl;
  uint8_t* const smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const uint32_t smem_a = smem_u32(smem), smem_b = smem_a + G::STAGES * A_BYTES;
  Segment* const seg = reinterpret_cast<Segment*>(smem + G::TABLE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &ctl.abort_flag;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_w);
    for (int i = 0; i < BOXES; ++i) prefetch_tensormap(&map_x.box[i]);
    for (int s = 0; s < G::STAGES; ++s) {
      mbar_init(smem_u32(&ctl.full[s]), 1);
      mbar_init(smem_u32(&ctl.empty[s]), 1);
    }
    for (int b = 0; b < G::BUFS; ++b) {
      mbar_init(smem_u32(&ctl.tfull[b]), 1);
      mbar_init(smem_u32(&ctl.tempty[b]), GRP_EPI_WARPS);
    }
    mbar_init(smem_u32(&ctl.done), 1);
    mbar_init(smem_u32(&ctl.ready), SPLIT);
    mbar_init(smem_u32(&ctl.freed), SPLIT);
    ctl.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem_base)), "r"(G::COLUMNS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // The offsets and the weights were there before the chain; only who reads the quantized rows and their scales waits for them.
  for (int e = threadIdx.x; e < p.t.experts; e += GRP_THREADS) {
    int64_t b, n;
    segment(p.t, e, b, n);
    const int count = (int)(n - b), tiles = tiles_of(count, p);
    seg[e].row = (int)b;
    seg[e].rows = count;
    seg[e].share = tiles ? ((count + tiles - 1) / tiles + 15) & ~15 : 0;   // equal tiles rather than full ones and a rest
    seg[e + 1].first = tiles * p.n_tiles;
  }
  if (threadIdx.x >= 2 && threadIdx.x <= RASTER) ctl.by[threadIdx.x] = 0xffffffffu / threadIdx.x + 1;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) {   // running sum of the tiles
    int64_t carry = 0;
    if (lane == 0) seg[0].first = 0;
    for (int e0 = 0; e0 < p.t.experts; e0 += 32) {
      int64_t up = e0 + lane < p.t.experts ? seg[e0 + lane + 1].first : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, up, d);
        if (lane >= d) up += v;
      }
      // More than there can be: offsets that decrease, whose segments overlap.  Nothing is computed then.
      if (e0 + lane < p.t.experts) seg[e0 + lane + 1].first = carry + up <= p.most ? (int)(carry + up) : 0;
      carry += __shfl_sync(0xffffffffu, up, 31);
    }
    if (lane == 0 && carry > p.most) seg[p.t.experts].first = 0;
  }
  __syncthreads();
  if (SPLIT > 1) cluster_sync_all();   // the others' barriers are initialised before anything arrives on them
  const uint32_t tmem_base = ctl.tmem_base;
  const int total = seg[p.t.experts].first, blocks = (int)((p.t.K + KBYTES - 1) / KBYTES);
  const int rank = SPLIT > 1 ? (int)cluster_ctarank() : 0, unit = (int)blockIdx.x / SPLIT, units = (int)gridDim.x / SPLIT;
  const int kb0 = rank * blocks / SPLIT, kb1 = (rank + 1) * blocks / SPLIT;   // this CTA's K blocks

  // Rows of no expert, a warp's share at a time: pieces of 4 KB go round the CTAs and their warps.
  auto clear_dead = [&](int w) {
    const int64_t before = seg[0].row, behind = (int64_t)seg[p.t.experts - 1].row + seg[p.t.experts - 1].rows, dead = before + p.t.rows - behind;
    const int64_t pieces = p.t.N * (p.t.out_f32 ? 4 : 2) / 16, front = before * pieces, all = dead * pieces, skip = (behind - before) * pieces;
    uint4* y = static_cast<uint4*>(p.t.y);
    for (int64_t i0 = ((int64_t)w * gridDim.x + blockIdx.x) * 256; i0 < all; i0 += (int64_t)gridDim.x * CLEAR_WARPS * 256)
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int64_t i = i0 + u * 32 + lane;
        if (i < all) y[i < front ? i : i + skip] = make_uint4(0, 0, 0, 0);
      }
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    const bool elected = elect_one();
    int s = 0;
    uint32_t ph = 0, issued = 0, issued_ph = 0;   // bit s: a load into stage s is (or was) in flight, with parity
    bool ok = true;
    int ahead = 0;   // K blocks of the first tile whose weights are on their way before the rows have been quantized
    if (unit < total && !p.withhold) {
      const Tile tile = tile_of<TOK>(unit, p, seg, ctl.by);
      ahead = kb1 - kb0 < G::STAGES ? kb1 - kb0 : G::STAGES;
      const uint32_t bytes = A_BYTES + boxes_of(tile.columns).tokens() * KBYTES;
      if (elected)
        for (int kb = 0; kb < ahead; ++kb) {
          mbar_expect_tx(smem_u32(&ctl.full[kb]), bytes);
          tma_load_2d(smem_a + kb * A_BYTES, &map_w, smem_u32(&ctl.full[kb]), (kb0 + kb) * KBYTES, (int)((int64_t)tile.expert * p.t.N) + tile.channel);
        }
    }
    chain_wait();
    for (int t = unit; t < total && ok; t += units) {
      const Tile tile = tile_of<TOK>(t, p, seg, ctl.by);
      const int w_row = (int)((int64_t)tile.expert * p.t.N) + tile.channel;
      const Boxes box = boxes_of(tile.columns);
      const uint32_t bytes = A_BYTES + box.tokens() * KBYTES;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = mbar_wait(smem_u32(&ctl.empty[s]), ph ^ 1u, abort_flag, p.max_polls))) break;
        if (p.withhold && t == unit && kb == kb1 - 1) {   // test hook: the waits that depend on this stage run out
          if (++s == G::STAGES) { s = 0; ph ^= 1u; }
          continue;
        }
        if (elected) {
          const uint32_t bar = smem_u32(&ctl.full[s]);
          if (t != unit || kb - kb0 >= ahead) {
            mbar_expect_tx(bar, bytes);
            tma_load_2d(smem_a + s * A_BYTES, &map_w, bar, kb * KBYTES, w_row);
          }
          const uint32_t to = smem_b + s * G::B_BYTES;
          tma_load_2d(to, &map_x.box[box.first], bar, kb * KBYTES, (int)tile.row);
          if (box.second >= 0) tma_load_2d(to + (16 << box.first) * KBYTES, &map_x.box[box.second], bar, kb * KBYTES, (int)tile.row + (16 << box.first));
        }
        issued |= 1u << s;
        issued_ph = (issued_ph & ~(1u << s)) | (ph << s);
        if (++s == G::STAGES) { s = 0; ph ^= 1u; }
      }
    }
    if (!ok) {   // copies in flight land before the CTA's shared memory is released
      for (int k = 0; k < G::STAGES; ++k)
        if (issued & (1u << k)) {
          int dummy = 0;
          mbar_wait(smem_u32(&ctl.full[k]), (issued_ph >> k) & 1u, &dummy, 1u << 15);
        }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    const bool elected = elect_one();
    int s = 0, ab = 0;
    uint32_t ph = 0, aph = 0;
    bool ok = true;
    for (int t = unit; t < total && ok; t += units) {
      const uint32_t idesc = mma_desc(tile_of<TOK>(t, p, seg, ctl.by).columns), d = tmem_base + ab * TOK;
      if (!(ok = mbar_wait(smem_u32(&ctl.tempty[ab]), aph ^ 1u, abort_flag, p.max_polls))) break;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = mbar_wait(smem_u32(&ctl.full[s]), ph, abort_flag, p.max_polls))) break;
        tc_fence_after();
        if (elected) {
          const uint64_t da = smem_desc(smem_a + s * A_BYTES), db = smem_desc(smem_b + s * G::B_BYTES);
#pragma unroll
          for (int k4 = 0; k4 < KBYTES / 32; ++k4) tc_mma_i8(d, da + 2 * k4, db + 2 * k4, idesc, (k4 > 0 || kb > kb0) ? 1u : 0u);
          tc_commit(smem_u32(&ctl.empty[s]));
          if (kb == kb1 - 1) tc_commit(smem_u32(&ctl.tfull[ab]));
        }
        __syncwarp();
        if (++s == G::STAGES) { s = 0; ph ^= 1u; }
      }
      if (++ab == G::BUFS) { ab = 0; aph ^= 1u; }
    }
    if (elected) tc_commit(smem_u32(&ctl.done));   // all MMAs have retired before tensor memory is freed
    __syncwarp();
    int dummy = 0;
    mbar_wait(smem_u32(&ctl.done), 0, &dummy);
  } else if (warp < 4) {
    clear_dead(warp - 2);
  } else {
    // ------------------------------------------------------------------ epilogue
    const int q = warp & 3, group = (warp - 4) >> 2;   // a quarter of the channels, 16 of every 64 tokens
    uint8_t* const turn = smem + G::RING + (warp - 4) * EPI_BYTES;
    constexpr int PARTS = TOK / 64;   // of 16 tokens
    if constexpr (SPLIT > 1) {
      int* const part = reinterpret_cast<int*>(smem + G::RING);   // [tokens, channels]: this CTA's sums
      const uint32_t part_at = smem_u32(part), ready = smem_u32(&ctl.ready), freed = smem_u32(&ctl.freed);
      // Once all of this CTA's epilogue warps are here.  None of them leaves the loop early, so that they all come; a CTA that has given up a
      // wait says so to the others, which store nothing from then on.
      auto arrive_everywhere = [&](uint32_t bar) {
        named_sync(1, GRP_EPI_WARPS * 32);
        if (threadIdx.x - 128 < SPLIT) {
          if (*abort_flag) store_remote(map_to_cta(smem_u32(&ctl.abort_flag), threadIdx.x - 128), 1);
          mbar_arrive_cluster(map_to_cta(bar, threadIdx.x - 128));
        }
      };
      int ab = 0;
      uint32_t aph = 0, ph = 0;
      chain_wait();
      for (int t = unit; t < total; t += units, ph ^= 1u) {
        const Tile tile = tile_of<TOK>(t, p, seg, ctl.by);
        mbar_wait_or_flag(smem_u32(&ctl.tfull[ab]), aph, abort_flag, p.max_polls);
        tc_fence_after();
        wait_cluster(freed, ph ^ 1u, abort_flag, p.max_polls);   // the tile before has been read by all
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
          const int j0 = group * EPI_TOKENS + i * 64;
          if (j0 >= tile.rows) break;
          uint32_t r[EPI_TOKENS];
          tc_ld16(tmem_base + ((uint32_t)(q * 32) << 16) + ab * TOK + j0, r);
          tc_ld_wait();
#pragma unroll
          for (int j = 0; j < EPI_TOKENS; ++j) part[(j0 + j) * CHANNELS + q * 32 + lane] = (int)r[j];
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl.tempty[ab]));
        if (++ab == G::BUFS) { ab = 0; aph ^= 1u; }
        arrive_everywhere(ready);
        wait_cluster(ready, ph, abort_flag, p.max_polls);
        const int from = rank * tile.rows / SPLIT, to = (rank + 1) * tile.rows / SPLIT, n = tile.channel + lane * 4;
        if (n < p.t.N && !*abort_flag) {   // N is a multiple of 8, n of 4
          const int64_t c = (int64_t)tile.expert * p.t.N + n;
          float sw[4], bias[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sw[i] = p.t.ws[c + i];
            bias[i] = p.t.bias ? __bfloat162float(p.t.bias[c + i]) : 0.f;
          }
          for (int j = from + warp - 4; j < to; j += GRP_EPI_WARPS) {
            int sum[4] = {0, 0, 0, 0};
#pragma unroll
            for (int r = 0; r < SPLIT; ++r) {
              const int4 v = load_remote(map_to_cta(part_at + (j * CHANNELS + lane * 4) * 4, r));
              sum[0] += v.x;
              sum[1] += v.y;
              sum[2] += v.z;
              sum[3] += v.w;
            }
            const float sx = p.xs[tile.row + j];
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              v[i] = __fmul_rn(__fmul_rn(__int2float_rn(sum[i]), sx), sw[i]);
              if (p.t.bias) v[i] = __fadd_rn(v[i], bias[i]);
            }
            const int64_t at = (tile.row + j) * p.t.N + n;
            if (p.t.out_f32) *reinterpret_cast<float4*>(static_cast<float*>(p.t.y) + at) = make_float4(v[0], v[1], v[2], v[3]);
            else {
              const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
              *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.t.y) + at) =
                  make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
            }
          }
        }
        arrive_everywhere(freed);
      }
    } else {
    float* const scale = ctl.scale[warp - 4];
    // What a tile needs besides the accumulator: fetched a tile ahead, behind the wait for the one in front.
    struct Ahead {
      Tile tile;
      float sw, bias, token[PARTS];   // scale and bias of the lane's channel, scales of the lane's tokens
    };
    auto fetch = [&](int t) {
      Ahead f;
      f.tile = tile_of<TOK>(t, p, seg, ctl.by);
      const int n = f.tile.channel + q * 32 + lane;
      const int64_t c = (int64_t)f.tile.expert * p.t.N + n;
      f.sw = n < p.t.N ? p.t.ws[c] : 0.f;
      f.bias = n < p.t.N && p.t.bias ? __bfloat162float(p.t.bias[c]) : 0.f;
#pragma unroll
      for (int i = 0; i < PARTS; ++i) {
        const int j = group * EPI_TOKENS + i * 64 + lane;
        f.token[i] = lane < EPI_TOKENS && j < f.tile.rows ? p.xs[f.tile.row + j] : 0.f;
      }
      return f;
    };
    int ab = 0;
    uint32_t aph = 0;
    chain_wait();
    Ahead next;
    if (unit < total) next = fetch(unit);
    for (int t = unit; t < total; t += units) {
      const Ahead now = next;
      if (!mbar_wait(smem_u32(&ctl.tfull[ab]), aph, abort_flag, p.max_polls)) break;
      tc_fence_after();
      if (t + units < total) next = fetch(t + units);
      const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + ab * TOK;
      const int n = now.tile.channel + q * 32 + lane;
      const float2 sw2 = make_float2(now.sw, now.sw);
#pragma unroll
      for (int i = 0; i < PARTS; ++i) {
        const int j0 = group * EPI_TOKENS + i * 64, left = now.tile.rows - j0;
        if (left <= 0) break;
        uint32_t r[EPI_TOKENS];
        tc_ld16(taddr + j0, r);
        if (lane < EPI_TOKENS) scale[lane] = now.token[i];
        __syncwarp();
        tc_ld_wait();
        float2 v[EPI_TOKENS / 2];   // two tokens each
#pragma unroll
        for (int j = 0; j < EPI_TOKENS / 2; j += 2) {
          const float4 sx = *reinterpret_cast<const float4*>(scale + 2 * j);
          v[j] = __fmul2_rn(__fmul2_rn(make_float2(__int2float_rn((int)r[2 * j]), __int2float_rn((int)r[2 * j + 1])), make_float2(sx.x, sx.y)), sw2);
          v[j + 1] = __fmul2_rn(__fmul2_rn(make_float2(__int2float_rn((int)r[2 * j + 2]), __int2float_rn((int)r[2 * j + 3])), make_float2(sx.z, sx.w)), sw2);
        }
        if (p.t.bias) {
#pragma unroll
          for (int j = 0; j < EPI_TOKENS / 2; ++j) v[j] = make_float2(__fadd_rn(v[j].x, now.bias), __fadd_rn(v[j].y, now.bias));
        }
        const int64_t row = now.tile.row + j0;
        if (p.t.out_f32) {
          float* y = static_cast<float*>(p.t.y) + row * p.t.N + n;
          if (n < p.t.N) {
#pragma unroll
            for (int j = 0; j < EPI_TOKENS / 2; ++j) {
              if (2 * j < left) y[2 * j * p.t.N] = v[j].x;
              if (2 * j + 1 < left) y[(2 * j + 1) * p.t.N] = v[j].y;
            }
          }
          __syncwarp();   // the scales have been read
        } else {
          uint32_t* words = reinterpret_cast<uint32_t*>(turn);   // [pairs of tokens, channels]
#pragma unroll
          for (int j = 0; j < EPI_TOKENS / 2; ++j) {
            const __nv_bfloat162 w = __floats2bfloat162_rn(v[j].x, v[j].y);
            words[j * 32 + lane] = *reinterpret_cast<const uint32_t*>(&w);
          }
          __syncwarp();
          const int pair = lane >> 2, piece = lane & 3, n8 = now.tile.channel + q * 32 + piece * 8;
          const uint4 lo = *reinterpret_cast<const uint4*>(words + pair * 32 + piece * 8), hi = *reinterpret_cast<const uint4*>(words + pair * 32 + piece * 8 + 4);
          __nv_bfloat16* y = static_cast<__nv_bfloat16*>(p.t.y) + (row + 2 * pair) * p.t.N + n8;
          if (n8 < p.t.N) {
            if (2 * pair < left)
              *reinterpret_cast<uint4*>(y) = make_uint4(__byte_perm(lo.x, lo.y, 0x5410), __byte_perm(lo.z, lo.w, 0x5410), __byte_perm(hi.x, hi.y, 0x5410), __byte_perm(hi.z, hi.w, 0x5410));
            if (2 * pair + 1 < left)
              *reinterpret_cast<uint4*>(y + p.t.N) = make_uint4(__byte_perm(lo.x, lo.y, 0x7632), __byte_perm(lo.z, lo.w, 0x7632), __byte_perm(hi.x, hi.y, 0x7632), __byte_perm(hi.z, hi.w, 0x7632));
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl.tempty[ab]));
      if (++ab == G::BUFS) { ab = 0; aph ^= 1u; }
    }
    }
    clear_dead(warp - 2);
  }
  tc_fence_before();
  __syncthreads();
  if (SPLIT > 1) cluster_sync_all();   // shared memory and barriers outlive the others' use of them
  if (threadIdx.x == 0 && ctl.abort_flag && p.status) {
    atomicExch(p.status, I8L_ERR_TIMEOUT);
    if (p.mirror) {
      __threadfence_system();   // who sees the mirror finds the word set
      *static_cast<volatile int32_t*>(p.mirror) = I8L_ERR_TIMEOUT;
    }
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(G::COLUMNS) : "memory");
  }
}

// ------------------------------------------------------------------------------------------ host
int64_t few_row_bytes(int64_t rows, int64_t K) { return rows <= 4 ? K : (K + MMA_K - 1) / MMA_K * MMA_K; }
// Whether the kernels for few rows take them.  Weights from memory, us here and on the tensor cores:
//   Every block quantizes all rows into its shared memory, 256 threads for as many as the next power of two: that many times K is at most
//   2^15.  One row x 4096x24576 21.0 and 26.3, x 1024x49152 26.4 and 22.6; two x 2048x16384 13.7 and 14.5, x 1024x40960 28.3 and 20.1;
//   four x 2048x8192 9.6 and 11.3, x 2048x11008 12.9 and 12.3; eight x 2048x4096 8.1 and 9.3, x 2048x6144 10.9 and 10.2, x 1024x11008 22.8
//   and 10.1.
//   Weights, of as many experts as the rows allow: 3 or 4 rows up to 40 MB, 4 x 8192x4096 11.8 and 12.9, x 11008x4096 14.1 and 13.4, 4 experts of
//   2048x4096 11.6 and 13.7, of 4096x4096 18.0 and 16.4, 3 of 5040x5984 24.7 and 20.0, but any number where K is short, 4 of 8192x2048
//   14.9 and 17.0; 5 to 8 rows up to 24 MB, 8 x 5120x4096 11.7 and 11.7, x 6144x4096 12.6 and 12.3, x 8192x4096 14.7 and 13.6.
//   5 to 8 rows of several experts, E if they are as many as the rows allow: an expert's channels are gone through once more by all blocks and
//   its rows fill less of the instructions, E * E * N up to 12 K.  8 rows, 2 experts of 2048x2048 8.5 and 9.1, of 4096x2048 10.6
//   and 9.7; 8 of 256x1024 6.6 and 7.3, of 512x1024 8.6 and 7.5; 5 rows, 5 experts of 512x1024 6.5 and 7.4, of 2048x1024 9.0 and 8.1.
// Over 90 sizes the choice costs 1 % against the better one, 10 % at most.
bool few_rows(int64_t rows, int64_t K, int64_t experts, int64_t N) {
  const int64_t padded = rows <= 2 ? rows : rows <= 4 ? 4 : 8, segments = experts < rows ? experts : rows;
  if (rows > FEW_ROWS || padded * K > 1 << 15) return false;
  if (rows <= 4) return rows <= 2 || K <= 2048 || segments * N * K <= 40 << 20;
  return segments == 1 ? N * K <= 24 << 20 : segments * segments * N <= 12 << 10;
}
template <typename Kernel, typename... Args>
int launch_few(Kernel kernel, const TokenArgs& a, int64_t channels, int warps, cudaStream_t st, Args... args) {
  const int64_t segments = a.experts < a.rows ? a.experts : a.rows, units = segments * ((a.N + channels - 1) / channels);
  const int64_t blocks = (units + warps - 1) / warps, budget = gemm_cta_budget();
  const int64_t resident = budget < sm_count() ? budget : 2 * sm_count();   // under a limit no more CTAs than it says
  const LaunchChain chain(st);
  (void)chain_first();   // it always waits
  I8L_CUDA_OK(launch(kernel, dim3((unsigned)(blocks < resident ? blocks : resident)), FEW_THREADS, (size_t)(a.rows * few_row_bytes(a.rows, a.K)), st,
                     a, args...));
  return I8L_OK;
}
int run_few(const TokenArgs& a, cudaStream_t st) {
  if (a.rows == 1) return launch_few(few_dp_kernel<1>, a, DP_CHANNELS, FEW_WARPS, st);
  if (a.rows == 2) return launch_few(few_dp_kernel<2>, a, DP_CHANNELS, FEW_WARPS, st);
  if (a.rows <= 4) return launch_few(few_dp_kernel<4>, a, DP_CHANNELS, FEW_WARPS, st);
  return launch_few(few_mma_kernel, a, MMA_CHANNELS, 1, st, (int)few_row_bytes(a.rows, a.K));
}

// Most tokens of a tile, from what the host knows: as if all rows belonged to experts, and to all alike.  A tile of s columns takes 0.4 + 0.6 *
// s / 256 of a full one (less for the MMAs, as much for the weights and the rest), and up to three waves of tiles end with the
// slowest.  us with 64, 128 and 256: dense 4096x4096 of 256 rows 13.3 / 13.9 / 16.0, 512 20.8 / 14.8 / 17.3, 1000 36 / 24 / 19.0;
// 64 experts of 1408x4096 with 32 rows each 70 / 68 / 73, 100 100 / 88 / 92, 500 377 / 258 / 223.  Over 100 sizes the choice costs
// 0.3 % against the best one, 8 % at most.  Where there is one segment the tiles are known, and any multiple of 16 from 64 on may fill the
// waves better: 439 rows x 9688x7280 48.9 -> 44.3 (160 for 256), 970 x 4768x4096 27.6 -> 25.3, 1705 x 1472x4096 20.0 -> 18.4 (144).
int tile_tokens(const TokenArgs& a) {
  const int64_t segments = a.experts < a.rows ? a.experts : a.rows, average = (a.rows + segments - 1) / segments;
  const int64_t n_tiles = (a.N + CHANNELS - 1) / CHANNELS;
  const int sms = gemm_cta_budget();
  int best = 0;
  double least = 0;
  for (int t = 64; t <= 256; t = segments == 1 ? t + 16 : t * 2) {
    double per = 1;   // tiles of a segment; uneven ones need half a tile more than their average
    if (segments == 1) per = (double)((average + t - 1) / t);
    else if (average * 4 > t * 3) per = (double)average / t + 0.5;
    if (per < 1) per = 1;
    int64_t share = ((average + (int64_t)per - 1) / (int64_t)per + 15) / 16 * 16;
    if (share > t) share = t;
    const double tiles = (double)segments * per * (double)n_tiles, waves = tiles / sms;
    const double cost = (segments == 1 || waves < 3 ? (double)(((int64_t)tiles + sms - 1) / sms) : waves + 0.5) * (0.4 + 0.6 * (double)share / 256);
    if (!best || cost < least) {
      best = t;
      least = cost;
    }
  }
  return best;
}

// CTAs that share a tile of 64 tokens, where there are few tiles and a long K: a share costs 2 us (the sums meet, clusters start later) and
// saves its part of 0.17 us a K block; clusters of eight find few places, and 32 of four nearly all that there are.  us with 1, 2, 4
// and 8: 9 rows x 512x8192 17.9 / 13.7 / 11.4 / 10.0, 256 rows 20.6 / 16.4 / 13.5 / 20.0; 16 rows x 4096x11008 23.6 / 17.8 / 16.0 /
// 23.4, 128 rows 25.5 / 19.6 / 27.1 / 36.2; 64 rows x 4096x4096 13.9 / 13.5 / 14.7 / 20.6, x 4096x2048 10.5 / 11.4 / 13.1 / 19.2,
// x 1000x2048 9.3 / 9.7 / 9.0 / 8.6, x 2176x1408 8.3 / 9.5 / 8.8 / 15.1.  9 rows x 4096x4096 lose by it: 12.7, and 11.8 with four.
int k_split(const TokenArgs& a) {
  const int64_t segments = a.experts < a.rows ? a.experts : a.rows, average = (a.rows + segments - 1) / segments;
  const int64_t tiles = segments * ((average + 63) / 64) * ((a.N + CHANNELS - 1) / CHANNELS), blocks = (a.K + KBYTES - 1) / KBYTES;
  if (gemm_cta_budget() < sm_count()) return 1;   // some SMs are kept free, and clusters need whole groups of them
  if (blocks >= 16 && tiles <= 8) return 8;
  if (blocks >= 16 && tiles <= 16) return 4;
  if (blocks >= 64 && tiles <= 32) return 4;
  return blocks >= 24 && tiles <= 64 ? 2 : 1;
}

template <int TOK, int SPLIT = 1> int launch_group(const int8_t* xq, GroupArgs& p, cudaStream_t st) {
  using G = Grp<TOK, SPLIT>;
  static std::atomic<int> allowed[MAX_SMEM_DEVICES];
  const TokenArgs& a = p.t;
  I8L_CUDA_OK(allow_smem(group_kernel<TOK, SPLIT>, allowed, G::smem(MAX_EXPERTS)));
  p.n_tiles = (int)((a.N + CHANNELS - 1) / CHANNELS);
  const int64_t most = (a.rows / (16 * p.cap) + (a.experts < a.rows ? a.experts : a.rows)) * p.n_tiles;   // tiles, whatever the offsets
  if (most >= (1ll << 31)) return fail(I8L_ERR_SHAPE, "i8l_token_linear: too large for 32-bit tile numbers");
  p.most = (int)most;
  CUtensorMap mw;
  TokenMaps mx;
  if (int e = make_tile_map_i8(&mw, a.wq, a.experts * a.N, a.K, a.K, CHANNELS)) return e;
  for (int i = 0; i < BOXES; ++i)
    if (int e = make_tile_map_i8(&mx.box[i], xq, a.rows, a.K, p.x_stride, 16 << i)) return e;
  const int64_t budget = gemm_cta_budget() / SPLIT > 0 ? gemm_cta_budget() / SPLIT : 1;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attrs[2];
  cfg.gridDim = dim3((unsigned)((most < budget ? most : budget) * SPLIT), 1, 1);
  cfg.blockDim = dim3(GRP_THREADS, 1, 1);
  cfg.dynamicSmemBytes = G::smem(a.experts);
  cfg.stream = st;
  if (SPLIT > 1) {
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.x = SPLIT;
    attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = 1;
  }
  chain_attribute(cfg, attrs);
  I8L_CUDA_OK(cudaLaunchKernelEx(&cfg, group_kernel<TOK, SPLIT>, mw, mx, p));
  return I8L_OK;
}

}  // namespace
}  // namespace i8l

using namespace i8l;

// Bytes from one quantized row to the next: whole lines, so that the tiles' copies do not straddle them (5717
// rows x 1112x10992 140 -> 104 us, 16484 x 16 experts of 2016x3088 161 -> 128), but for rows that are quantized in two sweeps.
static int64_t row_stride(int64_t K) { return K <= 16384 ? (K + 127) / 128 * 128 : K; }

extern "C" int64_t i8l_token_linear_workspace(int64_t rows, int experts, int64_t N, int64_t K) {
  if (rows <= 0 || K <= 0 || N <= 0 || experts <= 0 || rows > MAX_ROWS || N >= (1ll << 31) || K > MAX_K || few_rows(rows, K, experts, N)) return 0;
  return (rows * row_stride(K) + 255) / 256 * 256 + (4 * rows + 255) / 256 * 256;
}

extern "C" int i8l_token_linear(const void* x, const int8_t* w_q, const float* w_scale, const int32_t* offsets, const void* bias, void* y,
                                int64_t rows, int experts, int64_t N, int64_t K, int flags, void* workspace, int64_t workspace_bytes,
                                int32_t* status, void* stream) {
  if (rows < 0 || rows > MAX_ROWS || N < 8 || N % 8 || K < 16 || K % 16 || K > MAX_K || N >= (1ll << 31))
    return fail(I8L_ERR_SHAPE, "i8l_token_linear: rows=%lld N=%lld K=%lld: N a multiple of 8, K of 16 and at most %lld", (long long)rows,
                (long long)N, (long long)K, (long long)MAX_K);
  if (experts < 1 || experts > MAX_EXPERTS || (!offsets && experts != 1) || experts * N >= (1ll << 31))
    return fail(I8L_ERR_SHAPE, "i8l_token_linear: %d experts, 1 to %d are possible, and one without offsets", experts, MAX_EXPERTS);
  if (flags & ~I8L_GEMM_OUT_F32) return fail(I8L_ERR_ARG, "i8l_token_linear: unknown flags %d", flags);
  if (!w_q || !w_scale || (rows && (!x || !y))) return fail(I8L_ERR_ARG, "i8l_token_linear: null pointer");
  if (!aligned16(x) || !aligned16(w_q) || !aligned16(y) || !aligned16(bias) || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return fail(I8L_ERR_ALIGN, "i8l_token_linear: x, w_q, y and bias must be 16-byte aligned, the workspace 256-byte");
  if ((reinterpret_cast<uintptr_t>(w_scale) | reinterpret_cast<uintptr_t>(offsets) | reinterpret_cast<uintptr_t>(status)) & 3)
    return fail(I8L_ERR_ALIGN, "i8l_token_linear: w_scale, offsets and status are aligned to their elements");
  const int64_t need = i8l_token_linear_workspace(rows, experts, N, K);
  if (need && (!workspace || workspace_bytes < need))
    return fail(I8L_ERR_ARG, "i8l_token_linear: workspace of %lld bytes is too small", (long long)workspace_bytes);
  if (!rows) return I8L_OK;
  if (int e = check_arch()) return e;
  TokenArgs a{};
  a.x = static_cast<const __nv_bfloat16*>(x); a.wq = w_q; a.ws = w_scale; a.offsets = offsets;
  a.bias = static_cast<const __nv_bfloat16*>(bias); a.y = y;
  a.rows = rows; a.N = N; a.K = K; a.experts = experts; a.out_f32 = (flags & I8L_GEMM_OUT_F32) ? 1 : 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (few_rows(rows, K, experts, N)) return run_few(a, st);
  int8_t* xq = static_cast<int8_t*>(workspace);
  float* xs = reinterpret_cast<float*>(xq + (rows * row_stride(K) + 255) / 256 * 256);
  const LaunchChain chain(st);
  if (int e = quant_token_rows(x, rows, K, xq, row_stride(K), xs, offsets ? offsets + experts : nullptr, st)) return e;
  (void)chain_first();
  GroupArgs p{};
  p.t = a;
  p.xs = xs;
  p.x_stride = row_stride(K);
  p.status = status;
  p.mirror = status ? mirror_of(status) : nullptr;
  p.max_polls = gemm_wait_limit();
  p.withhold = gemm_withhold();
  const int tok = tile_tokens(a);
  p.cap = tok / 16;
  p.by_cap = 0xffffffffu / p.cap + 1;
  if (tok == 64) switch (k_split(a)) {
      case 8: return launch_group<64, 8>(xq, p, st);
      case 4: return launch_group<64, 4>(xq, p, st);
      case 2: return launch_group<64, 2>(xq, p, st);
    }
  if (tok == 64) return launch_group<64>(xq, p, st);
  return tok <= 128 ? launch_group<128>(xq, p, st) : launch_group<256>(xq, p, st);
}

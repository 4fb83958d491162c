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
// Up to eight rows in one launch: every block quantizes them into its shared memory, then its warps go through the channels of the
// experts that have rows, two at a time, and multiply the weights by dp4a.  Bound by the weights' bytes, so it is the loads that
// matter: while a warp works on a batch (2 KB of each of its two channels, eight loads of 16 bytes a lane) the next one is in flight,
// across channels and experts, and the first goes out ahead of the quantization.
constexpr int FEW_THREADS = 256, FEW_WARPS = FEW_THREADS / 32, FEW_COLS = 2, FEW_STEPS = 4, FEW_BATCH = FEW_STEPS * 512, FEW_ROWS = 8;

struct FewSegment {
  int expert, row, rows;
};
struct Batch {
  uint4 w[FEW_COLS][FEW_STEPS];
};
template <int MT, int CT>
__device__ __forceinline__ void multiply_batch(int (&acc)[FEW_COLS][MT], const Batch& w, const int8_t* rows, int count, int K, int limit, int k0) {
  int at[CT];   // of a row: CT may be above their number, and what is multiplied with the first one once more is not used
#pragma unroll
  for (int t = 0; t < CT; ++t) at[t] = t < count ? t * K : 0;
#pragma unroll
  for (int s = 0; s < FEW_STEPS; ++s) {
    const int k = k0 + s * 512;
    if (k >= limit) break;
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      const uint4 v = *reinterpret_cast<const uint4*>(rows + at[t] + k);
#pragma unroll
      for (int j = 0; j < FEW_COLS; ++j) {
        acc[j][t] = __dp4a((int)w.w[j][s].x, (int)v.x, acc[j][t]);
        acc[j][t] = __dp4a((int)w.w[j][s].y, (int)v.y, acc[j][t]);
        acc[j][t] = __dp4a((int)w.w[j][s].z, (int)v.z, acc[j][t]);
        acc[j][t] = __dp4a((int)w.w[j][s].w, (int)v.w, acc[j][t]);
      }
    }
  }
}

template <int MT>
__global__ void __launch_bounds__(FEW_THREADS, 2) few_rows_kernel(const TokenArgs a) {
  extern __shared__ __align__(16) int8_t xq[];   // [MT, K]
  __shared__ float xs[MT], red[FEW_WARPS];
  __shared__ FewSegment s_seg[FEW_ROWS];
  __shared__ int s_segments;
  constexpr int LANES = FEW_THREADS / MT;        // threads that quantize a row
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = (int)a.K;
  if (a.offsets) {   // the experts that have rows, at most as many as rows
    if (warp == 0) {
      int count = 0;
      for (int e0 = 0; e0 < a.experts; e0 += 32) {
        int64_t begin = 0, end = 0;
        if (e0 + lane < a.experts) segment(a, e0 + lane, begin, end);
        const unsigned set = __ballot_sync(0xffffffffu, end > begin);
        const int at = count + __popc(set & ((1u << lane) - 1));
        if (end > begin && at < FEW_ROWS) s_seg[at] = FewSegment{e0 + lane, (int)begin, (int)(end - begin)};
        count += __popc(set);
      }
      if (lane == 0) s_segments = count < FEW_ROWS ? count : FEW_ROWS;   // more only where offsets decrease
    }
  } else if (tid == 0) {
    s_seg[0] = FewSegment{0, 0, (int)a.rows};
    s_segments = 1;
  }
  __syncthreads();

  // Where a warp is: channels n and n + 1 of segment `seg`, K from k on.
  const int64_t step = (int64_t)gridDim.x * FEW_WARPS * FEW_COLS;
  struct Place {
    int seg, k;
    int64_t n;
  };
  const int segments = s_segments;
  auto settle = [&](Place& p) {   // into the segment that its channels belong to
    while (p.seg < segments && p.n >= a.N) {
      p.n -= a.N;
      ++p.seg;
    }
  };
  auto load = [&](Batch& b, const Place& p) {
    if (p.seg >= segments) return;
    const int8_t* w = a.wq + ((int64_t)s_seg[p.seg].expert * a.N + p.n) * a.K + lane * 16;
#pragma unroll
    for (int s = 0; s < FEW_STEPS; ++s)
#pragma unroll
      for (int j = 0; j < FEW_COLS; ++j)
        if (p.k + s * 512 + lane * 16 < K) b.w[j][s] = load_weights(w + (int64_t)j * K + p.k + s * 512);
  };
  Place now{0, 0, ((int64_t)warp * gridDim.x + blockIdx.x) * FEW_COLS};
  settle(now);
  Batch even, odd;
  load(even, now);

  {   // the rows in int8, a scale each
    const int t = tid / LANES, l = tid & (LANES - 1);
    const bool live = t < a.rows;
    const uint4* row = reinterpret_cast<const uint4*>(a.x + t * a.K);
    float m = 0.f;
    if (live)
#pragma unroll 4
      for (int c = l; c < K / 8; c += LANES) {
        float v[8];
        unpack8(row[c], v);
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) red[warp] = m;
    __syncthreads();
    m = red[t * (LANES / 32)];
#pragma unroll
    for (int i = 1; i < LANES / 32; ++i) m = fmaxf(m, red[t * (LANES / 32) + i]);
    float s, stored;
    make_scale<I8L_QMODE_ROWRCP>(m, s, stored);
    if (l == 0) xs[t] = stored;
    uint2* q = reinterpret_cast<uint2*>(xq + t * K);
#pragma unroll 4
    for (int c = l; c < K / 8; c += LANES) q[c] = live ? quant_piece<I8L_QMODE_ROWRCP>(row[c], s) : make_uint2(0, 0);
    __syncthreads();
  }

  int acc[FEW_COLS][MT];
#pragma unroll
  for (int j = 0; j < FEW_COLS; ++j)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[j][t] = 0;
  auto work = [&](Batch& mine, Batch& ahead) {
    Place next = now;
    next.k += FEW_BATCH;
    const bool last = next.k >= K;
    if (last) {
      next.k = 0;
      next.n += step;
      settle(next);
    }
    load(ahead, next);
    const FewSegment seg = s_seg[now.seg];
    const int8_t* rows = xq + (int64_t)seg.row * K + lane * 16;
    const int limit = K - lane * 16;   // of k, so that the lane's 16 bytes are inside the row
    if (MT == 1 || seg.rows == 1) multiply_batch<MT, 1>(acc, mine, rows, seg.rows, K, limit, now.k);
    else if (MT == 2 || seg.rows == 2) multiply_batch<MT, MT < 2 ? MT : 2>(acc, mine, rows, seg.rows, K, limit, now.k);
    else if (MT == 4 || seg.rows <= 4) multiply_batch<MT, MT < 4 ? MT : 4>(acc, mine, rows, seg.rows, K, limit, now.k);
    else multiply_batch<MT, MT>(acc, mine, rows, seg.rows, K, limit, now.k);
    if (last) {
      int sum = 0;   // lane j * MT + t has that of channel j and row t
#pragma unroll
      for (int j = 0; j < FEW_COLS; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const int all = __reduce_add_sync(0xffffffffu, acc[j][t]);
          if (lane == j * MT + t) sum = all;
          acc[j][t] = 0;
        }
      const int j = lane / MT, t = lane % MT;
      if (j < FEW_COLS && t < seg.rows) {
        const int64_t c = (int64_t)seg.expert * a.N + now.n + j, at = (int64_t)(seg.row + t) * a.N + now.n + j;
        float v = __fmul_rn(__fmul_rn(__int2float_rn(sum), xs[seg.row + t]), a.ws[c]);
        if (a.bias) v = __fadd_rn(v, __bfloat162float(a.bias[c]));
        if (a.out_f32) static_cast<float*>(a.y)[at] = v;
        else static_cast<__nv_bfloat16*>(a.y)[at] = __float2bfloat16_rn(v);
      }
    }
    now = next;
  };
  while (now.seg < segments) {
    work(even, odd);
    if (now.seg >= segments) break;
    work(odd, even);
  }
  if (a.offsets) {   // rows of no expert
    const int64_t pieces = a.N * (a.out_f32 ? 4 : 2) / 16;
    for (int64_t r = 0; r < a.rows; ++r) {
      bool some = false;
      for (int i = 0; i < segments; ++i) some |= r >= s_seg[i].row && r < s_seg[i].row + s_seg[i].rows;
      if (some) continue;
      for (int64_t c = (int64_t)blockIdx.x * FEW_THREADS + tid; c < pieces; c += (int64_t)gridDim.x * FEW_THREADS)
        static_cast<uint4*>(a.y)[r * pieces + c] = make_uint4(0, 0, 0, 0);
    }
  }
}

// ------------------------------------------------------------------------------------------ many rows
// The tensor cores with the operands exchanged: 128 output channels are the rows of an MMA and up to TOK tokens its columns, whose
// number is the instruction's N and may be any multiple of 16.  A segment of 17 rows costs 32 columns that way, where tokens as
// MMA rows would cost 128, and the weights, which bound the product until a segment has some hundred rows, are read once.
//
// Persistent, a CTA per SM, 384 threads: warp 0 brings K blocks of 128 bytes by TMA (128 weight rows and the tokens of the tile) into a
// ring, warp 1 issues tcgen05.mma kind::i8 into one of several accumulators in tensor memory, warps 4 to 11 take a finished one
// out: a lane is a channel there, a register a token, so a bf16 tile is turned in shared memory and leaves 16 bytes a lane.
// Warps 2 and 3 clear the rows of no expert.  Tiles come from the offsets in device memory: nothing waits for the host.
// All waits are bounded, as in gemm.cu: on expiry every role leaves, the status word says so.
constexpr int GRP_THREADS = 384, GRP_EPI_WARPS = 8, CHANNELS = 128, KBYTES = 128;
constexpr int A_BYTES = CHANNELS * KBYTES;
constexpr int BOXES = 5;   // maps of 16, 32, 64, 128 and 256 tokens
constexpr int EPI_BYTES = 32 * 32 * 2;        // 32 tokens x 32 channels in bf16
constexpr int RASTER = 16;                    // token tiles whose rows should stay in L2 while the channels are gone through

struct __align__(16) Segment {
  int row, rows;   // of an expert
  int share;       // tokens of each of its tiles
  int first;       // number of its first tile
};
template <int TOK> struct Grp {
  static constexpr int STAGES = TOK == 256 ? 4 : TOK == 128 ? 6 : 8, BUFS = 512 / TOK < 4 ? 512 / TOK : 4, COLUMNS = BUFS * TOK;
  static constexpr int B_BYTES = TOK * KBYTES;
  static constexpr int RING = STAGES * (A_BYTES + B_BYTES);
  static constexpr int TABLE = RING + GRP_EPI_WARPS * EPI_BYTES;   // then experts + 1 segments
  static int smem(int experts) { return TABLE + (experts + 1) * (int)sizeof(Segment) + 1024; }
};

struct GroupArgs {
  TokenArgs t;
  const float* xs;
  int32_t *status, *mirror;
  uint32_t max_polls;
  int n_tiles, withhold;
};
struct __align__(16) GroupCtl {
  uint64_t full[8], empty[8], tfull[4], tempty[4], done;
  int abort_flag;
  uint32_t tmem_base, by[RASTER + 1];
  __align__(16) float scale[GRP_EPI_WARPS][32];   // of the tokens that a warp takes out, read four at a time
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
  const int tiles = (s.rows + TOK - 1) / TOK, local = t - s.first, per_group = RASTER * p.n_tiles;
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

template <int TOK>
__global__ void __launch_bounds__(GRP_THREADS, 1)
group_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ TokenMaps map_x, const GroupArgs p) {
  using G = Grp<TOK>;
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
    const int count = (int)(n - b), tiles = (count + TOK - 1) / TOK;
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
    int carry = 0;
    if (lane == 0) seg[0].first = 0;
    for (int e0 = 0; e0 < p.t.experts; e0 += 32) {
      int up = e0 + lane < p.t.experts ? seg[e0 + lane + 1].first : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, up, d);
        if (lane >= d) up += v;
      }
      if (e0 + lane < p.t.experts) seg[e0 + lane + 1].first = carry + up;
      carry += __shfl_sync(0xffffffffu, up, 31);
    }
  }
  __syncthreads();
  const uint32_t tmem_base = ctl.tmem_base;
  const int total = seg[p.t.experts].first, KB = (int)((p.t.K + KBYTES - 1) / KBYTES);

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    const bool elected = elect_one();
    int s = 0;
    uint32_t ph = 0, issued = 0, issued_ph = 0;   // bit s: a load into stage s is (or was) in flight, with parity
    bool ok = true;
    int ahead = 0;   // K blocks of the first tile whose weights are on their way before the rows have been quantized
    if ((int)blockIdx.x < total && !p.withhold) {
      const Tile tile = tile_of<TOK>(blockIdx.x, p, seg, ctl.by);
      ahead = KB < G::STAGES ? KB : G::STAGES;
      const uint32_t bytes = A_BYTES + boxes_of(tile.columns).tokens() * KBYTES;
      if (elected)
        for (int kb = 0; kb < ahead; ++kb) {
          mbar_expect_tx(smem_u32(&ctl.full[kb]), bytes);
          tma_load_2d(smem_a + kb * A_BYTES, &map_w, smem_u32(&ctl.full[kb]), kb * KBYTES, (int)((int64_t)tile.expert * p.t.N) + tile.channel);
        }
    }
    chain_wait();
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      const Tile tile = tile_of<TOK>(t, p, seg, ctl.by);
      const int w_row = (int)((int64_t)tile.expert * p.t.N) + tile.channel;
      const Boxes box = boxes_of(tile.columns);
      const uint32_t bytes = A_BYTES + box.tokens() * KBYTES;
      for (int kb = 0; kb < KB; ++kb) {
        if (!(ok = mbar_wait(smem_u32(&ctl.empty[s]), ph ^ 1u, abort_flag, p.max_polls))) break;
        if (p.withhold && t == (int)blockIdx.x && kb == KB - 1) {   // test hook: the waits that depend on this stage run out
          if (++s == G::STAGES) { s = 0; ph ^= 1u; }
          continue;
        }
        if (elected) {
          const uint32_t bar = smem_u32(&ctl.full[s]);
          if (t != (int)blockIdx.x || kb >= ahead) {
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
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      const uint32_t idesc = mma_desc(tile_of<TOK>(t, p, seg, ctl.by).columns), d = tmem_base + ab * TOK;
      if (!(ok = mbar_wait(smem_u32(&ctl.tempty[ab]), aph ^ 1u, abort_flag, p.max_polls))) break;
      for (int kb = 0; kb < KB; ++kb) {
        if (!(ok = mbar_wait(smem_u32(&ctl.full[s]), ph, abort_flag, p.max_polls))) break;
        tc_fence_after();
        if (elected) {
          const uint64_t da = smem_desc(smem_a + s * A_BYTES), db = smem_desc(smem_b + s * G::B_BYTES);
#pragma unroll
          for (int k4 = 0; k4 < KBYTES / 32; ++k4) tc_mma_i8(d, da + 2 * k4, db + 2 * k4, idesc, (k4 > 0 || kb > 0) ? 1u : 0u);
          tc_commit(smem_u32(&ctl.empty[s]));
          if (kb == KB - 1) tc_commit(smem_u32(&ctl.tfull[ab]));
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
    // ------------------------------------------------------------------ rows of no expert
    const int64_t before = seg[0].row, behind = (int64_t)seg[p.t.experts - 1].row + seg[p.t.experts - 1].rows, dead = before + p.t.rows - behind;
    const int64_t pieces = p.t.N * (p.t.out_f32 ? 4 : 2) / 16;
    for (int64_t i = (int64_t)blockIdx.x * 64 + threadIdx.x - 64; i < dead * pieces; i += (int64_t)gridDim.x * 64) {
      const int64_t r = i / pieces;
      static_cast<uint4*>(p.t.y)[(r < before ? r : behind + r - before) * pieces + i - r * pieces] = make_uint4(0, 0, 0, 0);
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    const int q = warp & 3, half = (warp - 4) >> 2;   // a quarter of the channels, every other 32 tokens
    uint8_t* const turn = smem + G::RING + (warp - 4) * EPI_BYTES;
    float* const scale = ctl.scale[warp - 4];
    constexpr int PARTS = TOK / 64;   // of 32 tokens
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
        const int j = half * 32 + i * 64 + lane;
        f.token[i] = j < f.tile.rows ? p.xs[f.tile.row + j] : 0.f;
      }
      return f;
    };
    int ab = 0;
    uint32_t aph = 0;
    chain_wait();
    Ahead next;
    if ((int)blockIdx.x < total) next = fetch(blockIdx.x);
    for (int t = blockIdx.x; t < total; t += gridDim.x) {
      const Ahead now = next;
      if (!mbar_wait(smem_u32(&ctl.tfull[ab]), aph, abort_flag, p.max_polls)) break;
      tc_fence_after();
      if (t + (int)gridDim.x < total) next = fetch(t + gridDim.x);
      const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16) + ab * TOK;
      const int n = now.tile.channel + q * 32 + lane;
#pragma unroll
      for (int i = 0; i < PARTS; ++i) {
        const int j0 = half * 32 + i * 64, left = now.tile.rows - j0;
        if (left <= 0) break;
        uint32_t r[32];
        tc_ld16(taddr + j0, r);
        tc_ld16(taddr + j0 + 16, r + 16);
        scale[lane] = now.token[i];
        __syncwarp();
        tc_ld_wait();
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 sx = *reinterpret_cast<const float4*>(scale + j);
          v[j] = __fmul_rn(__fmul_rn(__int2float_rn((int)r[j]), sx.x), now.sw);
          v[j + 1] = __fmul_rn(__fmul_rn(__int2float_rn((int)r[j + 1]), sx.y), now.sw);
          v[j + 2] = __fmul_rn(__fmul_rn(__int2float_rn((int)r[j + 2]), sx.z), now.sw);
          v[j + 3] = __fmul_rn(__fmul_rn(__int2float_rn((int)r[j + 3]), sx.w), now.sw);
        }
        if (p.t.bias) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __fadd_rn(v[j], now.bias);
        }
        const int64_t row = now.tile.row + j0;
        if (p.t.out_f32) {
          float* y = static_cast<float*>(p.t.y) + row * p.t.N + n;
          if (n < p.t.N) {
            if (left >= 32) {
#pragma unroll
              for (int j = 0; j < 32; ++j) y[j * p.t.N] = v[j];
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (j < left) y[j * p.t.N] = v[j];
            }
          }
          __syncwarp();   // the scales have been read
        } else {
          __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(turn) + lane;
#pragma unroll
          for (int j = 0; j < 32; ++j) to[j * 32] = __float2bfloat16_rn(v[j]);
          __syncwarp();
          const int piece = lane & 3, n8 = now.tile.channel + q * 32 + piece * 8;
          __nv_bfloat16* y = static_cast<__nv_bfloat16*>(p.t.y) + (row + (lane >> 2)) * p.t.N + n8;
#pragma unroll
          for (int i8 = 0; i8 < 4; ++i8) {
            const int j = i8 * 8 + (lane >> 2);
            if (j < left && n8 < p.t.N)
              *reinterpret_cast<uint4*>(y + i8 * 8 * p.t.N) = *reinterpret_cast<const uint4*>(turn + j * 64 + piece * 16);
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
  tc_fence_before();
  __syncthreads();
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
// The rows that the kernel for few of them takes at once, 0: too many, or too long for its shared memory.
constexpr int FEW_SMEM = 64 * 1024;
int few_rows(int64_t rows, int64_t K) {
  const int mt = rows == 1 ? 1 : rows == 2 ? 2 : rows <= 4 ? 4 : 8;
  return rows <= FEW_ROWS && mt * K <= FEW_SMEM ? mt : 0;
}
template <int MT> int launch_few(const TokenArgs& a, cudaStream_t st) {
  static std::atomic<int> allowed[MAX_SMEM_DEVICES];
  I8L_CUDA_OK(allow_smem(few_rows_kernel<MT>, allowed, FEW_SMEM));
  const int64_t segments = a.experts < a.rows ? a.experts : a.rows;
  const int64_t blocks = (segments * a.N / FEW_COLS + FEW_WARPS - 1) / FEW_WARPS, resident = 2 * sm_count();
  few_rows_kernel<MT><<<(unsigned)(blocks < resident ? blocks : resident), FEW_THREADS, MT * a.K, st>>>(a);
  I8L_CUDA_OK(cudaGetLastError());
  return I8L_OK;
}

// Tokens of a tile, from what the host knows: as if all rows belonged to experts, and to all alike.  A tile of s columns takes 0.4 + 0.6 *
// s / 256 of a full one (less for the MMAs, as much for the weights and the rest), and up to three waves of tiles end with the
// slowest.  us with 64, 128 and 256: dense 4096x4096 of 256 rows 12.6 / 13.3 / 16.0, 512 20.1 / 14.6 / 16.9, 1000 35 / 23 / 18.8;
// 64 experts of 1408x4096 with 32 rows each 69 / 67 / 72, 100 102 / 87 / 91, 500 350 / 269 / 223.  Over 100 sizes the choice costs
// 0.7 % against the best one, 9 % at most.
int tile_tokens(const TokenArgs& a) {
  const int64_t segments = a.experts < a.rows ? a.experts : a.rows, average = (a.rows + segments - 1) / segments;
  const int64_t n_tiles = (a.N + CHANNELS - 1) / CHANNELS;
  const int sms = gemm_cta_budget();
  int best = 0;
  double least = 0;
  for (int t = 64; t <= 256; t *= 2) {
    double per = 1;   // tiles of a segment; uneven ones need half a tile more than their average
    if (segments == 1) per = (double)((average + t - 1) / t);
    else if (average * 4 > t * 3) per = (double)average / t + 0.5;
    if (per < 1) per = 1;
    int64_t share = ((average + (int64_t)per - 1) / (int64_t)per + 15) / 16 * 16;
    if (share > t) share = t;
    const double tiles = (double)segments * per * (double)n_tiles, waves = tiles / sms;
    const double cost = (waves < 3 ? (double)(((int64_t)tiles + sms - 1) / sms) : waves + 0.5) * (0.4 + 0.6 * (double)share / 256);
    if (!best || cost < least) {
      best = t;
      least = cost;
    }
  }
  return best;
}

template <int TOK> int launch_group(const int8_t* xq, GroupArgs& p, cudaStream_t st) {
  using G = Grp<TOK>;
  static std::atomic<int> allowed[MAX_SMEM_DEVICES];
  const TokenArgs& a = p.t;
  I8L_CUDA_OK(allow_smem(group_kernel<TOK>, allowed, G::smem(MAX_EXPERTS)));
  p.n_tiles = (int)((a.N + CHANNELS - 1) / CHANNELS);
  const int64_t most = (a.rows / TOK + (a.experts < a.rows ? a.experts : a.rows)) * p.n_tiles;   // tiles, whatever the offsets
  if (most >= (1ll << 31)) return fail(I8L_ERR_SHAPE, "i8l_token_linear: too large for 32-bit tile numbers");
  CUtensorMap mw;
  TokenMaps mx;
  if (int e = make_tile_map_i8(&mw, a.wq, a.experts * a.N, a.K, CHANNELS)) return e;
  for (int i = 0; i < BOXES; ++i)
    if (int e = make_tile_map_i8(&mx.box[i], xq, a.rows, a.K, 16 << i)) return e;
  const int budget = gemm_cta_budget();
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attrs[1];
  cfg.gridDim = dim3((unsigned)(most < budget ? most : budget), 1, 1);
  cfg.blockDim = dim3(GRP_THREADS, 1, 1);
  cfg.dynamicSmemBytes = G::smem(a.experts);
  cfg.stream = st;
  chain_attribute(cfg, attrs);
  I8L_CUDA_OK(cudaLaunchKernelEx(&cfg, group_kernel<TOK>, mw, mx, p));
  return I8L_OK;
}

}  // namespace
}  // namespace i8l

using namespace i8l;

extern "C" int64_t i8l_token_linear_workspace(int64_t rows, int64_t K) {
  if (rows <= 0 || K <= 0 || rows >= (1ll << 31) || K > MAX_K || few_rows(rows, K)) return 0;
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
  if (!w_q || !w_scale || (rows && (!x || !y))) return fail(I8L_ERR_ARG, "i8l_token_linear: null pointer");
  if (!aligned16(x) || !aligned16(w_q) || !aligned16(y) || !aligned16(bias) || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return fail(I8L_ERR_ALIGN, "i8l_token_linear: x, w_q, y and bias must be 16-byte aligned, the workspace 256-byte");
  const int64_t need = i8l_token_linear_workspace(rows, K);
  if (need && (!workspace || workspace_bytes < need))
    return fail(I8L_ERR_ARG, "i8l_token_linear: workspace of %lld bytes is too small", (long long)workspace_bytes);
  if (!rows) return I8L_OK;
  if (int e = check_arch()) return e;
  TokenArgs a{};
  a.x = static_cast<const __nv_bfloat16*>(x); a.wq = w_q; a.ws = w_scale; a.offsets = offsets;
  a.bias = static_cast<const __nv_bfloat16*>(bias); a.y = y;
  a.rows = rows; a.N = N; a.K = K; a.experts = experts; a.out_f32 = (flags & I8L_GEMM_OUT_F32) ? 1 : 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (few_rows(rows, K)) {
    case 1: return launch_few<1>(a, st);
    case 2: return launch_few<2>(a, st);
    case 4: return launch_few<4>(a, st);
    case 8: return launch_few<8>(a, st);
  }
  int8_t* xq = static_cast<int8_t*>(workspace);
  float* xs = reinterpret_cast<float*>(xq + (rows * K + 255) / 256 * 256);
  const LaunchChain chain(st);
  if (int e = quant_token_rows(x, rows, K, xq, xs, st)) return e;
  (void)chain_first();
  GroupArgs p{};
  p.t = a;
  p.xs = xs;
  p.status = status;
  p.mirror = status ? mirror_of(status) : nullptr;
  p.max_polls = gemm_wait_limit();
  p.withhold = gemm_withhold();
  const int tok = tile_tokens(a);
  if (tok == 128) return launch_group<128>(xq, p, st);
  return tok == 256 ? launch_group<256>(xq, p, st) : launch_group<64>(xq, p, st);
}

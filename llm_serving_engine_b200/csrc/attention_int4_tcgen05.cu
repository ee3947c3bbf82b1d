// Attention of prompt portions over keys and values held in 4 bits (int4_cache.cu), causal, on the 5th-generation tensor cores;
// bfloat16 queries, head sizes 64 and 128, pages of any size.
//
// Three kernels (four when a launch has few blocks).
//   measure   the largest magnitude of every tile of 128 keys, and of its values, that the scales and centres allow for.
//   expand    the codes of every request's keys, page by page, become float16 values in a workspace: [head][row][D], a request's
//             rows one after the other, rounded up to whole tiles of 128 with zeros.  Once for all query heads and row tiles that
//             read them.  Float16 because a value s (u - 8) + c rounded to bfloat16 would be off by up to 2^-8, as much as the result's own
//             rounding, and float16 by 2^-11.  So that this holds for numbers of any size, a request's keys of a head, and its values, are
//             multiplied by a power of two (exact) that takes the largest of them to 2^14 .. 2^15: a number down to 2^-28 of that is rounded
//             by 2^-11 of itself, a smaller one by 2^-39 of the largest.  (With fixed powers, keys below 2^-6 and values below
//             2^-14 lost their last bits.)  attend takes the powers back out of scores and results.  The queries become
//             float16 here as well, each row of a head by a power of its own.  A row with a key beyond 2^24 or a
//             value beyond 65,504, or that is not a number, becomes NaN in its key and zeros in its value: who attends to it gets
//             NaN, and nobody else does.
//   attend    one block = 128 score rows of one request and key/value head: (token, query head of the group) pairs, so that
//             keys are brought in once for all heads of a group and portions of a few tokens fill the rows.  Keys are walked in tiles
//             of 128, which go alternately to two groups of four softmax warps, each with its own key and value stage, accumulators in
//             tensor memory, probability tile, maxima and sums; the two results are merged at the end.
//               loader warp   TMA: the queries once, then a tile of keys or values per copy.
//               MMA warps     one thread issues S = Q K^T (tcgen05.mma, tensor memory), one of another warp O += P V.
//               softmax       a thread owns a row of its group's tiles: scores from tensor memory, maximum, exp2 in float32, float16
//                             probabilities (2^-11 of them; of those below 2^-14, 2^-25 of the largest) to shared memory in the
//                             layout that the tensor cores read.  O is rescaled when a maximum has grown by more than 2^8 (at once
//                             beyond 2^14: float16 ends at 2^16).
//   combine   with fewer blocks than SMs, several blocks share the keys of a tile; each leaves its part in a workspace of this
//             call, and another launch adds them up, in the order of the parts.
// What bounds attend: 2,048 rows behind 6,144 keys, 40 / 8 heads of 128 (301 GFLOP) take 297 us, 1.01 PFLOP/s (327 to 342 at the power cap): tensor
// cores busy for 58% of the cycles, the unit of the exponentials for 58% (128 x 128 a tile at 16 a cycle), and 656 blocks leave a
// fifth turn of the SMs half empty.  Side by side with 324 (before the scales were measured, 3 us): all exponentials of a tile before the wait for the product of the tile
// before 350, a quarter of them 338; a quarter of the exponentials by a polynomial 361; scores read twice from tensor memory, 32 at a
// time, 354.  Small launches: a block's way from its start to its first scores (2.7 us), through a few tiles and to its end is 8 us,
// and eight portions of about 200 rows (160 blocks, 25.6 us) make some SMs go it twice; starting the blocks with most keys first
// took 26.6 instead of 24.1 (the search for them costs every block more than the order wins).
// Every wait is bounded (see tcgen05.cuh); a block whose wait gave up leaves NaN in its rows, frees its tensor memory and returns.
#include <cuda_fp16.h>

#include "smem_allowance.cuh"
#include "tcgen05.cuh"

LSE_CHECK_DEFINE(lse_check_attention_int4_tc)

namespace {
using namespace tc;

constexpr int BM = 128, BN = 128, GROUPS = 2, GROUP_THREADS = 128;
constexpr int MMA_WARP = 8, LOADER_WARP = 9, PV_WARP = 10, THREADS = 352;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_STEP = 8.0f, REDO_STEP = 14.0f;   // in powers of two
// (two portions of 128 rows behind 2,000 keys of 12 / 2 heads, six parts: 21.2 us; two tiles a part 27.0, eight 23.8; a portion of 16 rows
// behind 30,000 keys of 28 / 4 heads, one part 240, two 139, four 86, eight 62)
constexpr int MIN_TILES_A_PART = 4, MAX_PARTS = 8;
constexpr uint32_t HALF_BYTES = 128 * 128;                // 128 rows x 64 float16
constexpr float MOST_KEY = 65504.0f * 256.0f, MOST_VALUE = 65504.0f;       // rows beyond become NaN

__device__ int lse_attn_int4_tc_error;

enum Bar { B_Q = 0, B_KF = 1, B_KE = 3, B_VF = 5, B_VE = 7, B_SF = 9, B_PF = 11, B_SR = 13, B_OD = 15, B_COUNT = 17 };

__device__ __forceinline__ float exp2_fast(float x) {   // 2^x, 2^-inf = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void pair_barrier(int quarter) {   // the warps of the two groups that own the same 32 rows
  asm volatile("bar.sync %0, %1;\n" ::"r"(1 + quarter), "r"(64) : "memory");
}
// D float32, A and B float16 (the type fields that bfloat16 sets to one are zero)
__device__ __forceinline__ uint32_t instr_desc_f16(int m, int n, bool a_mn, bool b_mn) {
  return instr_desc_bf16(m, n, a_mn, b_mn) & ~((7u << 7) | (7u << 10));
}
template <int D> constexpr size_t attend_smem() { return 1024 + (size_t)(D / 64) * HALF_BYTES * (1 + 2 * GROUPS) + (size_t)GROUPS * 2 * HALF_BYTES + 256; }

// What a block works on: the rank-th tile of rows, counted from the last request's last one backwards (late tiles walk the most keys and
// start first; ranks beyond the number of tiles have none: seg = -1).  The first warp looks at 32 requests at a time, once where there
// are no more, and leaves everything in `work`; the block has to meet before it is read.
struct Work { int seg, r0, rows, first_row, first_pos, tile0; };
__device__ __forceinline__ void find_work(const int* segment_start, const int* first_pos, int num_segments, int tokens_a_tile, int skip_single,
                                          int rank, Work* work) {
  const int lane = threadIdx.x & 31;
  struct Request { int start, rows, first, tiles, key_tiles; };
  auto look = [&](int s) {
    Request r = {0, 0, 0, 0, 0};
    if (s < num_segments) {
      r.start = segment_start[s];
      r.rows = max(segment_start[s + 1] - r.start, 0);
      r.first = first_pos[s];
      r.tiles = r.rows == 1 && skip_single ? 0 : (r.rows + tokens_a_tile - 1) / tokens_a_tile;
      r.key_tiles = r.rows > 0 ? (max(0, r.first + r.rows) + BN - 1) / BN : 0;
    }
    return r;
  };
  const Request first = look(lane);
  int all = first.tiles;
  for (int base = 32; base < num_segments; base += 32) all += look(base + lane).tiles;
  const int wanted = __reduce_add_sync(0xffffffffu, all) - 1 - rank;
  if (lane == 0) work->seg = -1;
  __syncwarp();
  int before = 0, keys_before = 0;
  for (int base = 0; base < num_segments && wanted >= before; base += 32) {
    const Request r = base == 0 ? first : look(base + lane);
    int incl = r.tiles, keys_incl = r.key_tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o), k = __shfl_up_sync(0xffffffffu, keys_incl, o);
      if (lane >= o) { incl += v; keys_incl += k; }
    }
    const int at = wanted - before - (incl - r.tiles);
    if (at >= 0 && at < r.tiles) *work = {base + lane, at * tokens_a_tile, r.rows, r.start, r.first, keys_before + keys_incl - r.key_tiles};
    before += __shfl_sync(0xffffffffu, incl, 31);
    keys_before += __shfl_sync(0xffffffffu, keys_incl, 31);
  }
}

// The power of two that takes numbers of this biased exponent (of float32) to 2^14 .. 2^15, and its inverse.  2^74 at most, so that
// the inverse times a weight stays a normal number: what is smaller than 2^-60 uses less of float16's range.
__device__ __forceinline__ float unit_up(uint32_t exponent) { return __uint_as_float((268u - min(max(exponent, 67u), 254u)) << 23); }
__device__ __forceinline__ float unit_down(uint32_t exponent) { return __uint_as_float((min(max(exponent, 67u), 254u) - 14u) << 23); }
// The largest magnitude that a row's codes could stand for (not a number where the row is not one).
__device__ __forceinline__ float most_of(float2 row) { return fabsf(row.y) + 8.f * fabsf(row.x); }

// Whose tile of keys the tile-th of the workspace is, by a whole warp, 32 requests at a time: the request (-1: behind the last
// request's tiles, -2: one that another kernel takes), its first key's number, the request's keys and its first tile.
struct KeyTile { int seg, key0, keys, first; };
__device__ __forceinline__ KeyTile find_keys(const int* segment_start, const int* first_pos, int num_segments, int skip_single, int tile) {
  const int lane = threadIdx.x & 31;
  KeyTile found = {-1, 0, 0, 0};
  int before = 0;
  for (int base = 0; base < num_segments && found.seg == -1; base += 32) {
    const int s = base + lane;
    int n = 0, ctx = 0, rows = 0;
    if (s < num_segments) {
      rows = segment_start[s + 1] - segment_start[s];
      ctx = rows > 0 ? max(0, first_pos[s] + rows) : 0;
      n = (ctx + BN - 1) / BN;
    }
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const unsigned vote = __ballot_sync(0xffffffffu, n > 0 && tile >= before + incl - n && tile < before + incl);
    if (vote) {
      const int src = __ffs(vote) - 1;
      found.first = before + __shfl_sync(0xffffffffu, incl - n, src);
      found.key0 = (tile - found.first) * BN;
      found.keys = __shfl_sync(0xffffffffu, ctx, src);
      found.seg = __shfl_sync(0xffffffffu, skip_single && rows == 1 ? 1 : 0, src) ? -2 : base + src;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return found;
}

// ------------------------------------------------------------------ measure
// One block = a tile and head: a thread a key's scale and centre, or its value's.
__global__ void __launch_bounds__(2 * BN)
measure_int4_kernel(const __nv_bfloat162* k_scales, const __nv_bfloat162* v_scales, uint2* __restrict__ tops,
                    const int* __restrict__ block_tables, int bt_stride, const int* __restrict__ segment_start,
                    const int* __restrict__ first_pos, int num_segments, int n_kv, int head0, int page_size, int num_pages, int skip_single) {
  __shared__ KeyTile found_s;
  __shared__ uint32_t top_s[2 * BN / 32];
  pdl_launch_dependents();
  const int tile = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
  if (tid < 32) {
    const KeyTile found = find_keys(segment_start, first_pos, num_segments, skip_single, tile);
    if (tid == 0) found_s = found;
  }
  __syncthreads();
  const KeyTile at = found_s;
  const int key = at.key0 + tid % BN;
  const bool live = at.seg >= 0 && key < at.keys;
  int page = 0;
  const int logical = (unsigned)key / (unsigned)page_size;
  if (live) page = LSE_CHECKED(block_tables[(size_t)at.seg * bt_stride + logical], 0, num_pages, 0, LSE_CHECK_TABLE_ENTRY);
  pdl_wait();
  float most = 0.f;
  if (live) {
    const size_t place = ((size_t)page * n_kv + head0 + head) * page_size + (key - logical * page_size);
    most = most_of(__bfloat1622float2((tid < BN ? k_scales : v_scales)[place]));
    if (!(most <= (tid < BN ? MOST_KEY : MOST_VALUE))) most = 0.f;       // (a row that becomes NaN)
  }
  const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));      // (as whole numbers: none is negative)
  if ((tid & 31) == 0) top_s[tid >> 5] = top;
  __syncthreads();
  if (tid == 0) {
    uint2 tops_here = make_uint2(0, 0);
    for (int w = 0; w < BN / 32; ++w) { tops_here.x = max(tops_here.x, top_s[w]); tops_here.y = max(tops_here.y, top_s[BN / 32 + w]); }
    tops[(size_t)head * gridDim.x + tile] = tops_here;
  }
}

// ------------------------------------------------------------------ expand
// One block = EXPAND_KEYS keys of a tile and one head, keys and values; 256 threads, LANES = D / 8 of them a row, eight values each, all loads
// of a thread on their way together (a block a tile, eight rows a thread one after the other: 17 us for 51 tiles of two heads).
constexpr int EXPAND_KEYS = 32;
// The blocks behind those (blockIdx.z) make the queries float16, QUERY_PIECES times 16 bytes a thread, a head's row by LANES neighbours.
constexpr int QUERY_PIECES = 4;
template <int D>
__global__ void __launch_bounds__(256)
expand_int4_kernel(const unsigned char* k_codes, const __nv_bfloat162* k_scales,
                   const unsigned char* v_codes, const __nv_bfloat162* v_scales, uint4* __restrict__ k_out,
                   uint4* __restrict__ v_out, const uint2* tops, float2* units, const int* __restrict__ block_tables, int bt_stride,
                   const int* __restrict__ segment_start, const int* __restrict__ first_pos, int num_segments, int n_kv, int head0, int page_size,
                   int num_pages, int skip_single, const uint4* q, uint4* q_out, float* q_units, long long q_pieces) {
  constexpr int LANES = D / 8, ROWS = 256 / LANES, MINE = EXPAND_KEYS / ROWS;      // rows at once, rows of a thread
  __shared__ KeyTile found_s;
  pdl_launch_dependents();
  const int tile = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, lane = tid & 31, capacity = gridDim.x;
  if (blockIdx.z >= BN / EXPAND_KEYS) {
    pdl_wait();
    const long long block = ((long long)(blockIdx.z - BN / EXPAND_KEYS) * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
    uint4 w[QUERY_PIECES];
#pragma unroll
    for (int k = 0; k < QUERY_PIECES; ++k) {
      const long long i = (block * QUERY_PIECES + k) * 256 + tid;
      w[k] = i < q_pieces ? q[i] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int k = 0; k < QUERY_PIECES; ++k) {
      const long long i = (block * QUERY_PIECES + k) * 256 + tid;
      uint32_t* x = &w[k].x;
      uint32_t top = 0;       // the largest magnitude of the row, as the bits of a bfloat16
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, max(x[e] & 0x7fffu, x[e] >> 16 & 0x7fffu));
#pragma unroll
      for (int o = 1; o < LANES; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float up = unit_up(top >> 7);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x[e]));
        x[e] = pack_f16(v.x * up, v.y * up);
      }
      if (i < q_pieces) {
        q_out[i] = w[k];
        if (i % LANES == 0) q_units[i / LANES] = unit_down(top >> 7);
      }
    }
    return;
  }
  if (tid < 32) {
    const KeyTile found = find_keys(segment_start, first_pos, num_segments, skip_single, tile);
    if (tid == 0) found_s = found;
  }
  __syncthreads();
  const int seg = found_s.seg, key0 = found_s.key0, keys = found_s.keys, first = found_s.first;
  pdl_wait();                // (before any return: a launch without work must not end before the one before it)
  if (seg < 0) return;
  const int c = tid % LANES, r0 = blockIdx.z * EXPAND_KEYS + tid / LANES;
  const size_t out0 = ((size_t)head * capacity + tile) * BN;
  const int* bt = block_tables + (size_t)seg * bt_stride;
  uint32_t kx[MINE], vx[MINE];
  __nv_bfloat162 ks[MINE], vs[MINE];
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    const int key = key0 + r0 + i * ROWS;
    kx[i] = vx[i] = 0u;
    ks[i] = vs[i] = __floats2bfloat162_rn(0.f, 0.f);      // (keys behind the last become zeros)
    if (key < keys) {
      const int logical = (unsigned)key / (unsigned)page_size;
      const int page = LSE_CHECKED(bt[logical], 0, num_pages, 0, LSE_CHECK_TABLE_ENTRY);
      const size_t place = ((size_t)page * n_kv + head0 + head) * page_size + (key - logical * page_size);
      kx[i] = reinterpret_cast<const uint32_t*>(k_codes + place * (D / 2))[c];
      vx[i] = reinterpret_cast<const uint32_t*>(v_codes + place * (D / 2))[c];
      ks[i] = k_scales[place];
      vs[i] = v_scales[place];
    }
  }
  // the largest of all the request's tiles, by every warp (the tiles that the workspace has no room for are not worked on)
  uint2 top = make_uint2(0, 0);
  for (int i = first + lane; i < min(capacity, first + (keys + BN - 1) / BN); i += 32) {
    const uint2 t = tops[(size_t)head * capacity + i];
    top.x = max(top.x, t.x); top.y = max(top.y, t.y);
  }
  const uint32_t k_exponent = __reduce_max_sync(0xffffffffu, top.x) >> 23, v_exponent = __reduce_max_sync(0xffffffffu, top.y) >> 23;
  const float k_up = unit_up(k_exponent), v_up = unit_up(v_exponent);
  if (tile == first && blockIdx.z == 0 && tid == 0) units[(size_t)head * capacity + tile] = make_float2(unit_down(k_exponent), unit_down(v_exponent));
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    float2 kf = __bfloat1622float2(ks[i]), vf = __bfloat1622float2(vs[i]);
    const bool fits = most_of(kf) <= MOST_KEY && most_of(vf) <= MOST_VALUE;      // false for what is not a number
    kf.x *= k_up; kf.y *= k_up;
    vf.x *= v_up; vf.y *= v_up;
    auto values = [](uint32_t x, float2 s) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = pack_f16(fmaf(s.x, (float)((int)(x >> (8 * j) & 15u) - 8), s.y), fmaf(s.x, (float)((int)(x >> (8 * j + 4) & 15u) - 8), s.y));
      return make_uint4(w[0], w[1], w[2], w[3]);
    };
    uint4 kw = make_uint4(0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u), vw = make_uint4(0, 0, 0, 0);
    if (fits) { kw = values(kx[i], kf); vw = values(vx[i], vf); }
    const size_t at = (out0 + r0 + i * ROWS) * LANES + c;
    k_out[at] = kw;
    v_out[at] = vw;
  }
}

// ------------------------------------------------------------------ attend
template <int D>
__global__ void __launch_bounds__(THREADS, 1)
attend_int4_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, __nv_bfloat16* __restrict__ out, const int* __restrict__ segment_start,
                   const int* __restrict__ first_pos, int num_segments, int n_q, int group, int heads, int head0, int tokens_a_tile,
                   float scale_log2e, int capacity, int skip_single, int parts, const float2* units, const float* q_units,
                   float* __restrict__ part_o, float2* __restrict__ part_ml) {
  constexpr int HALVES = D / 64;
  constexpr uint32_t Q_BYTES = HALVES * HALF_BYTES, KV_BYTES = HALVES * HALF_BYTES, P_BYTES = 2 * HALF_BYTES;
  constexpr uint32_t GROUP_BYTES = HALVES * 1024;          // 8 keys in a stage
  constexpr uint32_t S_COLS = BN, O_COL = GROUPS * BN;     // tensor memory: S of group 0, S of group 1, O of group 0, O of group 1
  constexpr int OD = D / 2;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* gbase = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t q_s = base, k_s = q_s + Q_BYTES, v_s = k_s + GROUPS * KV_BYTES, p_s = v_s + GROUPS * KV_BYTES;
  const uint32_t bars = p_s + GROUPS * P_BYTES;
  unsigned char* tail = gbase + (bars - base);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 8 * B_COUNT);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 8 * B_COUNT + 4);
  Work* work = reinterpret_cast<Work*>(tail + 8 * B_COUNT + 8);
  auto bar = [&](int i) { return bars + 8u * (uint32_t)i; };

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int head = blockIdx.x % heads;                      // key/value head, counted from head0
  const int part = (int)(blockIdx.x / heads) % parts;
  const int rank = (int)(blockIdx.x / heads) / parts;
  pdl_launch_dependents();
  if (tid == 0) {
    for (int i = 0; i < B_COUNT; ++i) mbar_init(bar(i), i >= B_PF && i < B_OD ? GROUP_THREADS : 1);
    *abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == MMA_WARP) tmem_alloc(tmem_slot, 512);
  if (warp == PV_WARP) find_work(segment_start, first_pos, num_segments, tokens_a_tile, skip_single, rank, work);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const int r0 = work->r0, cnt = work->rows, tile0 = work->tile0;
  const int ntok = min(tokens_a_tile, cnt - r0), nrows = ntok * group;
  const int row_base = work->first_row + r0;
  const int pos0 = work->first_pos + r0;
  const int last_pos = pos0 + ntok - 1;
  const int n_tiles = last_pos / BN + 1;
  const int sharing = max(1, min(parts, n_tiles / MIN_TILES_A_PART));
  if (work->seg < 0 || part >= sharing) {      // nothing to do (how many blocks share a tile is worked out by combine as well)
    pdl_wait();
    if (warp == MMA_WARP) tmem_dealloc(tmem_base, 512);
    return;
  }
  const int j_lo = sharing == 1 ? 0 : part * n_tiles / sharing, n_local = sharing == 1 ? n_tiles : (part + 1) * n_tiles / sharing - j_lo;
  int* const err = &lse_attn_int4_tc_error;
  const bool held = tile0 + (work->first_pos + cnt + BN - 1) / BN <= capacity;   // the workspace has all of the request's tiles

  pdl_wait();

  if (!held) {
    // fewer keys were announced than the requests hold: NaN, rather than what other requests' keys would give
  } else if (warp == LOADER_WARP) {
    if (lane == 0) {
      mbar_expect_tx(bar(B_Q), (uint32_t)(tokens_a_tile * group) * 128u * HALVES);
      for (int h = 0; h < HALVES; ++h) tma_load_3d(q_s + h * HALF_BYTES, &map_q, bar(B_Q), h * 64, (head0 + head) * group, row_base);
      // K of tile j + 1 goes before V of tile j: the scores are wanted first
      auto load = [&](int jj, uint32_t dst, const CUtensorMap* map, int full, int empty) {
        const int g = jj & 1;
        if (!mbar_wait(bar(empty + g), ((uint32_t)(jj >> 1) & 1u) ^ 1u, abort_flag, err)) return false;
        mbar_expect_tx(bar(full + g), KV_BYTES);
        tma_load_4d(dst + g * KV_BYTES, map, bar(full + g), 0, 0, 0, (head * capacity + tile0 + j_lo + jj) * (BN / 8));
        return true;
      };
      bool ok = load(0, k_s, &map_k, B_KF, B_KE);
      for (int jj = 0; jj < n_local && ok; ++jj) {
        if (jj + 1 < n_local) ok = load(jj + 1, k_s, &map_k, B_KF, B_KE);
        if (ok) ok = load(jj, v_s, &map_v, B_VF, B_VE);
      }
    }
    __syncwarp();
  } else if (warp == MMA_WARP) {
    if (lane == 0) {
      const uint32_t idesc_s = instr_desc_f16(BM, BN, false, false);
      bool ok = mbar_poll(bar(B_Q), 0, abort_flag, err);
      for (int j = 0; j < n_local && ok; ++j) {
        const int g = j & 1;
        const uint32_t parity = (uint32_t)(j >> 1) & 1u;
        ok = mbar_poll(bar(B_KF + g), parity, abort_flag, err);
        if (ok && j >= GROUPS) ok = mbar_poll(bar(B_SR + g), parity ^ 1u, abort_flag, err);
        if (!ok) break;
        fence_after_sync();
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t off = (uint32_t)(ks / 4) * HALF_BYTES + (uint32_t)(ks % 4) * 32u;
          const uint32_t k_off = (uint32_t)(ks / 4) * 1024u + (uint32_t)(ks % 4) * 32u;
          umma_bf16(tmem_base + g * S_COLS, smem_desc_k_major(q_s + off), smem_desc_k_major(k_s + g * KV_BYTES + k_off, GROUP_BYTES),
                    idesc_s, ks != 0 ? 1u : 0u);
        }
        umma_commit(bar(B_KE + g));
        umma_commit(bar(B_SF + g));
      }
    }
    __syncwarp();
  } else if (warp == PV_WARP) {
    if (lane == 0) {
      const uint32_t idesc_o = instr_desc_f16(BM, D, false, true);
      bool ok = true;
      for (int i = 0; i < n_local && ok; ++i) {
        const int g = i & 1;
        const uint32_t parity = (uint32_t)(i >> 1) & 1u;
        ok = mbar_poll(bar(B_VF + g), parity, abort_flag, err) && mbar_poll(bar(B_PF + g), parity, abort_flag, err);
        if (!ok) break;
        fence_after_sync();
#pragma unroll
        for (int ks = 0; ks < BN / 16; ++ks) {
          const uint32_t p_off = (uint32_t)(ks / 4) * HALF_BYTES + (uint32_t)(ks % 4) * 32u;
          umma_bf16(tmem_base + O_COL + g * D, smem_desc_k_major(p_s + g * P_BYTES + p_off),
                    smem_desc_mn_major(v_s + g * KV_BYTES + (uint32_t)ks * 2u * GROUP_BYTES, 1024u, GROUP_BYTES), idesc_o,
                    (i >= GROUPS || ks != 0) ? 1u : 0u);
        }
        umma_commit(bar(B_VE + g));
        umma_commit(bar(B_OD + g));
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax
    const int g = warp >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const bool live = row < nrows;      // (the other rows hold other tokens' queries or nothing at all, and decide nothing)
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_addr = lane_addr + g * S_COLS, o_addr = lane_addr + O_COL + g * D;
    const int my_pos = pos0 + min(row, nrows - 1) / group;
    unsigned char* prow = gbase + (p_s - base) + g * P_BYTES + row * 128;
    // the powers of two in this row's scores and in the values
    const float2 unit = units[(size_t)head * capacity + tile0];
    const int my_row = min(row, nrows - 1);
    const double exact_scale = (double)scale_log2e * (double)q_units[(long long)(row_base + my_row / group) * n_q + (head0 + head) * group + my_row % group] * (double)unit.x;
    const float row_scale = (float)fmin(fmax(exact_scale, 0x1p-126), 0x1p127);      // (beyond, scores are all alike, or infinitely far apart)
    const uint64_t scale_pair = f32_pair(row_scale, row_scale);      // (made here: 340 us for the 2,048 rows below; in the loop 347)
    float m_used = -INFINITY, m_seen = -INFINITY, l = 0.f;   // the maximum that O and l are relative to; the largest score seen
    bool pending = false;                                    // m_seen has outgrown m_used: O and l are to be rescaled
    bool ok = true;                                          // the same in all lanes of a warp (a vote after every wait)
    auto wait_all = [&](int which, uint32_t parity) {
      const bool done = mbar_test(bar(which), parity) || mbar_wait(bar(which), parity, abort_flag, err);
      return __all_sync(0xffffffffu, done ? 1 : 0) != 0;
    };
    for (int j = g; j < n_local && ok; j += GROUPS) {   // j counts this block's tiles
      const uint32_t parity = (uint32_t)(j >> 1) & 1u;
      ok = wait_all(B_SF + g, parity);
      if (!ok) break;
      fence_after_sync();
      const int kv0 = (j_lo + j) * BN;
      const bool diagonal = kv0 + BN - 1 > my_pos;
      // the whole row of scores into registers: the accumulator is free for the group's next tile at once
      uint32_t s[BN / 32][32];
#pragma unroll
      for (int c = 0; c < BN / 32; ++c) tmem_ld32(s_addr + 32 * c, s[c]);
      tmem_ld_wait();
      fence_before_sync();
      mbar_arrive(bar(B_SR + g));
      bool rescale = false;
      float alpha = 1.f, mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < BN / 32; ++c) {
        if (diagonal) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (kv0 + 32 * c + i > my_pos) s[c][i] = 0xff800000u;
        }
#pragma unroll
        for (int i = 0; i < 32; i += 2) mx = fmaxf(mx, fmaxf(__uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1])));
      }
      const float m_tile = mx * row_scale;
      if (j < GROUPS) {
        m_used = m_seen = m_tile;
      } else {
        m_seen = fmaxf(m_seen, m_tile);
        if (pending || __any_sync(0xffffffffu, live && m_tile > m_used + REDO_STEP)) {
          rescale = true;
          alpha = m_used == -INFINITY ? 0.f : exp2_fast(m_used - m_seen);
          m_used = m_seen;
          l *= alpha;
        }
      }
      pending = __any_sync(0xffffffffu, live && m_seen > m_used + RESCALE_STEP) != 0;
      if (j >= GROUPS) {   // P V of this group's tile before has read the probabilities and added to O
        ok = wait_all(B_OD + g, parity ^ 1u);
        if (!ok) break;
        fence_after_sync();
      }
      if (rescale) {
#pragma unroll 1
        for (int c = 0; c < D; c += 8) {
          uint32_t o[8];
          tmem_ld8(o_addr + c, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st8(o_addr + c, o);
        }
        tmem_st_wait();
      }
      const float neg = m_used == -INFINITY ? 0.f : -m_used;
      const uint64_t neg_pair = f32_pair(neg, neg);
      uint64_t sum_pair = 0;
#pragma unroll
      for (int c = 0; c < BN / 32; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float p0, p1;
          f32_halves(f32_pair_fma(f32_pair(__uint_as_float(s[c][2 * i]), __uint_as_float(s[c][2 * i + 1])), scale_pair, neg_pair), p0, p1);
          p0 = exp2_fast(p0); p1 = exp2_fast(p1);
          sum_pair = f32_pair_add(sum_pair, f32_pair(p0, p1));
          pk[i] = pack_f16(p0, p1);
        }
        unsigned char* box = prow + (c / 2) * HALF_BYTES;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int chunk = (c % 2) * 4 + k;
          *reinterpret_cast<uint4*>(box + ((chunk ^ (row & 7)) << 4)) = make_uint4(pk[4 * k], pk[4 * k + 1], pk[4 * k + 2], pk[4 * k + 3]);
        }
      }
      float sum_even, sum_odd;
      f32_halves(sum_pair, sum_even, sum_odd);
      l += sum_even + sum_odd;
      fence_async_smem();
      fence_before_sync();
      mbar_arrive(bar(B_PF + g));
    }
    // ---------------------------------------------------------------- merge of the two groups
    // A group hands its maxima and sums over in its own key stage, which nothing reads or writes any more.
    float* mine = reinterpret_cast<float*>(gbase + (k_s - base) + g * KV_BYTES);
    const float* other = reinterpret_cast<const float*>(gbase + (k_s - base) + (g ^ 1) * KV_BYTES);
    mine[row] = m_used;
    mine[128 + row] = l;
    pair_barrier(quarter);
    const float m_other = other[row], l_other = other[128 + row];
    const float m_all = fmaxf(m_used, m_other);
    // (a sum that is not a number keeps that, whatever its maximum)
    const float w_mine = m_used == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2_fast(m_used - m_all);
    const float w_other = m_other == -INFINITY ? (l_other == 0.f ? 0.f : 1.f) : exp2_fast(m_other - m_all);
    const float l_all = g == 0 ? fmaf(l_other, w_other, l * w_mine) : fmaf(l, w_mine, l_other * w_other);
    const bool shared = sharing > 1;
    const float inv = shared ? unit.y : unit.y / l_all;
    const float w0 = (g == 0 ? w_mine : w_other) * inv, w1 = (g == 0 ? w_other : w_mine) * inv;
    const int n0 = (n_local + 1) / 2, n1 = n_local / 2;     // tiles of the groups
    if (ok) ok = wait_all(B_OD + 0, (uint32_t)(n0 - 1) & 1u);
    if (ok && n1 > 0) ok = wait_all(B_OD + 1, (uint32_t)(n1 - 1) & 1u);
    // This thread has columns g * D / 2 .. of its row; they go by way of the group's probability tile, which nothing reads any more, so
    // that a warp stores whole lines (a thread its own row: 1.6 us a block).
    const long long out_row = (long long)(row_base + row / group) * n_q + (head0 + head) * group + row % group;
    if (ok) {
      fence_after_sync();
      unsigned char* const turn = gbase + (p_s - base) + g * P_BYTES + quarter * 8192;      // 32 rows of 256 bytes at most
      uint4* const outs = reinterpret_cast<uint4*>(shared ? (void*)(part_o + (long long)part * D + g * OD) : (void*)(out + g * OD));
      const int pieces = shared ? OD / 4 : OD / 8, piece_bits = 31 - __clz(pieces);       // 16 bytes each, of a row
      const long long row_pieces = shared ? (long long)parts * (D / 4) : D / 8;
#pragma unroll
      for (int c = 0; c < OD; c += 32) {
        uint32_t a[32], b[32];
        tmem_ld32(lane_addr + O_COL + g * OD + c, a);
        if (n1 > 0) tmem_ld32(lane_addr + O_COL + D + g * OD + c, b);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] = __uint_as_float(a[8 * i + e]) * w0;
            if (n1 > 0) v[e] = fmaf(__uint_as_float(b[8 * i + e]), w1, v[e]);
          }
          uint4* const mine_row = reinterpret_cast<uint4*>(turn) + lane * pieces;
          if (shared) {
            const int k = c / 4 + 2 * i;
            mine_row[k ^ (lane & 7)] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
            mine_row[(k + 1) ^ (lane & 7)] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
          } else {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const __nv_bfloat162 x = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
              w[e] = *reinterpret_cast<const uint32_t*>(&x);
            }
            mine_row[(c / 8 + i) ^ (lane & 7 & (pieces - 1))] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      __syncwarp();
#pragma unroll 4
      for (int i = lane; i < 32 * pieces; i += 32) {
        const int r = i >> piece_bits, k = i & (pieces - 1);
        const long long to = __shfl_sync(0xffffffffu, out_row, r);
        if (quarter * 32 + r < nrows) outs[to * row_pieces + k] = reinterpret_cast<const uint4*>(turn)[r * pieces + (k ^ (r & 7 & (pieces - 1)))];
      }
      if (shared && g == 0 && row < nrows) part_ml[out_row * parts + part] = make_float2(m_all, l_all);
    }
  }
  if (*abort_flag && tid == 0) {
    // a wait gave up: give copies that may still be in flight time to land before the block leaves
    for (int i = 0; i < 2000; ++i) __nanosleep(100);
  }
  fence_before_sync();
  __syncthreads();
  if (warp == MMA_WARP) tmem_dealloc(tmem_base, 512);
  if (!held || *abort_flag) {
    const float nan = __int_as_float(0x7fc00000);
    for (int i = tid; i < nrows; i += THREADS) {
      const size_t out_row = (size_t)(row_base + i / group) * n_q + (head0 + head) * group + i % group;
      if (sharing > 1) part_ml[out_row * parts + part] = make_float2(0.f, nan);
      for (int d = 0; d < D; ++d)
        if (sharing > 1) part_o[(out_row * parts + part) * D + d] = nan; else out[out_row * D + d] = __float2bfloat16_rn(nan);
    }
  }
}

// ------------------------------------------------------------------ combine
// One block = a tile of rows and a key/value head as attend's, eight (token, head) pairs of it; a warp adds up the parts of a pair.
template <int D>
__global__ void __launch_bounds__(256)
combine_tiles_kernel(const float* part_o, const float2* part_ml, __nv_bfloat16* __restrict__ out,
                     const int* __restrict__ segment_start, const int* __restrict__ first_pos, int num_segments, int n_q, int group,
                     int heads, int head0, int tokens_a_tile, int skip_single, int parts) {
  constexpr int V = D / 32;
  __shared__ int tile_slot[3];
  pdl_launch_dependents();
  const int head = blockIdx.x % heads, rank = blockIdx.x / heads, lane = threadIdx.x & 31;
  int seg, r0, cnt;
  lse_find_tile(segment_start, num_segments, tokens_a_tile, skip_single, rank, tile_slot, seg, r0, cnt);
  pdl_wait();
  if (seg < 0) return;
  const int ntok = min(tokens_a_tile, cnt - r0), row = (int)blockIdx.y * 8 + (threadIdx.x >> 5);
  const int n_tiles = (first_pos[seg] + r0 + ntok - 1) / BN + 1;
  const int sharing = max(1, min(parts, n_tiles / MIN_TILES_A_PART));
  if (sharing == 1 || row >= ntok * group) return;
  const size_t out_row = (size_t)(segment_start[seg] + r0 + row / group) * n_q + (head0 + head) * group + row % group;
  const float2 ml = lane < sharing ? part_ml[out_row * parts + lane] : make_float2(-INFINITY, 0.f);
  const float M = warp_max(ml.x);
  const float weight = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : exp2_fast(ml.x - M);
  const float inv = 1.0f / warp_sum(ml.y * weight);
  float o[V];
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = 0.f;
#pragma unroll
  for (int p = 0; p < MAX_PARTS; ++p) {
    if (p < sharing) {
      const float w = __shfl_sync(0xffffffffu, weight, p);
      const float* src = part_o + (out_row * parts + p) * D + lane * V;
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        const float2 v = *reinterpret_cast<const float2*>(src + i);
        o[i] = fmaf(v.x, w, o[i]); o[i + 1] = fmaf(v.y, w, o[i + 1]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; i += 2)
    *reinterpret_cast<__nv_bfloat162*>(out + out_row * D + lane * V + i) = __floats2bfloat162_rn(o[i] * inv, o[i + 1] * inv);
}

// Tensor map of a bfloat16 tensor [outer, middle, cols]; box = [box_outer, box_middle, 64 columns], 128-byte swizzle.
bool make_map_queries(CUtensorMap* map, const void* ptr, long long outer, int middle, int cols, int box_outer, int box_middle) {
  EncodeTiledFn fn = encode_tiled();
  if (fn == nullptr) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)middle, (cuuint64_t)outer};
  const cuuint64_t strides[2] = {(cuuint64_t)cols * 2, (cuuint64_t)cols * 2 * (cuuint64_t)middle};
  const cuuint32_t box[3] = {64u, (cuuint32_t)box_middle, (cuuint32_t)box_outer};
  const cuuint32_t elem[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D>
int launch_portions(const void* q, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, void* out,
                    const int* block_tables, int bt_stride, const int* segment_start, const int* first_pos, int num_segments, int tokens,
                    long long num_pages, int n_q, int n_kv, int page_size, float scale, int skip_single, int with_tiles, int capacity,
                    int heads_at_once, int parts, void* keys, void* values, void* queries, void* powers, float* scratch, cudaStream_t stream) {
  static SmemAllowance allowance;
  const size_t smem = attend_smem<D>();
  cudaError_t err = allow_smem(attend_int4_kernel<D>, smem, allowance);
  if (err != cudaSuccess) return (int)err;
  const int group = n_q / n_kv, tokens_a_tile = BM / group;
  const int tiles = (tokens + tokens_a_tile - 1) / tokens_a_tile + with_tiles;
  float* part_o = parts > 1 ? scratch : nullptr;
  float2* part_ml = parts > 1 ? reinterpret_cast<float2*>(scratch + (size_t)tokens * n_q * parts * D) : nullptr;
  float2* units = reinterpret_cast<float2*>(powers);
  uint2* tops = reinterpret_cast<uint2*>(units + (size_t)heads_at_once * capacity);
  float* q_units = reinterpret_cast<float*>(tops + (size_t)heads_at_once * capacity);
  CUtensorMap map_q, map_k, map_v;
  for (int head0 = 0; head0 < n_kv; head0 += heads_at_once) {
    const int heads = n_kv - head0 < heads_at_once ? n_kv - head0 : heads_at_once;
    if (!make_map_queries(&map_q, queries, tokens, n_q, D, tokens_a_tile, group) ||
        !make_map_row_groups(&map_k, keys, (long long)heads * capacity * BN, D, BN) ||
        !make_map_row_groups(&map_v, values, (long long)heads * capacity * BN, D, BN))
      return LSE_ERR_BAD_ARGUMENT;
    const long long q_pieces = head0 == 0 ? (long long)tokens * n_q * (D / 8) : 0, a_layer = (long long)capacity * heads * 256 * QUERY_PIECES;
    if (q_pieces / a_layer > 60000) return LSE_ERR_TOO_LARGE;
    err = lse_launch(measure_int4_kernel, dim3((unsigned)capacity, (unsigned)heads), dim3(2 * BN), 0, stream,
                     (const __nv_bfloat162*)k_scales, (const __nv_bfloat162*)v_scales, tops, block_tables, bt_stride, segment_start,
                     first_pos, num_segments, n_kv, head0, page_size, (int)num_pages, skip_single);
    if (err != cudaSuccess) return (int)err;
    err = lse_launch(expand_int4_kernel<D>, dim3((unsigned)capacity, (unsigned)heads, (unsigned)(BN / EXPAND_KEYS + (q_pieces + a_layer - 1) / a_layer)), dim3(256), 0,
                     stream, (const unsigned char*)k_codes, (const __nv_bfloat162*)k_scales, (const unsigned char*)v_codes, (const __nv_bfloat162*)v_scales,
                     (uint4*)keys, (uint4*)values, (const uint2*)tops, units, block_tables, bt_stride, segment_start, first_pos, num_segments, n_kv,
                     head0, page_size, (int)num_pages, skip_single, (const uint4*)q, (uint4*)queries, q_units, q_pieces);
    if (err != cudaSuccess) return (int)err;
    err = lse_launch(attend_int4_kernel<D>, dim3((unsigned)((long long)tiles * heads * parts)), dim3(THREADS), smem, stream, map_q, map_k,
                     map_v, (__nv_bfloat16*)out, segment_start, first_pos, num_segments, n_q, group, heads, head0, tokens_a_tile,
                     scale * LOG2E, capacity, skip_single, parts, (const float2*)units, (const float*)q_units, part_o, part_ml);
    if (err != cudaSuccess) return (int)err;
    if (parts > 1) {
      err = lse_launch(combine_tiles_kernel<D>, dim3((unsigned)(tiles * heads), BM / 8), dim3(256), 0, stream, (const float*)part_o,
                       (const float2*)part_ml, (__nv_bfloat16*)out, segment_start, first_pos, num_segments, n_q, group, heads, head0,
                       tokens_a_tile, skip_single, parts);
      if (err != cudaSuccess) return (int)err;
    }
  }
  LSE_LAUNCH_CHECK();
}
}  // namespace

// 0: no bounded wait has given up since the library was loaded (synchronises the device).
extern "C" int lse_attention_int4_tc_status(void) {
  int value = 0;
  if (cudaMemcpyFromSymbol(&value, lse_attn_int4_tc_error, sizeof(int)) != cudaSuccess) return -1;
  return value;
}
extern "C" int lse_attention_int4_tc_status_async(int* host_dst, cudaStream_t stream) {
  return (int)cudaMemcpyFromSymbolAsync(host_dst, lse_attn_int4_tc_error, sizeof(int), 0, cudaMemcpyDeviceToHost, stream);
}
extern "C" int lse_attention_int4_tc_status_reset(void) {
  const int zero = 0;
  return (int)cudaMemcpyToSymbol(lse_attn_int4_tc_error, &zero, sizeof(int));
}

// q, out bfloat16 [tokens, n_q, head_dim]; the cache as int4_cache.cu leaves it; segment_start [S + 1]: first row of each request's
// portion, first_pos [S]: that row's position.  keys, values: float16 [heads_at_once, capacity * 128, head_dim], capacity = tiles of 128
// keys of all requests together, each request's rounded up (rows of a request that does not fit come out as NaN).  with_tiles: requests
// that have rows here, at most.  queries: float16 [tokens, n_q, head_dim].  powers: 4 heads_at_once capacity + tokens n_q words.  parts > 1
// (at most 8): scratch holds tokens * n_q * parts * (head_dim + 2) float32.
extern "C" int lse_paged_attention_prefill_int4(const void* q, const void* k_codes, const void* k_scales, const void* v_codes,
                                                const void* v_scales, void* out, const int* block_tables, int bt_stride,
                                                const int* segment_start, const int* first_pos, int num_segments, int tokens,
                                                long long num_pages, int n_q, int n_kv, int head_dim, int page_size, float scale,
                                                int skip_single, int with_tiles, int capacity, int heads_at_once, int parts, void* keys,
                                                void* values, void* queries, void* powers, float* scratch, cudaStream_t stream) {
  if (tokens <= 0 || num_segments <= 0) return 0;
  if ((head_dim != 64 && head_dim != 128) || n_kv <= 0 || n_q % n_kv || n_q / n_kv > BM || page_size <= 0 || num_pages <= 0 ||
      num_pages * page_size > 0x7fffffffLL || !(scale > 0.f) || capacity < 1 || heads_at_once < 1 || parts < 1 || parts > MAX_PARTS ||
      with_tiles < 1 || keys == nullptr || values == nullptr || queries == nullptr || powers == nullptr || (parts > 1 && scratch == nullptr) ||
      (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)keys | (uintptr_t)values |
        (uintptr_t)queries | (uintptr_t)powers | (uintptr_t)scratch) & 15) || (((uintptr_t)k_scales | (uintptr_t)v_scales) & 3))
    return LSE_ERR_BAD_ARGUMENT;
  if (heads_at_once > 65535 || (long long)heads_at_once * capacity * (BN / 8) > 0x7fffffffLL) return LSE_ERR_TOO_LARGE;
#define LSE_INT4_ARGS q, k_codes, k_scales, v_codes, v_scales, out, block_tables, bt_stride, segment_start, first_pos, num_segments, \
  tokens, num_pages, n_q, n_kv, page_size, scale, skip_single, with_tiles, capacity, heads_at_once, parts, keys, values, queries, powers, scratch, stream
  return head_dim == 128 ? launch_portions<128>(LSE_INT4_ARGS) : launch_portions<64>(LSE_INT4_ARGS);
#undef LSE_INT4_ARGS
}

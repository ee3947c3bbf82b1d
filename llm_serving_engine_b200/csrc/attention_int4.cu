// Attention of single rows (decoding) over keys and values held in 4 bits (int4_cache.cu), bfloat16 queries, head sizes 64, 128.
//
// With a key's row held as s (u - 8) + c the score is  s (q . (u - 8)) + c sum(q),  and a value's part of the output is
// p s (u - 8) + p c: the products run over the whole numbers u - 8, exact in bfloat16, the scale of a key multiplies the finished
// score, the scale of a value its probability, and c costs one multiply-add a score.  (Making values of the codes first would
// round them to bfloat16 and cost a multiply-add a value.)
//
// One block = (row, up to 8 query heads of a key/value head, a part of the keys); its warps take tiles of 16 keys in turn.  Keys ride the
// M side of mma.sync m16n8k16, heads the N side (S^T = K Q^T, O^T = V^T P^T).  Codes go from global memory straight into the
// registers that the instruction wants them in: which d a thread holds where is free as long as q, or the output, follows, so
//   keys    lane 4 g + t reads D / 8 consecutive bytes of keys g and g + 8: its d are t D / 4 .. ;
//   values  lane 4 g + t reads D / 16 consecutive bytes of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9: its d are g D / 8 .. .
// Each warp load covers whole 64-byte rows.  Two nibbles 16 bits apart become a pair of bfloat16 by one shift, one
// and-or (0x4300 | u is 128 + u) and one subtraction of 136, which is exact.
//
// What bounds it: bytes at first sight (D + 8 bytes a token and key/value head), but the codes are unpacked on the 32-bit
// integer pipe, half as wide as the FMA pipe: 120 of a tile's about 280 instructions.
// Softmax in base two, float32; the maximum in use is raised only when a score outgrows it by 2^8 (the sums carry the same
// factor, so the quotient is exact either way).  Probabilities are rounded to bfloat16 for the second product, as everywhere here.
#include <cooperative_groups.h>

#include "common.cuh"
#include "mma_common.cuh"

namespace cg = cooperative_groups;

LSE_CHECK_DEFINE(lse_check_attention_int4)

namespace {

constexpr int TILE = 16;         // keys a warp takes at a time
constexpr int HEADS = 8;         // query heads of a group that a block takes: the N side of the instruction
constexpr int WARPS = 4;
constexpr int BT_STAGE = 1024;   // block-table entries a block keeps in shared memory
constexpr int MAX_CLUSTER = 8;   // parts that are added up through distributed shared memory
constexpr int AHEAD = 2;         // tiles of a warp in flight
constexpr float RAISE = 8.0f;    // in powers of two

// Values u - 8 of the nibbles at bits 4 n of each half of x, as two bfloat16.
template <int N> __device__ __forceinline__ uint32_t whole_pair(uint32_t x) {
  uint32_t magic;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;\n" : "=r"(magic) : "r"(N == 0 ? x : x >> (4 * N)));   // (a & b) | c
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&magic), __floats2bfloat162_rn(136.f, 136.f));
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <int BYTES> struct Chunk;
template <> struct Chunk<4> { uint32_t w[1]; __device__ __forceinline__ void load(const unsigned char* p) { w[0] = __ldcg(reinterpret_cast<const uint32_t*>(p)); } };
template <> struct Chunk<8> { uint32_t w[2]; __device__ __forceinline__ void load(const unsigned char* p) { const uint2 v = __ldcg(reinterpret_cast<const uint2*>(p)); w[0] = v.x; w[1] = v.y; } };
template <> struct Chunk<16> { uint32_t w[4]; __device__ __forceinline__ void load(const unsigned char* p) { const uint4 v = __ldcg(reinterpret_cast<const uint4*>(p)); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; } };

template <int D> struct Codes {       // a tile as a lane holds it
  Chunk<D / 8> k[2];                  // keys g, g + 8
  Chunk<D / 16> v[4];                 // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
  uint32_t ks[2], vs[2];              // scale and centre of keys g, g + 8
};
__device__ __forceinline__ float2 halves(uint32_t w) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w)); }

// CLUSTER: the parts of one (row, heads) are the blocks of a thread-block cluster and are added up through distributed shared
// memory; else each leaves its part in global memory for combine_parts_kernel (num_splits = 1: neither).
template <int D, bool CLUSTER>
__global__ void __launch_bounds__(WARPS * 32, 4)
attn_decode_int4_kernel(const __nv_bfloat16* __restrict__ q, const unsigned char* __restrict__ k_codes,
                        const uint32_t* __restrict__ k_scales, const unsigned char* __restrict__ v_codes,
                        const uint32_t* __restrict__ v_scales, __nv_bfloat16* __restrict__ out, float* __restrict__ part_o,
                        float2* __restrict__ part_ml, const int* __restrict__ block_tables, int bt_stride,
                        const int* __restrict__ segment_of_token, const int* __restrict__ positions, int n_q, int n_kv,
                        int page_size, float scale_log2e, int num_splits, int num_pages, int num_segments) {
  constexpr int KW = D / 32, VW = D / 64, TILES_D = D / 16;
  __shared__ int bt_s[BT_STAGE];
  __shared__ float mg_o[WARPS][HEADS][D];
  __shared__ float mg_m[WARPS][HEADS], mg_l[WARPS][HEADS];
  __shared__ float recv_o[HEADS * D + MAX_CLUSTER], recv_m[MAX_CLUSTER * HEADS], recv_l[MAX_CLUSTER * HEADS];
  pdl_launch_dependents();
  // segments, positions and block tables are the step's own data: read before the wait for the kernels before
  const int t_row = blockIdx.x;
  const int group = n_q / n_kv, gchunks = (group + HEADS - 1) / HEADS;
  const int kvh = blockIdx.y / gchunks, g0 = (blockIdx.y % gchunks) * HEADS;
  const int gcount = min(HEADS, group - g0);
  const int split = blockIdx.z;
  const int seg = LSE_CHECKED(segment_of_token[t_row], -1, num_segments, -1, LSE_CHECK_SEGMENT);
  if (seg < 0) {                   // a padding row (all blocks of its cluster leave together)
    pdl_wait();                    // (a launch without work must not end before the one before it)
    return;
  }
  const int ctx = positions[t_row] + 1;
  const int* bt = block_tables + (size_t)seg * bt_stride;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int first_head = kvh * group + g0;

  const int total_tiles = (max(ctx, 0) + TILE - 1) / TILE;
  const int per_split = (total_tiles + num_splits - 1) / num_splits;
  const int tile_lo = min(total_tiles, split * per_split), tile_hi = min(total_tiles, tile_lo + per_split);
  const PageMath pm(page_size);
  const int first_page = pm.page(tile_lo * TILE);
  const int n_pages = tile_lo < tile_hi ? pm.page(min(ctx, tile_hi * TILE) - 1) - first_page + 1 : 0;
  const bool staged = n_pages <= BT_STAGE;
  if (staged)
    for (int i = tid; i < n_pages; i += WARPS * 32) bt_s[i] = LSE_CHECKED(bt[first_page + i], 0, num_pages, 0, LSE_CHECK_TABLE_ENTRY);
  __syncthreads();
  cg::cluster_group cluster = cg::this_cluster();
  if (CLUSTER) cluster.barrier_arrive();   // waited for before the first store into another block's memory
  pdl_wait();

  // queries as the B operand: head g of the group, this lane's d
  uint32_t qf[4 * KW];
  float qsum = 0.f;
  {
    uint32_t raw[D / 8];       // D / 4 values
    const bool live = g < gcount;
    const uint4* src = reinterpret_cast<const uint4*>(q + ((size_t)t_row * n_q + first_head + (live ? g : 0)) * D + t * (D / 4));
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const uint4 w = live ? src[i] : make_uint4(0, 0, 0, 0);
      raw[4 * i] = w.x; raw[4 * i + 1] = w.y; raw[4 * i + 2] = w.z; raw[4 * i + 3] = w.w;
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i) { const float2 v = halves(raw[i]); qsum += v.x + v.y; }
    // pair n of word w: the values 8 w + n and 8 w + n + 4
#pragma unroll
    for (int w = 0; w < KW; ++w) {
#pragma unroll
      for (int n = 0; n < 4; ++n)
        qf[4 * w + n] = __byte_perm(raw[4 * w + n / 2], raw[4 * w + 2 + n / 2], n & 1 ? 0x7632 : 0x5410);
    }
  }
  qsum += __shfl_xor_sync(0xffffffffu, qsum, 1);
  qsum += __shfl_xor_sync(0xffffffffu, qsum, 2);
  const float qs0 = __shfl_sync(0xffffffffu, qsum, 8 * t), qs1 = __shfl_sync(0xffffffffu, qsum, 8 * t + 4);   // heads 2 t, 2 t + 1

  auto place_of = [&](int j) {           // row of the cache that key j lies in
    const int logical = pm.page(j);
    const int page = staged ? bt_s[logical - first_page] : LSE_CHECKED(bt[logical], 0, num_pages, 0, LSE_CHECK_TABLE_ENTRY);
    return ((size_t)page * n_kv + kvh) * page_size + pm.offset(j);
  };
  const bool page_tiles = (page_size % TILE) == 0;   // a tile never straddles pages
  auto fetch = [&](int tile, Codes<D>& c) {
    const int j0 = tile * TILE;
    size_t kp[2], vp[4];
    if (page_tiles) {      // a page that holds a tile's first key has room for all sixteen: nothing beyond it is read
      const size_t p0 = place_of(j0);
      kp[0] = p0 + g; kp[1] = p0 + g + 8;
      vp[0] = p0 + 2 * t; vp[1] = vp[0] + 1; vp[2] = vp[0] + 8; vp[3] = vp[0] + 9;
    } else {               // keys beyond the context are read from the last one's row and hidden below
      const int last = ctx - 1;
      kp[0] = place_of(min(j0 + g, last)); kp[1] = place_of(min(j0 + g + 8, last));
      vp[0] = place_of(min(j0 + 2 * t, last)); vp[1] = place_of(min(j0 + 2 * t + 1, last));
      vp[2] = place_of(min(j0 + 2 * t + 8, last)); vp[3] = place_of(min(j0 + 2 * t + 9, last));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      c.k[i].load(k_codes + kp[i] * (D / 2) + t * (D / 8));
      c.ks[i] = __ldcg(k_scales + kp[i]);
      c.vs[i] = __ldcg(v_scales + kp[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) c.v[i].load(v_codes + vp[i] * (D / 2) + g * (D / 16));
  };

  float acc[TILES_D][4];
#pragma unroll
  for (int i = 0; i < TILES_D; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, o0 = 0.f, o1 = 0.f;   // heads 2 t, 2 t + 1; sums over this lane's keys

  auto work = [&](int tile, const Codes<D>& c) {
    float s[4] = {0.f, 0.f, 0.f, 0.f}, s_odd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      const uint32_t a[4] = {whole_pair<0>(c.k[0].w[w]), whole_pair<0>(c.k[1].w[w]), whole_pair<1>(c.k[0].w[w]), whole_pair<1>(c.k[1].w[w])};
      const uint32_t b[4] = {whole_pair<2>(c.k[0].w[w]), whole_pair<2>(c.k[1].w[w]), whole_pair<3>(c.k[0].w[w]), whole_pair<3>(c.k[1].w[w])};
      mma_bf16(s, a, qf[4 * w], qf[4 * w + 1]);
      mma_bf16(s_odd, b, qf[4 * w + 2], qf[4 * w + 3]);
    }
    const int j0 = tile * TILE + g;
    const bool see0 = j0 < ctx, see1 = j0 + 8 < ctx;
    const float2 k0 = halves(c.ks[0]), k1 = halves(c.ks[1]);
    const float a0 = k0.x * scale_log2e, b0 = k0.y * scale_log2e, a1 = k1.x * scale_log2e, b1 = k1.y * scale_log2e;
    s[0] = see0 ? fmaf(s[0] + s_odd[0], a0, b0 * qs0) : -INFINITY;
    s[1] = see0 ? fmaf(s[1] + s_odd[1], a0, b0 * qs1) : -INFINITY;
    s[2] = see1 ? fmaf(s[2] + s_odd[2], a1, b1 * qs0) : -INFINITY;
    s[3] = see1 ? fmaf(s[3] + s_odd[3], a1, b1 * qs1) : -INFINITY;
    float mx0 = fmaxf(s[0], s[2]), mx1 = fmaxf(s[1], s[3]);
    // (a first tile, at maxima of minus infinity, always takes this way; its first key lies inside the context)
    if (__any_sync(0xffffffffu, mx0 > m0 + RAISE || mx1 > m1 + RAISE)) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, o));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, o));
      }
      const float n0 = fmaxf(m0, mx0), n1 = fmaxf(m1, mx1);
      const float c0 = m0 == -INFINITY ? 0.f : fast_exp2(m0 - n0), c1 = m1 == -INFINITY ? 0.f : fast_exp2(m1 - n1);
      m0 = n0; m1 = n1;
      l0 *= c0; l1 *= c1; o0 *= c0; o1 *= c1;
#pragma unroll
      for (int i = 0; i < TILES_D; ++i) { acc[i][0] *= c0; acc[i][1] *= c1; acc[i][2] *= c0; acc[i][3] *= c1; }
    }
    // a head whose scores are all minus infinity so far weighs nothing (and must not become infinity minus infinity)
    const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
    const float p0 = fast_exp2(s[0] - r0), p1 = fast_exp2(s[1] - r1), p2 = fast_exp2(s[2] - r0), p3 = fast_exp2(s[3] - r1);
    // what lies behind the last key may be anything, not a number among it: its scale and centre are left out
    const float2 v0 = see0 ? halves(c.vs[0]) : make_float2(0.f, 0.f), v1 = see1 ? halves(c.vs[1]) : make_float2(0.f, 0.f);
    l0 += p0 + p2; l1 += p1 + p3;
    o0 = fmaf(p0, v0.y, fmaf(p2, v1.y, o0));
    o1 = fmaf(p1, v0.y, fmaf(p3, v1.y, o1));
    // P^T as the B operand: [key][head] pieces transposed
    const uint32_t pb0 = movmatrix_trans(pack_bf16(p0 * v0.x, p1 * v0.x)), pb1 = movmatrix_trans(pack_bf16(p2 * v1.x, p3 * v1.x));
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      const uint32_t xl = __byte_perm(c.v[0].w[w], c.v[1].w[w], 0x5410), xh = __byte_perm(c.v[0].w[w], c.v[1].w[w], 0x7632);
      const uint32_t yl = __byte_perm(c.v[2].w[w], c.v[3].w[w], 0x5410), yh = __byte_perm(c.v[2].w[w], c.v[3].w[w], 0x7632);
      { const uint32_t a[4] = {whole_pair<0>(xl), whole_pair<0>(xh), whole_pair<0>(yl), whole_pair<0>(yh)}; mma_bf16(acc[4 * w], a, pb0, pb1); }
      { const uint32_t a[4] = {whole_pair<1>(xl), whole_pair<1>(xh), whole_pair<1>(yl), whole_pair<1>(yh)}; mma_bf16(acc[4 * w + 1], a, pb0, pb1); }
      { const uint32_t a[4] = {whole_pair<2>(xl), whole_pair<2>(xh), whole_pair<2>(yl), whole_pair<2>(yh)}; mma_bf16(acc[4 * w + 2], a, pb0, pb1); }
      { const uint32_t a[4] = {whole_pair<3>(xl), whole_pair<3>(xh), whole_pair<3>(yl), whole_pair<3>(yh)}; mma_bf16(acc[4 * w + 3], a, pb0, pb1); }
    }
  };

  // this warp's tiles: tile_lo + warp, + WARPS, ...
  Codes<D> held[AHEAD];
  int tile = tile_lo + warp;
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (tile + i * WARPS < tile_hi) fetch(tile + i * WARPS, held[i]);
  while (tile < tile_hi) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (tile < tile_hi) {      // the same in all lanes
        const Codes<D> now = held[i];
        if (tile + AHEAD * WARPS < tile_hi) fetch(tile + AHEAD * WARPS, held[i]);
        work(tile, now);
        tile += WARPS;
      }
    }
  }

  // sums of a head over the lanes that hold it, then the warps' parts
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, o); l1 += __shfl_xor_sync(0xffffffffu, l1, o);
    o0 += __shfl_xor_sync(0xffffffffu, o0, o); o1 += __shfl_xor_sync(0xffffffffu, o1, o);
  }
#pragma unroll
  for (int i = 0; i < TILES_D; ++i) {
    const int d = g * (D / 8) + 8 * (i / 4) + i % 4;
    mg_o[warp][2 * t][d] = acc[i][0] + o0; mg_o[warp][2 * t + 1][d] = acc[i][1] + o1;
    mg_o[warp][2 * t][d + 4] = acc[i][2] + o0; mg_o[warp][2 * t + 1][d + 4] = acc[i][3] + o1;
  }
  if (lane < 4) { mg_m[warp][2 * t] = m0; mg_m[warp][2 * t + 1] = m1; mg_l[warp][2 * t] = l0; mg_l[warp][2 * t + 1] = l1; }
  __syncthreads();
  if (CLUSTER) cluster.barrier_wait();
  const int push_per = (gcount * D + num_splits - 1) / num_splits;   // block r of a cluster finishes outputs r * push_per ..
  for (int e = tid; e < gcount * D; e += WARPS * 32) {
    const int h = e / D, d = e % D;
    float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) M = fmaxf(M, mg_m[w][h]);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float wgt = mg_m[w][h] == -INFINITY ? 0.f : fast_exp2(mg_m[w][h] - M);
      // a warp whose maximum is minus infinity may still carry a NaN of a key that is not a number
      L += mg_m[w][h] == -INFINITY ? mg_l[w][h] : mg_l[w][h] * wgt;
      O += mg_m[w][h] == -INFINITY ? mg_o[w][h][d] : mg_o[w][h][d] * wgt;
    }
    const int head = first_head + h;
    if (num_splits == 1) {
      out[((size_t)t_row * n_q + head) * D + d] = __float2bfloat16_rn(ctx > 0 ? O / L : 0.f);
    } else if (CLUSTER) {
      const int owner = e / push_per;
      cluster.map_shared_rank(recv_o, owner)[split * push_per + e % push_per] = O;
      if (d < num_splits) {
        cluster.map_shared_rank(recv_m, d)[split * HEADS + h] = M;
        cluster.map_shared_rank(recv_l, d)[split * HEADS + h] = L;
      }
    } else {
      const size_t at = ((size_t)t_row * n_q + head) * num_splits + split;
      part_o[at * D + d] = O;
      if (d == 0) part_ml[at] = make_float2(M, L);
    }
  }
  if (!CLUSTER) return;
  cluster.sync();      // every part is where it is finished
  const int items = gcount * D, mine = (int)cluster.block_rank() * push_per;
  for (int e = mine + tid; e < min(items, mine + push_per); e += WARPS * 32) {
    const int h = e / D, d = e % D;
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (int r = 0; r < num_splits; ++r) M = fmaxf(M, recv_m[r * HEADS + h]);
    for (int r = 0; r < num_splits; ++r) {
      const float mr = recv_m[r * HEADS + h], w = mr == -INFINITY ? 1.f : fast_exp2(mr - M);
      L += recv_l[r * HEADS + h] * w;
      O += recv_o[r * push_per + (e - mine)] * w;
    }
    out[((size_t)t_row * n_q + first_head + h) * D + d] = __float2bfloat16_rn(ctx > 0 ? O / L : 0.f);
  }
}

// Adds up the parts of a row's head: part_o [row][head][part][D] relative to their maxima, part_ml (maximum, sum).  One block =
// (row, head); a warp takes every eighth part, a lane D / 32 neighbouring values.
template <int D>
__global__ void __launch_bounds__(256)
combine_parts_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, const int* __restrict__ segment_of_token,
                     const int* __restrict__ positions, __nv_bfloat16* __restrict__ out, int parts) {
  constexpr int V = D / 32;
  __shared__ float sum_o[8][D], sum_l[8], top[8];
  const int row = blockIdx.x, head = blockIdx.y, n_q = gridDim.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  pdl_wait();
  if (segment_of_token[row] < 0) return;
  const size_t base = ((size_t)row * n_q + head) * parts;
  float M = -INFINITY;
  for (int p = threadIdx.x; p < parts; p += 256) M = fmaxf(M, part_ml[base + p].x);
  M = warp_max(M);
  if (lane == 0) top[warp] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) M = fmaxf(M, top[w]);
  float o[V], L = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = 0.f;
#pragma unroll 4
  for (int p = warp; p < parts; p += 8) {
    const float2 ml = part_ml[base + p];
    const float w = ml.x == -INFINITY ? 1.f : fast_exp2(ml.x - M);     // (sums of zero, or not a number)
    L = fmaf(ml.y, w, L);
    const float* src = part_o + (base + p) * D + lane * V;
    float v[V];
    if (V == 4) { const float4 x = *reinterpret_cast<const float4*>(src); v[0] = x.x; v[1] = x.y; v[2 % V] = x.z; v[3 % V] = x.w; }
    else { const float2 x = *reinterpret_cast<const float2*>(src); v[0] = x.x; v[1] = x.y; }
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = fmaf(v[i], w, o[i]);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) sum_o[warp][lane * V + i] = o[i];
  if (lane == 0) sum_l[warp] = L;
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += 256) {
    float O = 0.f, total = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) { O += sum_o[w][d]; total += sum_l[w]; }
    out[((size_t)row * n_q + head) * D + d] = __float2bfloat16_rn(positions[row] >= 0 ? O / total : 0.f);
  }
}

template <int D>
int launch_decode(const void* q, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, void* out,
                  float* scratch, const int* block_tables, int bt_stride, const int* segment_of_token, const int* positions,
                  int tokens, int n_q, int n_kv, int page_size, float scale, int num_splits, long long num_pages,
                  int num_segments, cudaStream_t stream) {
  const int gchunks = (n_q / n_kv + HEADS - 1) / HEADS;
  const dim3 grid((unsigned)tokens, (unsigned)(n_kv * gchunks), (unsigned)num_splits);
  const bool cluster = num_splits > 1 && num_splits <= MAX_CLUSTER;
  float* part_o = scratch;
  float2* part_ml = cluster || num_splits == 1 ? nullptr : reinterpret_cast<float2*>(scratch + (size_t)tokens * n_q * num_splits * D);
#define LSE_INT4_DECODE(CLUSTER, WIDTH)                                                                                      \
  lse_launch_cluster(attn_decode_int4_kernel<D, CLUSTER>, grid, dim3(WARPS * 32), 0, stream, WIDTH, (const __nv_bfloat16*)q,    \
                     (const unsigned char*)k_codes, (const uint32_t*)k_scales, (const unsigned char*)v_codes,                  \
                     (const uint32_t*)v_scales, (__nv_bfloat16*)out, part_o, part_ml, block_tables, bt_stride,                 \
                     segment_of_token, positions, n_q, n_kv, page_size, scale * LOG2E, num_splits, (int)num_pages, num_segments)
  cudaError_t err = cluster ? LSE_INT4_DECODE(true, (unsigned)num_splits) : LSE_INT4_DECODE(false, 1u);
#undef LSE_INT4_DECODE
  if (err != cudaSuccess) return (int)err;
  if (num_splits > MAX_CLUSTER) {
    err = lse_launch(combine_parts_kernel<D>, dim3((unsigned)tokens, (unsigned)n_q), dim3(256), 0, stream, (const float*)part_o,
                     (const float2*)part_ml, segment_of_token, positions, (__nv_bfloat16*)out, num_splits);
    if (err != cudaSuccess) return (int)err;
  }
  LSE_LAUNCH_CHECK();
}

}  // namespace

// q, out bfloat16 [tokens, n_q, head_dim]; the cache as int4_cache.cu leaves it; block_tables [num_segments, bt_stride].
// segment_of_token < 0: a padding row, left as it was; a row at a negative position sees no key and gets zeros.
// num_splits parts of the keys a row; more than 8: `scratch` holds tokens * n_q * num_splits * (head_dim + 2) float32.
extern "C" int lse_paged_attention_decode_int4(const void* q, const void* k_codes, const void* k_scales, const void* v_codes,
                                               const void* v_scales, void* out, float* scratch, const int* block_tables,
                                               int bt_stride, const int* segment_of_token, const int* positions, int tokens,
                                               int n_q, int n_kv, int head_dim, int page_size, float scale, int num_splits,
                                               long long num_pages, int num_segments, cudaStream_t stream) {
  if (tokens <= 0) return 0;
  if ((head_dim != 64 && head_dim != 128) || n_kv <= 0 || n_q % n_kv || page_size <= 0 || num_pages <= 0 || num_splits < 1 ||
      num_pages * page_size > 0x7fffffffLL || (num_splits > MAX_CLUSTER && scratch == nullptr) ||
      (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_codes | (uintptr_t)k_scales | (uintptr_t)v_codes | (uintptr_t)v_scales | (uintptr_t)scratch) & 15))
    return LSE_ERR_BAD_ARGUMENT;
  if (num_splits > 65535 || (long long)n_kv * ((n_q / n_kv + HEADS - 1) / HEADS) > 65535) return LSE_ERR_TOO_LARGE;
#define LSE_INT4_ARGS q, k_codes, k_scales, v_codes, v_scales, out, scratch, block_tables, bt_stride, segment_of_token, positions, \
  tokens, n_q, n_kv, page_size, scale, num_splits, num_pages, num_segments, stream
  return head_dim == 128 ? launch_decode<128>(LSE_INT4_ARGS) : launch_decode<64>(LSE_INT4_ARGS);
#undef LSE_INT4_ARGS
}

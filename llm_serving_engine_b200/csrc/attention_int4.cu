// Attention of single rows (decoding) over keys and values held in 4 bits (int4_cache.cu), bfloat16 queries, head sizes 64, 128.
//
// With a key's row held as s (u - 8) + c the score is  s (q . (u - 8)) + c sum(q),  and a value's part of the output is
// p s (u - 8) + p c: the products run over the whole numbers u - 8, exact in bfloat16, the scale of a key multiplies the finished
// score, the scale of a value its probability, and c costs one multiply-add a score.  (Making values of the codes first would
// round them to bfloat16 and cost a multiply-add a value.)
//
// One block = (row, up to 8 query heads of a key/value head, a part of the keys); its warps take tiles of 16 keys in turn.  Keys ride the
// M side of mma.sync m16n8k16, heads the N side (S^T = K Q^T, O^T = V^T P^T).  Every warp keeps a ring of tiles of its own, as they lie in
// the cache, filled by cp.async, and reads them into the registers that the instruction wants them in: which d a thread holds
// where is free as long as q, or the output, follows, so
//   keys    lane 4 g + t reads D / 8 consecutive bytes of keys g and g + 8: its d are t D / 4 .. ;
//   values  lane 4 g + t reads D / 16 consecutive bytes of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9: its d are g D / 8 .. .
// Two nibbles 16 bits apart become a pair of bfloat16 by one shift and one and-or.  For
// keys that is 16 + u, and the accumulators start at -24 sum(q); float32 rounds sums of 24 |q| instead of 8 |q| then, which is far
// below the rounding of a probability.  Values lose the offset by a subtraction, which is exact: sums of
// values run over the whole context, and an offset there would cost what the result loses by averaging.
// Softmax in base two, float32; the maximum in use is raised only when a score outgrows it by 2^8 (the sums carry the same
// factor, so the quotient is exact either way).  What is rounded to bfloat16 for the second product is a probability times its
// value's scale: a term is off by 2^-8 of s (u - 8), a thirty-second of a step of the codes at most.
// What bounds it: a row's chain of waits (positions, block table, tiles, the parts' meeting), then instructions, some 400 a warp and tile
// all told (half of them make bfloat16 of the codes).  64 rows of 12 / 2 heads of 128 over 950 to 2,850 keys (33.5 MB): 15.4 us, over
// 2,000 each 13.8 (24.1 over bfloat16 pages); 16 rows over 8,000: 17.7 (24.0); one row of 28 / 4 heads over 30,000 keys (16.3 MB): 13.5 us
// (18.6), 4 of them the second launch.
#include <cooperative_groups.h>

#include "common.cuh"
#include "mma_common.cuh"
#include "smem_allowance.cuh"

namespace cg = cooperative_groups;

LSE_CHECK_DEFINE(lse_check_attention_int4)

namespace {

constexpr int SIDE = 16, SIDES = 1, TILE = SIDE * SIDES;     // keys a warp takes at a time: SIDES times the instruction's M side
constexpr int HEADS = 8;         // query heads of a group that a block takes: the N side of the instruction
constexpr int WARPS = 4, BLOCKS = 4;     // warps of a block, blocks of an SM
constexpr int STAGE = 256;       // tiles whose places a block keeps in shared memory at a time
constexpr int MAX_CLUSTER = 8;   // parts that are added up through distributed shared memory
constexpr int STAGES = 4;        // tiles of a warp that are on their way or worked on
constexpr float RAISE = 8.0f;    // in powers of two

// Nibbles at bits 4 N of each half of x as two bfloat16: 16 + u (a shift to the mantissa's upper bits and one and-or; 24 too much,
// which the keys' accumulators start without) ...
template <int N> __device__ __forceinline__ uint32_t raised_pair(uint32_t x) {
  uint32_t v;
  asm("lop3.b32 %0, %1, 0x00780078, 0x41804180, 0xea;\n" : "=r"(v) : "r"(N == 0 ? x << 3 : x >> (4 * N - 3)));   // (a & b) | c
  return v;
}
// ... and u - 8 (128 + u, minus 136).
template <int N> __device__ __forceinline__ uint32_t whole_pair(uint32_t x) {
  uint32_t magic;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;\n" : "=r"(magic) : "r"(N == 0 ? x : x >> (4 * N)));   // (a & b) | c
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&magic), __floats2bfloat162_rn(136.f, 136.f));
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ float2 halves(uint32_t w) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w)); }

struct PageMath16 {     // page and offset of a key; shift < 0: the page size is no power of two
  int size, shift;
  __device__ __forceinline__ int page(int j) const { return shift >= 0 ? j >> shift : j / size; }
  __device__ __forceinline__ int offset(int j) const { return shift >= 0 ? j & (size - 1) : j % size; }
};
struct Cache4 {
  const unsigned char *k_codes, *v_codes;
  const uint32_t *k_scales, *v_scales;
  PageMath16 pm;
  int n_kv, num_pages;
};
// A tile in a warp's ring: codes of its keys, of its values, their scales.  Rows lie one after the other in lines of 128 bytes; the 16-byte
// pieces of a line of values are permuted by the line's number, so that reading two columns of every second row meets every bank once.
template <int D> struct TileBytes { static constexpr int CODES = TILE * D / 2, ALL = 2 * CODES + 2 * TILE * 4; };
template <int D, int UNIT> struct Shared4 {
  union {
    unsigned char ring[WARPS][STAGES][TileBytes<D>::ALL];
    float4 o[WARPS][D / 16][32];                            // the warps' results, once the ring has been worked through (see below)
  };
  uint32_t unit[UNIT == 1 ? 1 : STAGE * (TILE / UNIT)];     // places of a stage's units, in units
  float m[WARPS][HEADS], l[WARPS][HEADS];
};
template <int D> __device__ __forceinline__ int value_piece(int i) {     // where piece i (16 bytes) of a tile's values lies
  return i ^ (2 * (i >> 3 & (D == 128 ? 3 : 1)));
}

// The keys of tiles tile_lo .. tile_hi - 1 of a request (block table bt, ctx keys) for the query heads at q (gcount of them, rows of D)
// of key/value head kvh: every warp's outputs, maxima and sums are left in `sh`, and the block has met after that.
// UNIT: keys that certainly lie side by side in the cache (16, 8, or 1: by the page size).
template <int D, int UNIT>
__device__ __forceinline__ void attend_tiles(Shared4<D, UNIT>& sh, const Cache4& cache, const __nv_bfloat16* q, int gcount,
                                             int kvh, const int* __restrict__ bt, int ctx, int tile_lo, int tile_hi, float scale_log2e,
                                             bool wait) {
  constexpr int KW = D / 32, VW = D / 64, TILES_D = D / 16;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const PageMath16 pm = cache.pm;
  const int page_size = pm.size, n_kv = cache.n_kv;
  const unsigned char *k_codes = cache.k_codes, *v_codes = cache.v_codes;
  const uint32_t *k_scales = cache.k_scales, *v_scales = cache.v_scales;
  auto page_of = [&](int logical) { return LSE_CHECKED(bt[logical], 0, cache.num_pages, 0, LSE_CHECK_TABLE_ENTRY); };
  // places of the units of tiles from .. on, as many as there is room for; a unit behind the last key's takes the place of that one
  auto stage_units = [&](int from) {
    constexpr int A_TILE = TILE / UNIT;
    const int n = min(STAGE, tile_hi - from) * A_TILE;
    for (int i = tid; i < n; i += WARPS * 32) {
      const int key = min((from * A_TILE + i) * UNIT, ctx - 1);
      sh.unit[i] = ((uint32_t)page_of(pm.page(key)) * (uint32_t)n_kv + (uint32_t)kvh) * (uint32_t)(page_size / UNIT) + (uint32_t)(pm.offset(key) / UNIT);
    }
  };
  if (UNIT > 1) stage_units(tile_lo);
  __syncthreads();
  if (wait) pdl_wait();

  unsigned char* const ring = sh.ring[warp][0];
  const uint32_t ring_at = smem_u32(ring);
  constexpr int CODES = TileBytes<D>::CODES, ALL = TileBytes<D>::ALL, PIECES = CODES / 16, ROW = D / 2;
  // tile -> a slot of this warp's ring, one group of copies
  auto fetch = [&](int tile, int from, int slot) {
    const uint32_t dst = ring_at + (uint32_t)(slot * ALL);
    if (UNIT > 1) {
      constexpr int UNITS = TILE / UNIT, A_UNIT = UNIT * ROW / 16;       // units of a tile, pieces of a unit's codes
      const uint32_t* units = sh.unit + UNITS * (tile - from);
#pragma unroll
      for (int i = 0; i < PIECES; i += 32) {
        // (a unit's pieces are whole warps' where there are as many; else a warp's lanes hold several units)
        const int piece = i + lane;
        const size_t at = (size_t)units[A_UNIT % 32 == 0 ? i / A_UNIT : piece / A_UNIT] * (UNIT * ROW) + (A_UNIT % 32 == 0 ? i % A_UNIT + lane : piece % A_UNIT) * 16;
        cp_async16(dst + piece * 16, k_codes + at, true);
        cp_async16(dst + CODES + value_piece<D>(piece) * 16, v_codes + at, true);
      }
      if (lane < TILE / 2) {      // four keys' scales each
        const uint32_t* src = lane < TILE / 4 ? k_scales : v_scales;
        const int key = (lane & (TILE / 4 - 1)) * 4;
        cp_async16(dst + 2 * CODES + lane * 16, src + (size_t)units[key / UNIT] * UNIT + key % UNIT, true);
      }
    } else {       // pages of any size, key by key; keys behind the last are read from the last one's row and hidden below
      const int j0 = tile * TILE, last = ctx - 1;
      auto row_of = [&](int j) { j = min(j, last); return ((size_t)page_of(pm.page(j)) * n_kv + kvh) * page_size + pm.offset(j); };
#pragma unroll
      for (int i = 0; i < PIECES; i += 32) {
        const int piece = i + lane;
        const size_t at = row_of(j0 + piece / (ROW / 16)) * ROW + (size_t)(piece % (ROW / 16)) * 16;
        cp_async16(dst + piece * 16, k_codes + at, true);
        cp_async16(dst + CODES + value_piece<D>(piece) * 16, v_codes + at, true);
      }
      if (lane < TILE) {
        const size_t row = row_of(j0 + lane);
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(dst + 2 * CODES + lane * 4), "l"(k_scales + row));
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(dst + 2 * CODES + (TILE + lane) * 4), "l"(v_scales + row));
      }
    }
  };
  auto words = [](const unsigned char* p, uint32_t* w, int n) {
    if (n == 4) { const uint4 v = *reinterpret_cast<const uint4*>(p); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
    else if (n == 2) { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
    else w[0] = *reinterpret_cast<const uint32_t*>(p);
  };

  // the first tiles of a stage set out
  auto fill = [&](int from, int to) {
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
      if (from + warp + i * WARPS < to) fetch(from + warp + i * WARPS, from, i);
      cp_async_commit();
    }
  };
  fill(tile_lo, min(tile_hi, tile_lo + STAGE));

  // queries as the B operand: head g of the group, this lane's d
  uint32_t qf[4 * KW];
  float qsum = 0.f;
  {
    uint32_t raw[D / 8];       // D / 4 values
    const bool live = g < gcount;
    const uint4* src = reinterpret_cast<const uint4*>(q + (live ? g : 0) * D + t * (D / 4));
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
  const float sum0 = __shfl_sync(0xffffffffu, qsum, 8 * t), sum1 = __shfl_sync(0xffffffffu, qsum, 8 * t + 4);   // heads 2 t, 2 t + 1
  const float start0 = -24.f * sum0, start1 = -24.f * sum1, qs0 = sum0 * scale_log2e, qs1 = sum1 * scale_log2e;

  float acc[TILES_D][4];
#pragma unroll
  for (int i = 0; i < TILES_D; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, o0 = 0.f, o1 = 0.f;   // heads 2 t, 2 t + 1; sums over this lane's keys
  float r0 = 0.f, r1 = 0.f;       // the maxima as they are taken off the scores: zero while a head has seen minus infinity only

  // this lane's places in a side of a tile: keys g and g + 8 from byte t D / 8 on, values 2 t, 2 t + 1, 2 t + 8, 2 t + 9 from byte g D / 16 on
  const int k_place = g * ROW + t * (D / 8);
  int v_place[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = (2 * t + (i & 1) + 8 * (i >> 1)) * ROW + g * (D / 16);
    v_place[i] = CODES + value_piece<D>(at >> 4) * 16 + (at & 15);
  }
  auto work = [&](int tile, const unsigned char* c) {
    const uint32_t* scales = reinterpret_cast<const uint32_t*>(c + 2 * CODES);
    float s[SIDES][4];
    float2 v[SIDES][2];
#pragma unroll
    for (int i = 0; i < SIDES; ++i) {
      uint32_t kw[2][KW];
      words(c + k_place + (SIDE * i) * ROW, kw[0], KW);
      words(c + k_place + (SIDE * i + 8) * ROW, kw[1], KW);
      s[i][0] = s[i][2] = start0; s[i][1] = s[i][3] = start1;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const uint32_t a[4] = {raised_pair<0>(kw[0][w]), raised_pair<0>(kw[1][w]), raised_pair<1>(kw[0][w]), raised_pair<1>(kw[1][w])};
        const uint32_t b[4] = {raised_pair<2>(kw[0][w]), raised_pair<2>(kw[1][w]), raised_pair<3>(kw[0][w]), raised_pair<3>(kw[1][w])};
        mma_bf16(s[i], a, qf[4 * w], qf[4 * w + 1]);
        mma_bf16(s[i], b, qf[4 * w + 2], qf[4 * w + 3]);
      }
    }
#pragma unroll
    for (int i = 0; i < SIDES; ++i) {
      const float2 k0 = halves(scales[SIDE * i + g]), k1 = halves(scales[SIDE * i + g + 8]);
      v[i][0] = halves(scales[TILE + SIDE * i + g]); v[i][1] = halves(scales[TILE + SIDE * i + g + 8]);
      const float a0 = k0.x * scale_log2e, a1 = k1.x * scale_log2e;
      s[i][0] = fmaf(s[i][0], a0, k0.y * qs0); s[i][1] = fmaf(s[i][1], a0, k0.y * qs1);
      s[i][2] = fmaf(s[i][2], a1, k1.y * qs0); s[i][3] = fmaf(s[i][3], a1, k1.y * qs1);
    }
    if ((tile + 1) * TILE > ctx) {     // what lies behind the last key may be anything, not a number among it
#pragma unroll
      for (int i = 0; i < SIDES; ++i) {
        const int j0 = tile * TILE + SIDE * i + g;
        if (j0 >= ctx) { s[i][0] = s[i][1] = -INFINITY; v[i][0] = make_float2(0.f, 0.f); }
        if (j0 + 8 >= ctx) { s[i][2] = s[i][3] = -INFINITY; v[i][1] = make_float2(0.f, 0.f); }
      }
    }
    float mx0 = fmaxf(s[0][0], s[0][2]), mx1 = fmaxf(s[0][1], s[0][3]);
#pragma unroll
    for (int i = 1; i < SIDES; ++i) { mx0 = fmaxf(mx0, fmaxf(s[i][0], s[i][2])); mx1 = fmaxf(mx1, fmaxf(s[i][1], s[i][3])); }
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
      r0 = n0 == -INFINITY ? 0.f : n0; r1 = n1 == -INFINITY ? 0.f : n1;
      l0 *= c0; l1 *= c1; o0 *= c0; o1 *= c1;
#pragma unroll
      for (int i = 0; i < TILES_D; ++i) { acc[i][0] *= c0; acc[i][1] *= c1; acc[i][2] *= c0; acc[i][3] *= c1; }
    }
    uint32_t pb[SIDES][2];       // P^T as the B operand: [key][head] pieces transposed
#pragma unroll
    for (int i = 0; i < SIDES; ++i) {
      const float p0 = fast_exp2(s[i][0] - r0), p1 = fast_exp2(s[i][1] - r1), p2 = fast_exp2(s[i][2] - r0), p3 = fast_exp2(s[i][3] - r1);
      l0 += p0 + p2; l1 += p1 + p3;
      o0 = fmaf(p0, v[i][0].y, fmaf(p2, v[i][1].y, o0));
      o1 = fmaf(p1, v[i][0].y, fmaf(p3, v[i][1].y, o1));
      pb[i][0] = movmatrix_trans(pack_bf16(p0 * v[i][0].x, p1 * v[i][0].x));
      pb[i][1] = movmatrix_trans(pack_bf16(p2 * v[i][1].x, p3 * v[i][1].x));
    }
#pragma unroll
    for (int i = 0; i < SIDES; ++i) {
      uint32_t vw[4][VW];
#pragma unroll
      for (int k = 0; k < 4; ++k) words(c + v_place[k] + i * (SIDE * ROW), vw[k], VW);
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        const uint32_t xl = __byte_perm(vw[0][w], vw[1][w], 0x5410), xh = __byte_perm(vw[0][w], vw[1][w], 0x7632);
        const uint32_t yl = __byte_perm(vw[2][w], vw[3][w], 0x5410), yh = __byte_perm(vw[2][w], vw[3][w], 0x7632);
        { const uint32_t a[4] = {whole_pair<0>(xl), whole_pair<0>(xh), whole_pair<0>(yl), whole_pair<0>(yh)}; mma_bf16(acc[4 * w], a, pb[i][0], pb[i][1]); }
        { const uint32_t a[4] = {whole_pair<1>(xl), whole_pair<1>(xh), whole_pair<1>(yl), whole_pair<1>(yh)}; mma_bf16(acc[4 * w + 1], a, pb[i][0], pb[i][1]); }
        { const uint32_t a[4] = {whole_pair<2>(xl), whole_pair<2>(xh), whole_pair<2>(yl), whole_pair<2>(yh)}; mma_bf16(acc[4 * w + 2], a, pb[i][0], pb[i][1]); }
        { const uint32_t a[4] = {whole_pair<3>(xl), whole_pair<3>(xh), whole_pair<3>(yl), whole_pair<3>(yh)}; mma_bf16(acc[4 * w + 3], a, pb[i][0], pb[i][1]); }
      }
    }
  };

  // this warp's tiles of a stage: its first + warp, + WARPS, ...
  for (int from = tile_lo; from < tile_hi; from += STAGE) {
    const int to = min(tile_hi, from + STAGE);
    if (from > tile_lo) {
      __syncthreads();
      if (UNIT > 1) stage_units(from);
      __syncthreads();
      fill(from, to);
    }
    int slot = 0;
    for (int tile = from + warp; tile < to; tile += WARPS) {
      cp_async_wait<STAGES - 2>();     // all but the newest STAGES - 2 groups have landed: this tile is there
      __syncwarp();                    // (every lane's copies; and every lane is done with the tile before)
      const int ahead = tile + (STAGES - 1) * WARPS;
      if (ahead < to) fetch(ahead, from, slot == 0 ? STAGES - 1 : slot - 1);     // into the slot of the tile before
      cp_async_commit();
      work(tile, ring + slot * ALL);
      slot = slot == STAGES - 1 ? 0 : slot + 1;
    }
    cp_async_wait<0>();
    __syncwarp();
  }

  __syncthreads();     // (the results take the ring's place)
  // Sums of a head over the lanes that hold it, then the warps' parts.  A lane leaves its results as fours of neighbouring d, each
  // lane its own 16 bytes (o[warp][piece][lane], piece = (8 d's of the lane, head 2 t or 2 t + 1, half)): no two lanes share a bank.
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, o); l1 += __shfl_xor_sync(0xffffffffu, l1, o);
    o0 += __shfl_xor_sync(0xffffffffu, o0, o); o1 += __shfl_xor_sync(0xffffffffu, o1, o);
  }
#pragma unroll
  for (int w = 0; w < VW; ++w) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {      // head 2 t + (k >> 1), d 8 w + 4 (k & 1) ..
      const int e = 2 * (k & 1) + (k >> 1);
      const float add = k >> 1 ? o1 : o0;
      sh.o[warp][4 * w + k][lane] = make_float4(acc[4 * w][e] + add, acc[4 * w + 1][e] + add, acc[4 * w + 2][e] + add, acc[4 * w + 3][e] + add);
    }
  }
  if (lane < 4) { sh.m[warp][2 * t] = m0; sh.m[warp][2 * t + 1] = m1; sh.l[warp][2 * t] = l0; sh.l[warp][2 * t + 1] = l1; }
  __syncthreads();
}

// A maximum of minus infinity: weight 1 (its sums are zero, or not a number, which must stay).
__device__ __forceinline__ float part_weight(float m, float top) { return m == -INFINITY ? 1.f : fast_exp2(m - top); }
template <int D> constexpr int ITEM_BITS = D == 128 ? 8 : 7;     // fours of a block's outputs: 8 heads of D
// Head of the group and first d of an item.
template <int D> __device__ __forceinline__ void item_place(int item, int& h, int& d) {
  const int l = item & 31, piece = item >> 5;
  h = 2 * (l & 3) + (piece >> 1 & 1);
  d = (l >> 2) * (D / 8) + 8 * (piece >> 2) + 4 * (piece & 1);
}
__device__ __forceinline__ void add_part(float4& O, float& L, float4 x, float l, float w) {
  L = fmaf(l, w, L);
  O.x = fmaf(x.x, w, O.x); O.y = fmaf(x.y, w, O.y); O.z = fmaf(x.z, w, O.z); O.w = fmaf(x.w, w, O.w);
}
// An item of the block: its warps' parts added up.
template <int D, int UNIT>
__device__ __forceinline__ void add_warps(const Shared4<D, UNIT>& sh, int item, int h, float4& O, float& M, float& L) {
  M = sh.m[0][h]; L = 0.f; O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int w = 1; w < WARPS; ++w) M = fmaxf(M, sh.m[w][h]);
#pragma unroll
  for (int w = 0; w < WARPS; ++w) add_part(O, L, sh.o[w][item >> 5][item & 31], sh.l[w][h], part_weight(sh.m[w][h], M));
}
__device__ __forceinline__ void store_result(__nv_bfloat16* out, float4 o, float l) {
  const float inv = 1.0f / l;
  *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
}

// Where a launch's rows lie: row r of q at positions[r], of request segment_of_token[r] (negative: a padding row); or (segment_start given:
// a step that also holds prompt portions) row r is the one token of request r, and requests of other counts have none.
struct Rows {
  const int *segment_of_token, *positions, *segment_start;
  // the token, and its request; a negative request: there is nothing to do
  __device__ __forceinline__ int find(int r, int& token) const {
    token = r;
    if (segment_start != nullptr) {
      token = segment_start[r];
      if (segment_start[r + 1] - token != 1) return -1;
    }
    return segment_of_token[token];
  }
};

// Few tiles: a block for (row, up to 8 heads of a key/value head, part of the keys), grid (rows, n_kv * gchunks, 1 << cshift).  The parts
// are a thread-block cluster and are added up through distributed shared memory: one launch.
template <int D, int UNIT, bool CLUSTER>
__global__ void __launch_bounds__(WARPS * 32, BLOCKS)
attn_decode_int4_kernel(const __nv_bfloat16* q, const Cache4 cache, __nv_bfloat16* out,
                        const int* __restrict__ block_tables, int bt_stride, const Rows rows, int n_q, float scale_log2e, int cshift, int group,
                        int gchunks, int num_segments) {
  extern __shared__ __align__(16) unsigned char smem[];
  Shared4<D, UNIT>& sh = *reinterpret_cast<Shared4<D, UNIT>*>(smem);
  __shared__ float4 recv_o[CLUSTER ? 1 << ITEM_BITS<D> : 1];
  __shared__ float recv_m[MAX_CLUSTER * HEADS], recv_l[MAX_CLUSTER * HEADS];
  pdl_launch_dependents();
  // segments, positions and block tables are the step's own data: read before the wait for the kernels before
  int token;
  const int kvh = gchunks == 1 ? blockIdx.y : blockIdx.y / gchunks, g0 = gchunks == 1 ? 0 : (blockIdx.y % gchunks) * HEADS;
  const int gcount = min(HEADS, group - g0);
  const int seg = LSE_CHECKED(rows.find(blockIdx.x, token), -1, num_segments, -1, LSE_CHECK_SEGMENT);
  if (seg < 0) {                   // a padding row (all blocks of its cluster leave together)
    pdl_wait();                    // (a launch without work must not end before the one before it)
    return;
  }
  const int ctx = rows.positions[token] + 1, csize = 1 << cshift, rank = blockIdx.z, tid = threadIdx.x;
  const size_t first_head = (size_t)token * n_q + kvh * group + g0;
  const int total = (max(ctx, 0) + TILE - 1) / TILE, a_part = (total + csize - 1) >> cshift;
  const int tile_lo = min(total, rank * a_part), tile_hi = min(total, tile_lo + a_part);
  cg::cluster_group cluster = cg::this_cluster();
  if (CLUSTER) cluster.barrier_arrive();   // waited for before the first store into another block's memory
  attend_tiles<D, UNIT>(sh, cache, q + first_head * D, gcount, kvh, block_tables + (size_t)seg * bt_stride, ctx, tile_lo, tile_hi, scale_log2e, true);
  if (CLUSTER) cluster.barrier_wait();
  const int push_bits = ITEM_BITS<D> - cshift, push_per = 1 << push_bits;  // block r of a cluster finishes items r * push_per ..
  auto finish = [&](int h, int d, float4 o, float l) {
    if (h >= gcount) return;
    if (ctx <= 0) { o = make_float4(0.f, 0.f, 0.f, 0.f); l = 1.f; }
    store_result(out + (first_head + h) * D + d, o, l);
  };
#pragma unroll
  for (int item = tid; item < 1 << ITEM_BITS<D>; item += WARPS * 32) {
    int h, d;
    float4 O;
    float M, L;
    item_place<D>(item, h, d);
    add_warps<D, UNIT>(sh, item, h, O, M, L);
    if (!CLUSTER) {
      finish(h, d, O, L);
    } else {
      cluster.map_shared_rank(recv_o, item >> push_bits)[(rank << push_bits) + (item & (push_per - 1))] = O;
      if (d < MAX_CLUSTER) {        // (lanes with g = 0 hold d = 0 and 4 of a head: four destinations each)
        for (int r = d; r < min(d + 4, csize); ++r) {
          cluster.map_shared_rank(recv_m, r)[rank * HEADS + h] = M;
          cluster.map_shared_rank(recv_l, r)[rank * HEADS + h] = L;
        }
      }
    }
  }
  if (!CLUSTER) return;
  cluster.sync();      // every part is where it is finished
  const int mine = rank << push_bits;
  for (int item = mine + tid; item < mine + push_per; item += WARPS * 32) {
    int h, d;
    item_place<D>(item, h, d);
    float M = -INFINITY, L = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < MAX_CLUSTER; ++r)
      if (r < csize) M = fmaxf(M, recv_m[r * HEADS + h]);
#pragma unroll
    for (int r = 0; r < MAX_CLUSTER; ++r)
      if (r < csize) add_part(O, L, recv_o[(r << push_bits) + (item - mine)], recv_l[r * HEADS + h], part_weight(recv_m[r * HEADS + h], M));
    finish(h, d, O, L);
  }
}

// Many tiles: all tiles of the launch, ordered by row, heads (n_kv * gchunks = `columns` of them) and key, are cut into as many runs as there
// are blocks, alike but for one tile, whatever the rows' contexts are.  A row's heads whose tiles lie in one block are finished by it;
// else each block leaves its part (slot 2 b: a part that does not begin at the first key, 2 b + 1: one that does), and
// combine_runs_kernel adds the parts up.
__device__ __forceinline__ unsigned tiles_of(const Rows& rows, int row) {
  int token;
  return rows.find(row, token) >= 0 ? (unsigned)(max(rows.positions[token] + 1, 0) + TILE - 1) / TILE : 0u;
}
struct Runs {                  // `work` tiles over `blocks` blocks: the first `longer` of them get one more than the others
  unsigned a_block, longer;
  __device__ __forceinline__ Runs(unsigned work, unsigned blocks) : a_block(work / blocks), longer(work % blocks) {}
  __device__ __forceinline__ unsigned begin(unsigned block) const { return block * a_block + min(block, longer); }
  __device__ __forceinline__ unsigned block_of(unsigned tile) const {
    const unsigned edge = longer * (a_block + 1);
    return tile < edge ? tile / (a_block + 1) : longer + (tile - edge) / a_block;      // (a_block = 0: every tile lies before the edge)
  }
};
// Running sums of the rows' tiles by a whole block, as many rows at a time as it has threads: at(base, mine, before) gets every
// thread's row base + threadIdx.x, its tiles and those of all rows before it.  Returns the sum of all.
template <int THREADS, typename At>
__device__ __forceinline__ unsigned walk_rows(const Rows& rows, int tokens, unsigned (&sums)[THREADS / 32], At at) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned before = 0;
  for (int base = 0; base < tokens; base += THREADS) {
    const unsigned mine = base + tid < tokens ? tiles_of(rows, base + tid) : 0u;
    unsigned incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (base > 0) __syncthreads();
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    unsigned all = 0, earlier = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w == warp) earlier = all;
      all += sums[w];
    }
    at(base, mine, before + earlier + incl - mine);
    before += all;
  }
  return before;
}

template <int D, int UNIT>
__global__ void __launch_bounds__(WARPS * 32, BLOCKS)
attn_runs_int4_kernel(const __nv_bfloat16* q, const Cache4 cache, __nv_bfloat16* out, float4* part_o,
                      float2* part_ml, int2* shares, const int* __restrict__ block_tables, int bt_stride,
                      const Rows rows, int tokens, int n_q, float scale_log2e, int group, int gchunks, int num_segments) {
  constexpr int THREADS = WARPS * 32;
  extern __shared__ __align__(16) unsigned char smem[];
  Shared4<D, UNIT>& sh = *reinterpret_cast<Shared4<D, UNIT>*>(smem);
  __shared__ unsigned sums[WARPS], start_s[3];
  pdl_launch_dependents();
  const unsigned columns = cache.n_kv * gchunks;
  const int tid = threadIdx.x;
  unsigned mine_0 = 0, before_0 = 0;      // (a launch of up to 128 rows: they are looked at once)
  const unsigned all = walk_rows<THREADS>(rows, tokens, sums,
                                          [&](int base, unsigned mine, unsigned before) { if (base == 0) { mine_0 = mine; before_0 = before; } });
  const Runs runs(all * columns, gridDim.x);
  const unsigned begin = runs.begin(blockIdx.x), end = runs.begin(blockIdx.x + 1);
  // the row that `begin` lies in, its tiles and those before it
  if (begin < end) {
    auto look = [&](int base, unsigned mine, unsigned before) {
      if (begin >= before * columns && begin < (before + mine) * columns) { start_s[0] = base + tid; start_s[1] = mine; start_s[2] = before; }
    };
    if (tokens <= THREADS) look(0, mine_0, before_0);
    else { __syncthreads(); walk_rows<THREADS>(rows, tokens, sums, look); }
  }
  __syncthreads();
  int row = start_s[0], n = start_s[1];
  const unsigned inside = begin - start_s[2] * columns;
  unsigned at = begin, column = begin < end ? inside / n : 0;
  int tile = begin < end ? inside - column * n : 0;
  // A row that sees nothing gets zeros, a padding row nothing at all: the first block's threads, a row each.
  if (blockIdx.x == 0) {
    pdl_wait();
    for (int r = tid; r < tokens; r += THREADS) {
      if (tiles_of(rows, r) > 0) continue;
      for (unsigned k = 0; k < columns; ++k) shares[(size_t)r * columns + k] = make_int2(0, 1);
      int token;
      if (rows.find(r, token) >= 0)
        for (int i = 0; i < n_q * D / 8; ++i) reinterpret_cast<uint4*>(out + (size_t)token * n_q * D)[i] = make_uint4(0, 0, 0, 0);
    }
  }
  bool first = true;
  if (begin >= end) pdl_wait();
  while (at < end) {
    const int tile_hi = (int)min((unsigned)n, tile + (end - at));
    const int kvh = gchunks == 1 ? column : column / gchunks, g0 = gchunks == 1 ? 0 : (column % gchunks) * HEADS;
    const int gcount = min(HEADS, group - g0);
    int token;
    const int seg = LSE_CHECKED(rows.find(row, token), 0, num_segments, 0, LSE_CHECK_SEGMENT);
    const size_t first_head = (size_t)token * n_q + kvh * group + g0;
    if (!first) __syncthreads();       // the results of the run before have been read
    attend_tiles<D, UNIT>(sh, cache, q + first_head * D, gcount, kvh, block_tables + (size_t)seg * bt_stride, rows.positions[token] + 1, tile, tile_hi,
                          scale_log2e, first);
    first = false;
    const bool whole = tile == 0 && tile_hi == n;
    // whoever has the first of a row's tiles says how many blocks have some of them
    if (tile == 0 && tid == 0)
      shares[(size_t)row * columns + column] = make_int2(blockIdx.x, whole ? 1 : (int)(runs.block_of(at + n - 1) - blockIdx.x) + 1);
    const size_t slot = 2 * (size_t)blockIdx.x + (tile == 0 ? 1 : 0);
#pragma unroll
    for (int item = tid; item < 1 << ITEM_BITS<D>; item += THREADS) {
      int h, d;
      float4 O;
      float M, L;
      item_place<D>(item, h, d);
      add_warps<D, UNIT>(sh, item, h, O, M, L);
      if (h >= gcount) continue;
      if (whole) {
        store_result(out + (first_head + h) * D + d, O, L);
      } else {
        part_o[(slot << ITEM_BITS<D>) + item] = O;
        if (d == 0) part_ml[slot * HEADS + h] = make_float2(M, L);
      }
    }
    at += tile_hi - tile;
    tile = 0;
    if (tile_hi == n && ++column == columns) {
      column = 0;
      do ++row; while (at < end && (n = (int)tiles_of(rows, row)) == 0);
    }
  }
}

// One block = some items (fours of outputs) of a row's heads: their parts in the blocks' runs added up, PARTS_AT_ONCE of them side by
// side.  grid (rows, columns, slices): a slice is all items where a row has few parts, an eighth of them where it has many.
constexpr int COMBINE_THREADS = 256;
template <int D, int SLICES>
__global__ void __launch_bounds__(COMBINE_THREADS)
combine_runs_kernel(const float4* part_o, const float2* part_ml, const int2* shares,
                    const Rows rows, __nv_bfloat16* out, int n_q, int group, int gchunks) {
  constexpr int ITEMS = (1 << ITEM_BITS<D>) / SLICES, PARTS_AT_ONCE = COMBINE_THREADS / ITEMS;
  __shared__ float4 sum_o[COMBINE_THREADS];
  __shared__ float sum_m[COMBINE_THREADS], sum_l[COMBINE_THREADS];
  const int row = blockIdx.x, column = blockIdx.y;
  pdl_launch_dependents();
  pdl_wait();
  const int2 share = shares[(size_t)row * gridDim.y + column];
  const int b0 = share.x, parts = share.y;
  if (parts == 1) return;  // finished there
  const int item = blockIdx.z * ITEMS + threadIdx.x % ITEMS, lane_part = threadIdx.x / ITEMS;
  int h, d;
  item_place<D>(item, h, d);
  const int kvh = column / gchunks, g0 = column % gchunks * HEADS;
  const bool live = h < min(HEADS, group - g0);
  int token;
  rows.find(row, token);
  __nv_bfloat16* dst = out + ((size_t)token * n_q + kvh * group + g0 + h) * D + d;
  float M = -INFINITY, L = 0.f;
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int AT_ONCE = 4;       // loads in flight
  for (int p0 = lane_part; p0 < parts; p0 += AT_ONCE * PARTS_AT_ONCE) {
    float4 o[AT_ONCE];
    float2 ml[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int p = p0 + i * PARTS_AT_ONCE;
      const size_t slot = (size_t)2 * (b0 + p) + (p == 0 ? 1 : 0);
      ml[i] = make_float2(-INFINITY, 0.f);
      o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (live && p < parts) {
        o[i] = part_o[(slot << ITEM_BITS<D>) + item];
        ml[i] = part_ml[slot * HEADS + h];
      }
    }
    float top = M;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) top = fmaxf(top, ml[i].x);
    const float w = part_weight(M, top);
    L *= w; O.x *= w; O.y *= w; O.z *= w; O.w *= w;
    M = top;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) add_part(O, L, o[i], ml[i].y, part_weight(ml[i].x, M));
  }
  if (PARTS_AT_ONCE > 1) {
    sum_o[threadIdx.x] = O; sum_m[threadIdx.x] = M; sum_l[threadIdx.x] = L;
    __syncthreads();
    if (lane_part > 0) return;
#pragma unroll
    for (int k = 0; k < PARTS_AT_ONCE; ++k) M = fmaxf(M, sum_m[k * ITEMS + threadIdx.x]);
    L = 0.f; O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < PARTS_AT_ONCE; ++k) {
      const int at = k * ITEMS + threadIdx.x;
      add_part(O, L, sum_o[at], sum_l[at], part_weight(sum_m[at], M));
    }
  }
  if (live) store_result(dst, O, L);
}

template <int D, int UNIT>
int launch_rows(const void* q, const Cache4& cache, void* out, float* scratch, const int* block_tables, int bt_stride,
                const Rows& rows, int tokens, int n_q, float scale, int splits, int runs, int num_segments, cudaStream_t stream) {
  const int group = n_q / cache.n_kv, gchunks = (group + HEADS - 1) / HEADS, columns = cache.n_kv * gchunks;
  constexpr size_t smem = sizeof(Shared4<D, UNIT>), limit = smem + 8192;     // (what is static counts towards the 48 KB that need no leave)
  static SmemAllowance allowance[3];
  cudaError_t err;
  if (runs > 0) {
    err = allow_smem(attn_runs_int4_kernel<D, UNIT>, limit, allowance[0]);
    if (err != cudaSuccess) return (int)err;
    float4* part_o = reinterpret_cast<float4*>(scratch);
    float2* part_ml = reinterpret_cast<float2*>(scratch + (size_t)2 * runs * HEADS * D);
    int2* shares = reinterpret_cast<int2*>(part_ml + (size_t)2 * runs * HEADS);
    err = lse_launch(attn_runs_int4_kernel<D, UNIT>, dim3((unsigned)runs), dim3(WARPS * 32), smem, stream, (const __nv_bfloat16*)q, cache,
                     (__nv_bfloat16*)out, part_o, part_ml, shares, block_tables, bt_stride, rows, tokens, n_q, scale * LOG2E,
                     group, gchunks, num_segments);
    if (err != cudaSuccess) return (int)err;
    // More than eight parts a row on average: eight slices, so that the parts of one long row are added up by more than its few blocks.
    // One slice and eight, us of both launches: a row of 28 / 4 heads over 30,000 keys (148 parts) 30.2 and 13.5, four of 12 / 2 over 8,000
    // (74) 19.5 and 10.6, four of 40 / 8 over 8,000 (18) 18.1 and 17.4, sixteen of 8 heads of 64 over 6,000 (5) 21.5 and 23.2.
#define LSE_INT4_COMBINE(SLICES)                                                                                                 \
  lse_launch(combine_runs_kernel<D, SLICES>, dim3((unsigned)tokens, (unsigned)columns, SLICES), dim3(COMBINE_THREADS), 0, stream,       \
             (const float4*)part_o, (const float2*)part_ml, (const int2*)shares, rows, (__nv_bfloat16*)out, n_q, group, gchunks)
    err = (long long)tokens * columns * 8 < runs ? LSE_INT4_COMBINE(8) : LSE_INT4_COMBINE(1);
#undef LSE_INT4_COMBINE
  } else {
    const int cshift = splits >= 8 ? 3 : splits >= 4 ? 2 : splits >= 2 ? 1 : 0;
    const dim3 grid((unsigned)tokens, (unsigned)columns, 1u << cshift);
    err = cshift ? allow_smem(attn_decode_int4_kernel<D, UNIT, true>, limit, allowance[1])
                 : allow_smem(attn_decode_int4_kernel<D, UNIT, false>, limit, allowance[2]);
    if (err != cudaSuccess) return (int)err;
#define LSE_INT4_ROWS(CLUSTER)                                                                                                   \
  lse_launch_cluster(attn_decode_int4_kernel<D, UNIT, CLUSTER>, grid, dim3(WARPS * 32), smem, stream, 1u << cshift, (const __nv_bfloat16*)q, cache, \
                     (__nv_bfloat16*)out, block_tables, bt_stride, rows, n_q, scale * LOG2E, cshift, group, gchunks, \
                     num_segments)
    err = cshift ? LSE_INT4_ROWS(true) : LSE_INT4_ROWS(false);
#undef LSE_INT4_ROWS
  }
  if (err != cudaSuccess) return (int)err;
  LSE_LAUNCH_CHECK();
}

}  // namespace

// q, out bfloat16 [tokens, n_q, head_dim]; the cache as int4_cache.cu leaves it; block_tables [num_segments, bt_stride].
// segment_of_token < 0: a padding row, left as it was; a row at a negative position sees no key and gets zeros.  segment_start (may be
// null): `tokens` counts requests, and the rows are those of requests with one token (see Rows).
// runs = 0: a row's keys are shared by `splits` blocks (1, 2, 4 or 8); runs > 0: all rows' tiles are cut into so many equal runs, and `scratch`
// holds 16 runs (head_dim + 2) + 2 tokens n_kv ceil(n_q / n_kv / 8) words.
extern "C" int lse_paged_attention_decode_int4(const void* q, const void* k_codes, const void* k_scales, const void* v_codes,
                                               const void* v_scales, void* out, float* scratch, const int* block_tables,
                                               int bt_stride, const int* segment_of_token, const int* positions,
                                               const int* segment_start, int tokens, int n_q, int n_kv, int head_dim, int page_size,
                                               float scale, int splits, int runs,
                                               long long num_pages, int num_segments, cudaStream_t stream) {
  if (tokens <= 0) return 0;
  const int unit = page_size <= 0 ? 0 : page_size % 16 == 0 ? 16 : page_size % 8 == 0 ? 8 : 1;
  if ((head_dim != 64 && head_dim != 128) || n_kv <= 0 || n_q % n_kv || page_size <= 0 || num_pages <= 0 || splits < 1 || runs < 0 ||
      num_pages * page_size > 0x7fffffffLL || (runs > 0 && scratch == nullptr) ||
      (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)scratch) & 15) ||
      (((uintptr_t)k_scales | (uintptr_t)v_scales) & (unit > 1 ? 15 : 3)))      // scales come four rows at a time, or row by row
    return LSE_ERR_BAD_ARGUMENT;
  if (num_pages * page_size / 8 * n_kv > 0xffffffffLL || n_q > 65535 ||
      (long long)tokens * (((long long)bt_stride * page_size + TILE - 1) / TILE) * n_kv * ((n_q / n_kv + HEADS - 1) / HEADS) > 0x7fffffffLL) return LSE_ERR_TOO_LARGE;
  Cache4 cache = {(const unsigned char*)k_codes, (const unsigned char*)v_codes, (const uint32_t*)k_scales, (const uint32_t*)v_scales,
                  {page_size, -1}, n_kv, (int)num_pages};
  if ((page_size & (page_size - 1)) == 0)
    for (cache.pm.shift = 0; 1 << cache.pm.shift < page_size;) ++cache.pm.shift;
  const Rows rows = {segment_of_token, positions, segment_start};
#define LSE_INT4_ARGS q, cache, out, scratch, block_tables, bt_stride, rows, tokens, n_q, scale, splits, runs, num_segments, stream
  if (head_dim == 128) return unit == 16 ? launch_rows<128, 16>(LSE_INT4_ARGS) : unit == 8 ? launch_rows<128, 8>(LSE_INT4_ARGS) : launch_rows<128, 1>(LSE_INT4_ARGS);
  return unit == 16 ? launch_rows<64, 16>(LSE_INT4_ARGS) : unit == 8 ? launch_rows<64, 8>(LSE_INT4_ARGS) : launch_rows<64, 1>(LSE_INT4_ARGS);
#undef LSE_INT4_ARGS
}

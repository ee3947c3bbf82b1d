// Keys and values held in 4 bits: the write (bias + rotation + quantisation) and the way back.
//
// A row of D values x of one token and one key/value head is held as codes u in 0 .. 15 with a scale and a centre, both bfloat16:
//   s = bf16((max x - min x) / 15),  c = bf16(min x + 8 s),  u = clamp(rint((x - c) / s) + 8, 0, 15)
// and stands for  s (u - 8) + c.  One scale a row: both products of the attention then see whole numbers in -8 .. 7, exact in
// bfloat16, and take scale and centre outside.  Rows whose values are all alike have s = 0 and stand for c; a row with a value
// that is not finite stands for NaN everywhere (c = NaN), as it would reach every score from a cache of floating-point values.
//
// Storage: codes uint8 [page][kv head][offset][D / 2], byte b holding d = 2 b in its low and 2 b + 1 in its high half; scales
// bfloat16 [page][kv head][offset][2] = (s, c).
//
// The code is that of 64-bit arithmetic throughout: a code next to the border between two flips with the last bit of x, and a
// flipped code is a whole step of the row's range.  (Scale and centre come from float32 where that provably gives the same.)  With float32 rotations about two codes in a million depended on how the
// sine was rounded.  (FP64 runs at half the float32 rate here; sines are taken once a token, not once a head.)
#include "common.cuh"

LSE_CHECK_DEFINE(lse_check_int4_cache)

namespace {

template <typename T> __device__ __forceinline__ void load_four(const T* p, float (&v)[4]);
template <> __device__ __forceinline__ void load_four<float>(const float* p, float (&v)[4]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
}
template <> __device__ __forceinline__ void load_four<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[4]) {
  const uint2 a = *reinterpret_cast<const uint2*>(p);
  const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&a.x));
  const float2 hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&a.y));
  v[0] = lo.x; v[1] = lo.y; v[2] = hi.x; v[3] = hi.y;
}

__device__ __forceinline__ double shfl_xor_double(double v, int o) {
  return __hiloint2double(__shfl_xor_sync(0xffffffffu, __double2hiint(v), o), __shfl_xor_sync(0xffffffffu, __double2loint(v), o));
}
// double to bfloat16 by way of float32, as a tensor library converts
__device__ __forceinline__ __nv_bfloat16 bf16_of(double v) { return __float2bfloat16_rn((float)v); }

// One block = TOKENS tokens x their key and value heads (blockIdx.y < kv_blocks), or x their query heads.  It works out the tokens' sines
// (a thread each), then its threads walk the heads of a token each, with the next head's projections on their way.  A thread owns
// eight values of a head: pairing 0 the neighbours 8 c .. 8 c + 7 (four pairs), pairing 1 the runs 4 c .. and D / 2 + 4 c .. (pairs across
// the halves).  LANES = D / 8 threads share a head and find its extremes by shuffles.
// What bounds it: neither memory nor instructions alone (2,001 rows of 40 / 8 heads of 128 in float32: 82 MB in 27.4 us, 3.0 TB/s; 52% of
// the issue slots), but a block's chain of loads, sines, 64-bit rotations and shuffles.  The keys' and values' blocks alone take 16.3 us,
// the queries' alone 18.0; either without the sines 0.1 less.  Extremes, scale and centre all in 64 bits: 32.3 us.  Two rows on
// their way instead of one: 29.3; two, four or eight tokens a block, blocks of 128 threads, either kind of block first: 27.0 to 28.2.
constexpr int THREADS = 256;
template <typename TI, int D, int PAIRING, int TOKENS>
__global__ void __launch_bounds__(THREADS, 4)
rope_kv_write_int4_kernel(const TI* qkv, int n_partials, long long partial_stride, const float* __restrict__ bias,
                          const int* __restrict__ positions, const int* __restrict__ slot_mapping,
                          const float* __restrict__ inv_freq, __nv_bfloat16* __restrict__ q_out, unsigned char* __restrict__ k_codes,
                          __nv_bfloat162* __restrict__ k_scales, unsigned char* __restrict__ v_codes,
                          __nv_bfloat162* __restrict__ v_scales, int tokens, int n_q, int n_kv, int page_size, long long qkv_stride,
                          long long num_slots, int q_blocks) {
  constexpr int LANES = D / 8, HALF = D / 2, HEADS = THREADS / LANES;
  __shared__ double2 turn_s[TOKENS * HALF];      // cosines and sines of the tokens' angles
  pdl_launch_dependents();
  const int t0 = blockIdx.x * TOKENS, count = min(TOKENS, tokens - t0);
  const int kv_blocks = (int)gridDim.y - q_blocks;      // first in the grid: they take longer
  const bool queries = (int)blockIdx.y >= kv_blocks;
  const int heads = queries ? n_q : 2 * n_kv, head0 = queries ? 0 : n_q;         // of a token; its first among a row's heads
  // a thread keeps its token and goes on by `step` heads
  constexpr int AT_ONCE = HEADS / TOKENS;
  const int step = AT_ONCE * (queries ? q_blocks : kv_blocks), begin = (queries ? (int)blockIdx.y - kv_blocks : (int)blockIdx.y) * AT_ONCE;
  const int token = threadIdx.x / LANES % TOKENS, offset = threadIdx.x / LANES / TOKENS;
  const bool here = token < count;
  const int c = threadIdx.x % LANES;
  const int e0 = PAIRING == 0 ? 8 * c : 4 * c, e1 = PAIRING == 0 ? 8 * c + 4 : HALF + 4 * c;
  // positions, slots, frequencies and bias are the step's or the model's own data: read before the wait for the kernel that makes the
  // projections
  for (int i = threadIdx.x; i < count * HALF; i += THREADS) {
    double angle = (double)positions[t0 + i / HALF] * (double)inv_freq[i % HALF];
    angle -= 6.283185307179586 * rint(angle * 0.15915494309189535);
    if (queries) {
      float sn, cs;
      sincosf((float)angle, &sn, &cs);
      reinterpret_cast<float2*>(turn_s)[i] = make_float2(cs, sn);
    } else {
      double sn, cs;
      sincos(angle, &sn, &cs);
      turn_s[i] = make_double2(cs, sn);
    }
  }
  pdl_wait();
  auto load_eight = [&](const auto* p, float (&to)[8]) {
    float lo[4], hi[4];
    load_four(p + e0, lo);
    load_four(p + e1, hi);
#pragma unroll
    for (int j = 0; j < 4; ++j) { to[j] = lo[j]; to[4 + j] = hi[j]; }
  };
  const TI* const mine_in = qkv + (size_t)(t0 + token) * qkv_stride + (size_t)head0 * D;      // (read only where the token is there)
  auto load_row = [&](int head, float (&to)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) to[j] = 0.f;
    if (!here || head >= heads) return;
    const TI* row = mine_in + head * D;
    if (n_partials == 1) {
      load_eight(row, to);
      return;
    }
#pragma unroll 4
    for (int k = 0; k < n_partials; ++k) {
      float a[8];
      load_eight(row + (size_t)k * partial_stride, a);
#pragma unroll
      for (int j = 0; j < 8; ++j) to[j] += a[j];
    }
  };
  float g[8];
  load_row(begin + offset, g);
  __syncthreads();
  float2 turn_q[4];
  if (queries) {
#pragma unroll
    for (int j = 0; j < 4; ++j) turn_q[j] = reinterpret_cast<const float2*>(turn_s)[token * HALF + 4 * c + j];
  }
  const int slot = !queries && here ? LSE_CHECKED(slot_mapping[t0 + token], -1, (int)num_slots, -1, LSE_CHECK_CACHE_SLOT) : -1;
  const size_t page = (unsigned)max(slot, 0) / (unsigned)page_size, off = (unsigned)max(slot, 0) % (unsigned)page_size;
  for (int base = begin; base < heads; base += step) {      // the same in the whole block: shuffles take whole warps
    const int head = base + offset;
    const bool live = here && head < heads;
    float ahead[8];
    load_row(head + step, ahead);
    float b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = 0.f;
    if (live && bias) load_eight(bias + (size_t)(head0 + head) * D, b);
    if (queries) {
      if (live) {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] += b[j];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float& x = PAIRING == 0 ? g[2 * j] : g[j];
          float& y = PAIRING == 0 ? g[2 * j + 1] : g[4 + j];
          const float rx = x * turn_q[j].x - y * turn_q[j].y, ry = y * turn_q[j].x + x * turn_q[j].y;
          x = rx; y = ry;
        }
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __nv_bfloat162 v = __floats2bfloat162_rn(g[2 * j], g[2 * j + 1]);
          w[j] = *reinterpret_cast<const uint32_t*>(&v);
        }
        __nv_bfloat16* dst = q_out + ((size_t)(t0 + token) * n_q + head) * D;
        if (PAIRING == 0) {
          *reinterpret_cast<uint4*>(dst + e0) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
          *reinterpret_cast<uint2*>(dst + e0) = make_uint2(w[0], w[1]);
          *reinterpret_cast<uint2*>(dst + e1) = make_uint2(w[2], w[3]);
        }
      }
    } else {
      const bool is_k = head < n_kv;
      double x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = (double)g[j];
      if (bias) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] += (double)b[j];
      }
      if (is_k && live) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const double2 turn = turn_s[token * HALF + 4 * c + j];
          double& p = PAIRING == 0 ? x[2 * j] : x[j];
          double& q = PAIRING == 0 ? x[2 * j + 1] : x[4 + j];
          const double rp = p * turn.x - q * turn.y, rq = q * turn.x + p * turn.y;
          p = rp; q = rq;
        }
      }
      // a row's lanes are LANES neighbours of a warp
      const unsigned mine = ((1u << LANES) - 1u) << (threadIdx.x & 31 & ~(LANES - 1));
      __nv_bfloat16 scale, centre;
      bool whole = true;       // every value of the row is finite
      {
        // The extremes as float32: scale and centre are those of the exact ones where either end of what these can be off by
        // (and more: half a unit of the last place each, then two roundings of each expression) rounds to the same bfloat16.
        float low = (float)x[0], high = low, none = low * 0.f;      // `none`: zero where every value is finite
#pragma unroll
        for (int j = 1; j < 8; ++j) {
          const float v = (float)x[j];
          low = fminf(low, v); high = fmaxf(high, v);
          none = fmaf(v, 0.f, none);
        }
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) {
          low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
          high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
        }
        const float range = high - low, floor = range != 0.f ? 0x1p-120f : 0.f, off = fmaf(0x1p-21f, fabsf(high) + fabsf(low), floor);
        const float s0 = __bfloat162float(__float2bfloat16_rn((range - off) * (1.f / 15.f)));
        scale = __float2bfloat16_rn((range + off) * (1.f / 15.f));
        const float s1 = __bfloat162float(scale), at = fmaf(8.f, s1, low), at_off = fmaf(0x1p-21f, fabsf(low) + 8.f * s1, floor);
        const float c0 = __bfloat162float(__float2bfloat16_rn(at - at_off));
        centre = __float2bfloat16_rn(at + at_off);
        if (!__all_sync(0xffffffffu, none == 0.f && range < 1e37f && s0 == s1 && c0 == __bfloat162float(centre))) {
          double lo = x[0], hi = x[0], all = x[0] * 0.0;
#pragma unroll 1
          for (int o = 0; o < LANES; o = o == 0 ? 1 : o << 1) {
#pragma unroll
            for (int j = 1; j < 8; ++j) {
              if (o > 0) break;
              lo = x[j] < lo ? x[j] : lo;
              hi = x[j] > hi ? x[j] : hi;
              all = fma(x[j], 0.0, all);
            }
            const double l = shfl_xor_double(lo, o), h = shfl_xor_double(hi, o);
            lo = l < lo ? l : lo;
            hi = h > hi ? h : hi;
          }
          whole = (__ballot_sync(0xffffffffu, all == 0.0) & mine) == mine;
          scale = bf16_of((hi - lo) / 15.0);
          centre = bf16_of(lo + 8.0 * (double)__bfloat162float(scale));
          if (!whole) { scale = __float2bfloat16_rn(0.f); centre = __float2bfloat16_rn(__int_as_float(0x7fc00000)); }
        }
      }
      if (live && slot >= 0) {
        const float s_float = __bfloat162float(scale);
        const double s = (double)s_float, m = (double)__bfloat162float(centre), half = 0.5 * s;
        double inverse = (double)__fdividef(1.f, s_float);      // (an estimate will do)
        if (!(s_float >= 0x1p-120f && s_float <= 0x1p120f)) inverse = s != 0.0 ? 1.0 / s : 0.0;
        // the quotient (x - c) / s to nearest, halves to even: its estimate, rounded by the addition of a number whose last place is 1,
        // is off by one at most, and what is left of x decides (exactly: rows that come in bfloat16 do lie half way between two codes)
        constexpr double ONES = 0x1.8p52;
        int q[8];
        bool near = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const double from_centre = x[j] - m, rounded = fma(from_centre, inverse, ONES);
          q[j] = __double2loint(rounded);
          near |= fabs(fma(ONES - rounded, s, from_centre)) >= half;
        }
        if (near) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const double from_centre = x[j] - m, twice = 2.0 * fma(-(double)q[j], s, from_centre);
            if (twice > s || (twice == s && (q[j] & 1))) ++q[j];
            else if (twice < -s || (twice == -s && (q[j] & 1))) --q[j];
          }
        }
        uint32_t code[2] = {0u, 0u};      // four codes each: those of e0 .., those of e1 ..
#pragma unroll
        for (int j = 0; j < 8; ++j) code[j >> 2] |= (uint32_t)(min(max(q[j], -8), 7) + 8) << (4 * (j & 3));
        if (!whole || s == 0.0) code[0] = code[1] = 0x8888u;
        const size_t place = (page * n_kv + (is_k ? head : head - n_kv)) * page_size + off;
        unsigned char* dst = (is_k ? k_codes : v_codes) + place * (D / 2);
        if (PAIRING == 0) {
          *reinterpret_cast<uint32_t*>(dst + 4 * c) = code[0] | code[1] << 16;
        } else {
          *reinterpret_cast<unsigned short*>(dst + 2 * c) = (unsigned short)code[0];
          *reinterpret_cast<unsigned short*>(dst + D / 4 + 2 * c) = (unsigned short)code[1];
        }
        if (c == 0) (is_k ? k_scales : v_scales)[place] = __nv_bfloat162(scale, centre);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = ahead[j];
  }
}

// Eight values a thread: keys (blockIdx.y = 0) or values (1) of the slots, as bfloat16.
template <int D>
__global__ void __launch_bounds__(256)
kv_read_int4_kernel(const unsigned char* k_codes, const __nv_bfloat162* k_scales,
                    const unsigned char* v_codes, const __nv_bfloat162* v_scales,
                    const int* __restrict__ slot_mapping, __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out,
                    int tokens, int n_kv, int page_size, long long num_slots) {
  constexpr int LANES = D / 8;
  pdl_launch_dependents();
  const long long item = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int c = (int)(item % LANES);
  const long long row = item / LANES;
  const int t = (int)(row / n_kv), head = (int)(row % n_kv);
  const int slot = t < tokens ? LSE_CHECKED(slot_mapping[t], -1, (int)num_slots, -1, LSE_CHECK_CACHE_SLOT) : -1;
  pdl_wait();
  if (slot < 0) return;
  const size_t place = ((size_t)(slot / page_size) * n_kv + head) * page_size + slot % page_size;
  const uint32_t word = *reinterpret_cast<const uint32_t*>((blockIdx.y ? v_codes : k_codes) + place * (D / 2) + 4 * c);
  const float2 sc = __bfloat1622float2((blockIdx.y ? v_scales : k_scales)[place]);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = fmaf(sc.x, (float)((int)(word >> (8 * j) & 15u) - 8), sc.y), b = fmaf(sc.x, (float)((int)(word >> (8 * j + 4) & 15u) - 8), sc.y);
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    w[j] = *reinterpret_cast<const uint32_t*>(&v);
  }
  *reinterpret_cast<uint4*>((blockIdx.y ? v_out : k_out) + row * D + 8 * c) = make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename TI, int D>
int launch_write(const void* qkv, int n_partials, long long partial_stride, const float* bias, const int* positions,
                 const int* slot_mapping, const float* inv_freq, void* q_out, void* k_codes, void* k_scales, void* v_codes,
                 void* v_scales, int tokens, int n_q, int n_kv, int page_size, int pairing, long long qkv_stride,
                 long long num_slots, cudaStream_t stream) {
  constexpr int HEADS = THREADS / (D / 8);
  // Many tokens: four a block, whose angles take all its threads; few: a block for every pass over a token's heads.  Few and many, us:
  // 28 / 4 heads in bfloat16, 64 tokens 4.1 and 6.3, 512 7.9 and 8.7, 768 10.5 and 8.2; 40 / 8 in float32, 64 tokens 4.3 and 7.5, 768
  // 12.4 and 13.8, 1,024 15.2 and 13.7; 12 / 2 in bfloat16, 64 tokens 3.9 and 4.1, 512 5.8 and 5.3, 1,024 9.5 and 6.4.
  const bool many = tokens >= 512;
  const int q_blocks = many ? 1 : (n_q + HEADS - 1) / HEADS, kv_blocks = many ? 1 : (2 * n_kv + HEADS - 1) / HEADS;
  const dim3 grid((unsigned)(many ? (tokens + 3) / 4 : tokens), (unsigned)(q_blocks + kv_blocks));
#define LSE_INT4_WRITE(PAIRING, TOKENS)                                                                                  \
  lse_launch(rope_kv_write_int4_kernel<TI, D, PAIRING, TOKENS>, grid, dim3(THREADS), 0, stream, (const TI*)qkv, n_partials, partial_stride, \
             bias, positions, slot_mapping, inv_freq, (__nv_bfloat16*)q_out, (unsigned char*)k_codes,                   \
             (__nv_bfloat162*)k_scales, (unsigned char*)v_codes, (__nv_bfloat162*)v_scales, tokens, n_q, n_kv, page_size, qkv_stride, \
             num_slots, q_blocks)
  const cudaError_t err = pairing == 0 ? (many ? LSE_INT4_WRITE(0, 4) : LSE_INT4_WRITE(0, 1)) : (many ? LSE_INT4_WRITE(1, 4) : LSE_INT4_WRITE(1, 1));
#undef LSE_INT4_WRITE
  if (err != cudaSuccess) return (int)err;
  LSE_LAUNCH_CHECK();
}

bool bad_cache(int n_kv, int head_dim, int page_size, long long num_pages) {
  return (head_dim != 64 && head_dim != 128) || n_kv <= 0 || page_size <= 0 || num_pages <= 0 || num_pages * page_size > 0x7fffffffLL;
}

}  // namespace

// qkv [tokens, width] (rows qkv_stride apart; or n_partials such sums partial_stride apart), width = (n_q + 2 n_kv) head_dim;
// q_out bfloat16 [tokens, n_q, head_dim].  A row whose slot is negative has its queries rotated and nothing cached.
extern "C" int lse_rope_kv_write_int4(const void* qkv, int in_dtype, int n_partials, long long partial_stride, const float* bias,
                                      const int* positions, const int* slot_mapping, const float* inv_freq, void* q_out,
                                      void* k_codes, void* k_scales, void* v_codes, void* v_scales, int tokens, int n_q, int n_kv,
                                      int head_dim, int page_size, int pairing, long long qkv_stride, long long num_pages,
                                      cudaStream_t stream) {
  if (tokens <= 0) return 0;
  const int align = in_dtype == LSE_DTYPE_F32 ? 15 : 7;
  if (bad_cache(n_kv, head_dim, page_size, num_pages) || n_q <= 0 || (pairing != 0 && pairing != 1) || n_partials < 1 ||
      qkv_stride % 4 || partial_stride % 4 || ((uintptr_t)qkv & align) ||
      (((uintptr_t)bias | (uintptr_t)inv_freq | (uintptr_t)q_out | (uintptr_t)k_codes | (uintptr_t)v_codes) & 15) ||
      (((uintptr_t)k_scales | (uintptr_t)v_scales) & 3))      // (a layer's parts of a cache whose pages are no multiple of four rows)
    return LSE_ERR_BAD_ARGUMENT;
#define LSE_INT4_ARGS qkv, n_partials, partial_stride, bias, positions, slot_mapping, inv_freq, q_out, k_codes, k_scales, v_codes, \
  v_scales, tokens, n_q, n_kv, page_size, pairing, qkv_stride, num_pages * page_size, stream
  if (in_dtype == LSE_DTYPE_BF16)
    return head_dim == 128 ? launch_write<__nv_bfloat16, 128>(LSE_INT4_ARGS) : launch_write<__nv_bfloat16, 64>(LSE_INT4_ARGS);
  if (in_dtype == LSE_DTYPE_F32)
    return head_dim == 128 ? launch_write<float, 128>(LSE_INT4_ARGS) : launch_write<float, 64>(LSE_INT4_ARGS);
#undef LSE_INT4_ARGS
  return LSE_ERR_BAD_ARGUMENT;
}

// k_out, v_out bfloat16 [tokens, n_kv, head_dim]: what the cache holds at each slot; rows whose slot is negative are left alone.
extern "C" int lse_kv_read_int4(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                                const int* slot_mapping, void* k_out, void* v_out, int tokens, int n_kv, int head_dim,
                                int page_size, long long num_pages, cudaStream_t stream) {
  if (tokens <= 0) return 0;
  if (bad_cache(n_kv, head_dim, page_size, num_pages) ||
      (((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_out | (uintptr_t)v_out) & 15) ||
      (((uintptr_t)k_scales | (uintptr_t)v_scales) & 3))
    return LSE_ERR_BAD_ARGUMENT;
  const long long items = (long long)tokens * n_kv * (head_dim / 8);
  const dim3 grid((unsigned)((items + 255) / 256), 2);
#define LSE_INT4_READ(D)                                                                                               \
  lse_launch(kv_read_int4_kernel<D>, grid, dim3(256), 0, stream, (const unsigned char*)k_codes, (const __nv_bfloat162*)k_scales, \
             (const unsigned char*)v_codes, (const __nv_bfloat162*)v_scales, slot_mapping, (__nv_bfloat16*)k_out,       \
             (__nv_bfloat16*)v_out, tokens, n_kv, page_size, num_pages * page_size)
  const cudaError_t err = head_dim == 128 ? LSE_INT4_READ(128) : LSE_INT4_READ(64);
#undef LSE_INT4_READ
  if (err != cudaSuccess) return (int)err;
  LSE_LAUNCH_CHECK();
}

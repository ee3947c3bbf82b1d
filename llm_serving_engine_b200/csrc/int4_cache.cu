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
// Everything up to the code is worked out in 64 bits: a code next to the border between two flips with the last bit of x, and a
// flipped code is a whole step of the row's range.  With float32 rotations about two codes in a million depended on how the
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

// One block = one token x a range of heads (queries, then keys, then values).  A thread owns eight values of a head: pairing 0
// the neighbours 8 c .. 8 c + 7 (four pairs), pairing 1 the runs 4 c .. and D / 2 + 4 c .. (pairs across the halves).
// LANES = D / 8 threads share a head and find its extremes by shuffles.
template <typename TI, int D, int PAIRING>
__global__ void __launch_bounds__(256)
rope_kv_write_int4_kernel(const TI* __restrict__ qkv, int n_partials, long long partial_stride, const float* __restrict__ bias,
                          const int* __restrict__ positions, const int* __restrict__ slot_mapping,
                          const float* __restrict__ inv_freq, __nv_bfloat16* __restrict__ q_out, unsigned char* __restrict__ k_codes,
                          __nv_bfloat162* __restrict__ k_scales, unsigned char* __restrict__ v_codes,
                          __nv_bfloat162* __restrict__ v_scales, int n_q, int n_kv, int page_size, long long qkv_stride,
                          long long num_slots, int heads_a_block) {
  constexpr int LANES = D / 8, HALF = D / 2;
  __shared__ double2 turn_s[HALF];      // cosine and sine of the token's angles
  pdl_launch_dependents();
  const int t = blockIdx.x;
  const int heads = n_q + 2 * n_kv;
  const int first_head = blockIdx.y * heads_a_block, last_head = min(heads, first_head + heads_a_block);
  // position, slot and frequencies are the step's own data: read before the wait for the kernel that makes the projections
  const int slot = LSE_CHECKED(slot_mapping[t], -1, (int)num_slots, -1, LSE_CHECK_CACHE_SLOT);
  if (first_head < n_q + n_kv)
    for (int i = threadIdx.x; i < HALF; i += blockDim.x) {
      double angle = (double)positions[t] * (double)inv_freq[i];
      angle -= 6.283185307179586 * rint(angle * 0.15915494309189535);
      double sn, cs;
      sincos(angle, &sn, &cs);
      turn_s[i] = make_double2(cs, sn);
    }
  __syncthreads();
  pdl_wait();
  const int c = threadIdx.x % LANES, rows_at_once = blockDim.x / LANES;
  const int e0 = PAIRING == 0 ? 8 * c : 4 * c, e1 = PAIRING == 0 ? 8 * c + 4 : HALF + 4 * c;
  // all lanes of a warp stay in the loop: the shuffles take whole warps
  for (int base = first_head; base < last_head; base += rows_at_once) {
    const int head = base + threadIdx.x / LANES;
    const bool is_q = head < n_q, is_k = !is_q && head < n_q + n_kv;
    const bool live = head < last_head && (is_q || slot >= 0);
    float g0[4] = {0.f, 0.f, 0.f, 0.f}, g1[4] = {0.f, 0.f, 0.f, 0.f};
    if (live) {
      const TI* row = qkv + (size_t)t * qkv_stride + (size_t)head * D;
      for (int p = 0; p < n_partials; ++p) {
        float a[4], b[4];
        load_four<TI>(row + (size_t)p * partial_stride + e0, a);
        load_four<TI>(row + (size_t)p * partial_stride + e1, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) { g0[j] += a[j]; g1[j] += b[j]; }
      }
    }
    float b0[4] = {0.f, 0.f, 0.f, 0.f}, b1[4] = {0.f, 0.f, 0.f, 0.f};
    if (live && bias) {
      load_four<float>(bias + (size_t)head * D + e0, b0);
      load_four<float>(bias + (size_t)head * D + e1, b1);
    }
    if (is_q && live) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) { x[j] = g0[j] + b0[j]; x[4 + j] = g1[j] + b1[j]; }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double2 turn = turn_s[4 * c + j];
        const float cs = (float)turn.x, sn = (float)turn.y;
        float& a = PAIRING == 0 ? x[2 * j] : x[j];
        float& b = PAIRING == 0 ? x[2 * j + 1] : x[4 + j];
        const float ra = a * cs - b * sn, rb = b * cs + a * sn;
        a = ra; b = rb;
      }
      __nv_bfloat16* dst = q_out + ((size_t)t * n_q + head) * D;
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&v);
      }
      *reinterpret_cast<uint2*>(dst + e0) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(dst + e1) = make_uint2(w[2], w[3]);
    }
    if (base + rows_at_once <= n_q) continue;     // the same for the whole block: queries only
    double x[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) { x[j] = (double)g0[j] + (double)b0[j]; x[4 + j] = (double)g1[j] + (double)b1[j]; }
    if (is_k) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double2 turn = turn_s[4 * c + j];
        double& a = PAIRING == 0 ? x[2 * j] : x[j];
        double& b = PAIRING == 0 ? x[2 * j + 1] : x[4 + j];
        const double ra = a * turn.x - b * turn.y, rb = b * turn.x + a * turn.y;
        a = ra; b = rb;
      }
    }
    double low = x[0], high = x[0];
    bool finite = isfinite(x[0]);
#pragma unroll
    for (int j = 1; j < 8; ++j) { low = fmin(low, x[j]); high = fmax(high, x[j]); finite = finite && isfinite(x[j]); }
    int whole = finite ? 1 : 0;
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) {
      low = fmin(low, shfl_xor_double(low, o));
      high = fmax(high, shfl_xor_double(high, o));
      whole &= __shfl_xor_sync(0xffffffffu, whole, o);
    }
    if (is_q || !live) continue;
    __nv_bfloat16 scale = bf16_of((high - low) / 15.0);
    __nv_bfloat16 centre = bf16_of(low + 8.0 * (double)__bfloat162float(scale));
    if (!whole) { scale = __float2bfloat16_rn(0.f); centre = __float2bfloat16_rn(__int_as_float(0x7fc00000)); }
    const double s = (double)__bfloat162float(scale), m = (double)__bfloat162float(centre);
    uint32_t code[2] = {0u, 0u};      // four codes each: those of e0 .., those of e1 ..
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double step = whole && s != 0.0 ? rint((x[j] - m) / s) : 0.0;
      const int u = (int)fmin(fmax(step + 8.0, 0.0), 15.0);
      code[j >> 2] |= (uint32_t)u << (4 * (j & 3));
    }
    const size_t page = slot / page_size, off = slot % page_size;
    const size_t place = (page * n_kv + (is_k ? head - n_q : head - n_q - n_kv)) * page_size + off;
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

// Eight values a thread: keys (blockIdx.y = 0) or values (1) of the slots, as bfloat16.
template <int D>
__global__ void __launch_bounds__(256)
kv_read_int4_kernel(const unsigned char* __restrict__ k_codes, const __nv_bfloat162* __restrict__ k_scales,
                    const unsigned char* __restrict__ v_codes, const __nv_bfloat162* __restrict__ v_scales,
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
  const int heads = n_q + 2 * n_kv, rows_at_once = 256 / (D / 8);
  // few tokens: a block for every pass over the heads, so that the launch is one round trip long; many: a token's sines once
  const int heads_a_block = tokens <= 512 ? rows_at_once : heads;
  const dim3 grid((unsigned)tokens, (unsigned)((heads + heads_a_block - 1) / heads_a_block));
#define LSE_INT4_WRITE(PAIRING)                                                                                          \
  lse_launch(rope_kv_write_int4_kernel<TI, D, PAIRING>, grid, dim3(256), 0, stream, (const TI*)qkv, n_partials, partial_stride, \
             bias, positions, slot_mapping, inv_freq, (__nv_bfloat16*)q_out, (unsigned char*)k_codes,                   \
             (__nv_bfloat162*)k_scales, (unsigned char*)v_codes, (__nv_bfloat162*)v_scales, n_q, n_kv, page_size, qkv_stride, \
             num_slots, heads_a_block)
  const cudaError_t err = pairing == 0 ? LSE_INT4_WRITE(0) : LSE_INT4_WRITE(1);
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
      (((uintptr_t)bias | (uintptr_t)inv_freq | (uintptr_t)q_out | (uintptr_t)k_codes | (uintptr_t)k_scales | (uintptr_t)v_codes |
        (uintptr_t)v_scales) & 15))
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
      (((uintptr_t)k_codes | (uintptr_t)k_scales | (uintptr_t)v_codes | (uintptr_t)v_scales | (uintptr_t)k_out | (uintptr_t)v_out) & 15))
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

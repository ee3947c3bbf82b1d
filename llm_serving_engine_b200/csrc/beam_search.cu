// Beam search on the device: the choice of the best continuations, and what follows from it for block tables, pages and states.
//
// A request has K beams (at most 32), each with a score (sum of log probabilities).  Beam k offers score_k + logit_kv - lse_k for
// every token v, lse_k = log sum_v exp(logit_kv); a beam that has ended offers itself once more (its end token, its score
// unchanged).  The K best of all K V offers are the next beams, the best first; of equal ones the lower beam, then the lower token.
// A beam whose score is minus infinity, or whose lse is not a number, offers nothing.
//
// Two launches.  chunk: a warp takes a piece of a beam's row, once from memory into registers, and leaves its maximum and its sum of
// exponentials, a block its K best logits (only these can be among the request's K best).  Candidates are found without a sort: of the
// lanes' 32 maxima the K-th largest is a bound that at least K values reach, and hardly more than K do.
// merge: a block per request, from the chunks' leavings.  Warps' sums are added up, and offers made and compared, in 64 bits: two beams'
// offers can be closer than float32 tells apart.  A warp's own sum is float32 (a logit's exponential is off by |logit - maximum| 2^-22
// and the approximation's 2^-22, the 64 additions a lane by 2^-24 each), so a row's lse is off by 2^-22 as a rule, and two beams'
// offers that are closer than that may come in either order; offers of one beam share its lse, and may not.
// What bounds the choice: the logits are read once, 4 bytes each.  256 rows of 151,936 (32 requests of 8 beams, 156 MB) take 36 us for
// both launches, 4.3 TB/s: the second turn of the SMs' blocks ends unevenly, and merge is 4 us; 4 rows 8.9 us, most of it the two
// launches' latencies.  Pieces of twice the length 37 to 40 us, one more block an SM 38, loads past the L1 44.
//
// The last kernels of a step: the next step's read its block tables before they wait for the kernels before them (scores, tokens and parents
// after that).  So merge and reorder never let the next kernel start early, reorder's threads that write tables end with a fence, and the
// engine's beam search has ordinary launches between them and the step.
#include "common.cuh"

namespace {

constexpr int MAX_BEAMS = 32;
constexpr int SMS = 148;             // of a B200, which all this is compiled for
constexpr float LOG2E = 1.4426950408889634f;

struct Best { float value; int token; };
struct Sum { double sum; float maximum; };      // of a chunk: its exponentials add up to sum exp(maximum)

constexpr int CHUNK_WARPS = 4, GROUPS = 32;
constexpr int LIST = 512;          // candidates above the bound that merge has room for (ties can make them any number)
constexpr int WARP_LIST = 64;      // ... and a warp of the chunks

__device__ __forceinline__ double shfl_xor_double(double v, int o) {
  return __hiloint2double(__shfl_xor_sync(0xffffffffu, __double2hiint(v), o), __shfl_xor_sync(0xffffffffu, __double2loint(v), o));
}

// The K-th largest of 32 values, one a lane (K <= 32; equal ones count as often as they are there): every lane gets it.
__device__ __forceinline__ double kth_of_lanes(double mine, int k) {
  int rank = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const double other = __hiloint2double(__shfl_sync(0xffffffffu, __double2hiint(mine), i), __shfl_sync(0xffffffffu, __double2loint(mine), i));
    rank += other > mine || (other == mine && i < (int)(threadIdx.x & 31)) ? 1 : 0;
  }
  const unsigned who = __ballot_sync(0xffffffffu, rank == k - 1);
  const int lane = __ffs(who) - 1;
  return __hiloint2double(__shfl_sync(0xffffffffu, __double2hiint(mine), lane), __shfl_sync(0xffffffffu, __double2loint(mine), lane));
}
__device__ __forceinline__ float kth_of_lanes(float mine, int k) {
  const unsigned bits = __float_as_uint(mine);
  unsigned key = bits & 0x80000000u ? ~bits : bits | 0x80000000u;      // in the order of the values
  for (;;) {                                                           // (the largest are taken out until K are: at most K times)
    const unsigned largest = __reduce_max_sync(0xffffffffu, key);
    const unsigned who = __ballot_sync(0xffffffffu, key == largest);
    k -= __popc(who);
    if (k <= 0) return __uint_as_float(largest & 0x80000000u ? largest & 0x7fffffffu : ~largest);
    if (key == largest) key = 0u;                                      // (below the key of minus infinity)
  }
}
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) { uint64_t v; asm("mov.b64 %0, {%1, %2};\n" : "=l"(v) : "f"(lo), "f"(hi)); return v; }
__device__ __forceinline__ void halves_of(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;\n" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t add_pairs(uint64_t a, uint64_t b) { uint64_t v; asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(v) : "l"(a), "l"(b)); return v; }
__device__ __forceinline__ uint64_t mul_pairs(uint64_t a, uint64_t b) { uint64_t v; asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(v) : "l"(a), "l"(b)); return v; }

// A warp takes STEPS * 512 neighbouring values of a row, sixteen a lane at a time with the next sixteen on their way, by itself: nothing
// waits at a block's barrier (a block for a piece, with four barriers, took 41 us for 256 rows of 151,936 values, 79 us with the
// next pieces copied ahead).  Of every step a lane keeps its largest value only.  In the end the K-th largest of the lanes' 32 maxima is
// a bound, and the few (lane, step) whose largest reaches it are read once more; looking for candidates among all values as they
// pass cost as much as the exponentials (46 us).  The block's warps then leave the K best of all of them together.
// Values are read one a lane, in the order of the row, whatever its alignment: equal rows leave equal sums.
constexpr int STEP = 16;
template <int STEPS>
__global__ void __launch_bounds__(CHUNK_WARPS * 32, 9)
beam_chunk_kernel(const float* logits, long long row_stride, int vocab, int beams, const float* scores,
                  const int* ended, Best* best, Sum* sums) {
  __shared__ Best list[CHUNK_WARPS][WARP_LIST], kept[CHUNK_WARPS * MAX_BEAMS];
  __shared__ float warp_max_s[CHUNK_WARPS], warp_sum_s[CHUNK_WARPS];
  __shared__ unsigned short pair_s[CHUNK_WARPS][WARP_LIST];
  pdl_launch_dependents();     // (merge: it waits before it reads anything)
  pdl_wait();
  const int row = blockIdx.y, chunk = blockIdx.x, chunks = gridDim.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (ended[row] != 0 || scores[row] == -INFINITY) return;      // what this beam offers needs no logits
  const float* src = logits + (size_t)row * row_stride;
  const int first = (chunk * CHUNK_WARPS + warp) * (STEPS * STEP * 32) + lane;
  float v[2][STEP];
  auto load = [&](int s, float (&to)[STEP]) {
    const int at = first + s * (STEP * 32);
    if (at - lane + STEP * 32 <= vocab) {
#pragma unroll
      for (int j = 0; j < STEP; ++j) to[j] = src[at + j * 32];
    } else {
#pragma unroll
      for (int j = 0; j < STEP; ++j) to[j] = at + j * 32 < vocab ? src[at + j * 32] : -INFINITY;
    }
  };
  load(0, v[0]);
  float step_top[STEPS], maximum = -INFINITY;      // `maximum`: what the sum is relative to, within e^40 of the largest
  uint64_t sums_2 = 0;
  const uint64_t log2e = pair_of(LOG2E, LOG2E);
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    if (s + 1 < STEPS) load(s + 1, v[(s + 1) & 1]);
    const float (&x)[STEP] = v[s & 1];
    float top = x[0];
#pragma unroll
    for (int j = 1; j < STEP; ++j) top = fmaxf(top, x[j]);
    if (isnan(top)) top = -INFINITY;
    step_top[s] = top;
    if (__any_sync(0xffffffffu, top > maximum + 40.f)) {
      const float higher = warp_max(fmaxf(top, maximum));
      const float w = maximum == -INFINITY ? 1.f : exp2f((maximum - higher) * LOG2E);      // (a sum of zero, or not a number, stays)
      sums_2 = mul_pairs(sums_2, pair_of(w, w));
      maximum = higher;
    }
    const float zero = maximum == -INFINITY ? 0.f : maximum;
    const uint64_t less = pair_of(-zero, -zero);
#pragma unroll
    for (int j = 0; j < STEP; j += 2) {
      float a, b;
      halves_of(mul_pairs(add_pairs(pair_of(x[j], x[j + 1]), less), log2e), a, b);
      asm("ex2.approx.ftz.f32 %0, %0;\n" : "+f"(a));
      asm("ex2.approx.ftz.f32 %0, %0;\n" : "+f"(b));
      sums_2 = add_pairs(sums_2, pair_of(a, b));
    }
  }
  float sum, more, top = step_top[0];
#pragma unroll
  for (int s = 1; s < STEPS; ++s) top = fmaxf(top, step_top[s]);
  halves_of(sums_2, sum, more);
  sum = warp_sum(sum + more);
  const float bound = fmaxf(kth_of_lanes(top, beams), -3.402823466e38f);      // (minus infinity is no candidate, nor what stands behind the row)
  if (lane == 0) { warp_max_s[warp] = maximum; warp_sum_s[warp] = sum; }
  // the warp's K best: what reaches the bound, ranked
  Best* mine = kept + warp * beams;
  if (lane < beams) mine[lane] = {-INFINITY, -1};
  __syncwarp();
  // the (step, lane) whose largest reaches the bound, then their values: eight of them on their way at a time, two a load
  int pairs = 0, found = 0;       // the same in all lanes
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const unsigned who = __ballot_sync(0xffffffffu, step_top[s] >= bound);
    const int at = pairs + __popc(who & ((1u << lane) - 1u));
    if (step_top[s] >= bound && at < WARP_LIST) pair_s[warp][at] = (unsigned short)(s * 32 + lane);
    pairs += __popc(who);
  }
  __syncwarp();
  if (pairs > WARP_LIST) found = pairs;
  else
    for (int p0 = 0; p0 < pairs; p0 += 8) {
      float value[4];
      int token[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int p = p0 + 2 * u + (lane >> 4), pair = p < pairs ? pair_s[warp][p] : 0;
        token[u] = first - lane + (pair >> 5) * (STEP * 32) + (pair & 31) + (lane & 15) * 32;
        value[u] = p < pairs && token[u] < vocab ? src[token[u]] : -INFINITY;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const unsigned reach = __ballot_sync(0xffffffffu, value[u] >= bound);
        const int at = found + __popc(reach & ((1u << lane) - 1u));
        if (value[u] >= bound && at < WARP_LIST) list[warp][at] = {value[u], token[u]};
        found += __popc(reach);
      }
    }
  __syncwarp();
  if (found <= WARP_LIST) {
    for (int i = lane; i < found; i += 32) {
      const Best b = list[warp][i];
      int rank = 0;
      for (int k = 0; k < found; ++k) {
        const Best o = list[warp][k];
        rank += o.value > b.value || (o.value == b.value && o.token < b.token) ? 1 : 0;
      }
      if (rank < beams) mine[rank] = b;
    }
  } else {
    // more ties than the list has room for: one by one, each the best of what comes after the one before
    float last_v = INFINITY;
    int last_t = -1;
    for (int k = 0; k < beams; ++k) {
      float bv = -INFINITY;
      int bt = 0x7fffffff;
#pragma unroll 4
      for (int i = first; i < min(vocab, first + STEPS * STEP * 32); i += 32) {
        const float x = src[i];
        const bool after = x < last_v || (x == last_v && i > last_t);
        if (after && x > bv) { bv = x; bt = i; }       // (tokens ascend: the first of equal ones stays)
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
        const int ot = __shfl_xor_sync(0xffffffffu, bt, o);
        if (ov > bv || (ov == bv && ot < bt)) { bv = ov; bt = ot; }
      }
      last_v = bv; last_t = bt;
      if (lane == 0 && bv != -INFINITY) mine[k] = {bv, bt};
    }
  }
  __syncthreads();
  if (warp == 0) {       // the block's sum, relative to its maximum
    const float m = lane < CHUNK_WARPS ? warp_max_s[lane] : -INFINITY, highest = warp_max(m);
    double s = lane < CHUNK_WARPS ? (double)warp_sum_s[lane] : 0.0;
    if (m != -INFINITY && m != highest) s *= exp((double)m - (double)highest);
#pragma unroll
    for (int o = CHUNK_WARPS / 2; o > 0; o >>= 1) s += shfl_xor_double(s, o);
    if (lane == 0) sums[(size_t)row * chunks + chunk] = {s, highest};
  }
  // The block's best: one's rank is its place in its own warp's list and how far it comes in the others', which are in order too.
  Best* out = best + ((size_t)row * chunks + chunk) * beams;
  for (int i = tid; i < CHUNK_WARPS * beams; i += CHUNK_WARPS * 32) {
    const int own = i / beams;
    int rank = i - own * beams;
    const Best b = kept[i];
    for (int w = 0; w < CHUNK_WARPS; ++w) {
      if (w == own) continue;
      // (of equal values the lower token is in the lower warp; an empty place is behind every other, and counts once)
      for (int k = 0; k < beams && rank < beams; ++k, ++rank) {
        const float other = kept[w * beams + k].value;
        if (!(other > b.value || (other == b.value && w < own))) break;
      }
    }
    if (rank < beams) out[rank] = b;
  }
}

// One block per request.  HELD: offers a thread keeps in registers; beyond them they are read again.
template <int MERGE_THREADS, int HELD>
__global__ void __launch_bounds__(MERGE_THREADS)
beam_merge_kernel(const Best* best, const Sum* sums, int chunks, int beams,
                  const float* scores, const int* ended, int end_token, float* out_scores,
                  int* out_tokens, int* out_parents, int* out_ended) {
  constexpr int WARPS = MERGE_THREADS / 32, GROUP_LANES = MERGE_THREADS / GROUPS;
  __shared__ double lse[MAX_BEAMS], group_top[GROUPS], bound_s, list_v[LIST];
  __shared__ long long list_at[LIST];
  __shared__ int over[MAX_BEAMS], count;
  __shared__ float score[MAX_BEAMS];
  pdl_wait();
  const int request = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t row0 = (size_t)request * beams;
  // what beam b offers: all that its chunks left, or (ended) itself; numbered beam by beam
  const int a_beam = chunks * beams, total = a_beam * beams;
  const Best* mine = best + row0 * a_beam;
  Best held[HELD];
#pragma unroll
  for (int j = 0; j < HELD; ++j) {      // (what beams without logits have left is anything at all, and is not looked at below)
    const int i = tid + j * MERGE_THREADS;
    held[j] = i < total ? mine[i] : Best{-INFINITY, -1};
  }
  if (tid == 0) count = 0;
  for (int beam = warp; beam < beams; beam += WARPS) {
    const int stopped = ended[row0 + beam] != 0;
    const float before = scores[row0 + beam];
    double sum = 0.0;
    float top = -INFINITY;
    if (!stopped && before != -INFINITY) {
      const Sum* parts = sums + (row0 + beam) * chunks;
      for (int c = lane; c < chunks; c += 32) {
        const Sum s = parts[c];
        // a chunk of nothing but minus infinity has a sum of zero (or not a number, which must stay)
        if (s.maximum > top) { sum = (top == -INFINITY ? sum : sum * exp((double)top - (double)s.maximum)) + s.sum; top = s.maximum; }
        else sum += s.maximum == -INFINITY ? s.sum : s.sum * exp((double)s.maximum - (double)top);
      }
    }
    const float highest = warp_max(top);
    if (top != -INFINITY && top != highest) sum *= exp((double)top - (double)highest);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += shfl_xor_double(sum, o);
    if (lane == 0) { lse[beam] = (double)highest + log(sum); over[beam] = stopped; score[beam] = before; }
  }
  __syncthreads();
  auto offer = [&](int i, Best b, double& value, long long& at) {
    const int beam = (unsigned)i / (unsigned)a_beam;
    value = -INFINITY;
    at = 0x7fffffffffffffffLL;
    if (score[beam] == -INFINITY) return;
    if (over[beam]) {
      if (i == beam * a_beam) { value = (double)score[beam]; at = (long long)beam << 32 | end_token; }
      return;
    }
    if (b.token < 0) return;
    const double v = (double)score[beam] + ((double)b.value - lse[beam]);
    if (v > -INFINITY) { value = v; at = (long long)beam << 32 | b.token; }     // (not a number: nothing)
  };
  double value[HELD];
  long long at[HELD];
  double top = -INFINITY;
#pragma unroll
  for (int j = 0; j < HELD; ++j) {
    const int i = tid + j * MERGE_THREADS;
    value[j] = -INFINITY;
    at[j] = 0x7fffffffffffffffLL;
    if (i < total) offer(i, held[j], value[j], at[j]);
    top = fmax(top, value[j]);
  }
  for (int i = tid + HELD * MERGE_THREADS; i < total; i += MERGE_THREADS) {
    double v; long long a;
    offer(i, mine[i], v, a);
    top = fmax(top, v);
  }
#pragma unroll
  for (int o = 1; o < GROUP_LANES; o <<= 1) top = fmax(top, shfl_xor_double(top, o));
  if ((tid & (GROUP_LANES - 1)) == 0) group_top[tid / GROUP_LANES] = top;
  __syncthreads();
  if (warp == 0) {
    const double bound = kth_of_lanes(group_top[lane], beams);
    if (lane == 0) bound_s = bound;
  }
  __syncthreads();
  const double bound = bound_s;
  auto take = [&](double v, long long a) {
    if (v >= bound && v > -INFINITY) {
      const int place = atomicAdd(&count, 1);
      if (place < LIST) { list_v[place] = v; list_at[place] = a; }
    }
  };
#pragma unroll
  for (int j = 0; j < HELD; ++j) take(value[j], at[j]);
  for (int i = tid + HELD * MERGE_THREADS; i < total; i += MERGE_THREADS) {
    double v; long long a;
    offer(i, mine[i], v, a);
    take(v, a);
  }
  __syncthreads();
  auto put = [&](int rank, double value, long long at) {
    const int parent = (int)(at >> 32), token = (int)(at & 0xffffffffLL);
    out_scores[row0 + rank] = (float)value;
    out_tokens[row0 + rank] = token;
    out_parents[row0 + rank] = parent;
    out_ended[row0 + rank] = over[parent] || token == end_token ? 1 : 0;
  };
  auto nothing = [&](int rank) {
    out_scores[row0 + rank] = -INFINITY;
    out_tokens[row0 + rank] = end_token;
    out_parents[row0 + rank] = rank;
    out_ended[row0 + rank] = 1;
  };
  const int found = count;
  if (found <= LIST) {
    for (int i = tid; i < found; i += MERGE_THREADS) {
      int rank = 0;
      for (int k = 0; k < found; ++k) rank += list_v[k] > list_v[i] || (list_v[k] == list_v[i] && list_at[k] < list_at[i]) ? 1 : 0;
      if (rank < beams) put(rank, list_v[i], list_at[i]);
    }
    for (int i = found + tid; i < beams; i += MERGE_THREADS) nothing(i);
    return;
  }
  // more ties than the list has room for: one by one
  __shared__ double win_v[WARPS];
  __shared__ long long win_at[WARPS];
  double last_v = INFINITY;
  long long last_at = -1;
  for (int k = 0; k < beams; ++k) {
    double bv = -INFINITY;
    long long ba = 0x7fffffffffffffffLL;
    for (int i = tid; i < total; i += MERGE_THREADS) {
      double v; long long a;
      offer(i, mine[i], v, a);
      const bool after = v < last_v || (v == last_v && a > last_at);
      if (after && (v > bv || (v == bv && a < ba))) { bv = v; ba = a; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ov = shfl_xor_double(bv, o);
      const long long oa = __shfl_xor_sync(0xffffffffu, ba, o);
      if (ov > bv || (ov == bv && oa < ba)) { bv = ov; ba = oa; }
    }
    __syncthreads();
    if (lane == 0) { win_v[warp] = bv; win_at[warp] = ba; }
    __syncthreads();
    last_v = win_v[0]; last_at = win_at[0];
    for (int w = 1; w < WARPS; ++w)
      if (win_v[w] > last_v || (win_v[w] == last_v && win_at[w] < last_at)) { last_v = win_v[w]; last_at = win_at[w]; }
    if (tid == 0) { if (last_v > -INFINITY) put(k, last_v, last_at); else nothing(k); }
  }
}

// ------------------------------------------------------------------ after the choice
// New block tables.  All beams of a request hold `length` tokens: `length / page_size` full pages, which several beams may share,
// and, unless that divides, a page that is being filled, which is a beam's own.  Pages behind it are the row's and empty.
// Beam i goes on from parents[i]: its full pages are the parent's.  The first of a parent's children takes over the page that
// the parent was filling; every further child takes that of a beam without a child (there are as many of either), and the
// parent's page is copied into it.  No page is read that another child's copy writes, so the copies need no order.
// What bounds it: the bytes of the pages that have to be copied, read and written once (16 requests of 8 beams, 28 layers of 4 heads of
// 128 in bfloat16: 77 MB in 18 to 21 us, 3.7 to 4.4 TB/s), or the launch where there are few (2.9 us).
constexpr int MAX_STORAGES = 24;
// A page's words (of sizeof V) are copied in pieces of PIECE; 1 << lane_bits threads take a piece's words, the rest of a block's further
// outer parts; `items` pieces for the whole storage.
constexpr int PIECE = 2048;
struct Storage { unsigned char* base; long long outer_stride, page_stride; int outer, pages, words, lane_bits, pieces, items; };
struct Storages { Storage s[MAX_STORAGES]; int n; };

template <typename V>
__global__ void __launch_bounds__(256)
beam_reorder_kernel(const int* parents, int beams, const int* tables, int table_stride, int width,
                    const int* lengths, int page_size, int* new_tables, int new_stride,
                    const __grid_constant__ Storages storages) {
  pdl_wait();
  const int row = blockIdx.x, request = row / beams, beam = row - request * beams, lane = threadIdx.x & 31;
  // every warp works out all beams' sources, a beam a lane
  const bool live = lane < beams;
  const int parent = live ? min(max(parents[(size_t)request * beams + lane], 0), beams - 1) : beams + lane;
  const bool first = __ffs(__match_any_sync(0xffffffffu, parent)) - 1 == lane;
  const unsigned more = __ballot_sync(0xffffffffu, live && !first);
  const unsigned with_child = __reduce_or_sync(0xffffffffu, live ? 1u << parent : 0u);
  const unsigned childless = ~with_child & (beams == 32 ? 0xffffffffu : (1u << beams) - 1u);
  const int my_parent = __shfl_sync(0xffffffffu, parent, beam);
  const bool copies = (more >> beam & 1u) != 0;
  unsigned left = childless;       // (as many childless beams as further children: the n-th takes over the n-th)
  for (int n = __popc(more & ((1u << beam) - 1u)); copies && n > 0; --n) left &= left - 1u;
  const int taken = copies ? __ffs(left) - 1 : my_parent;

  const int length = lengths[request], full = length / page_size;
  const bool filling = length > 0 && length % page_size != 0 && full < width;
  const int* from = tables + ((size_t)request * beams + my_parent) * table_stride;
  const int* own = tables + (size_t)row * table_stride;
  const int source = filling ? from[full] : -1, target = filling ? tables[((size_t)request * beams + taken) * table_stride + full] : -1;
  if (blockIdx.y == 0 && new_tables != nullptr)
    for (int i = threadIdx.x; i < width; i += blockDim.x)
      new_tables[(size_t)row * new_stride + i] = i < full ? from[i] : (i == full && filling) ? target : own[i];
  if (blockIdx.y == 0) __threadfence();
  if (!copies || !filling) return;
  for (int k = 0; k < storages.n; ++k) {
    const Storage& s = storages.s[k];
    if (source < 0 || source >= s.pages || target < 0 || target >= s.pages || source == target) continue;
    const unsigned char* src = s.base + source * s.page_stride;
    unsigned char* dst = s.base + target * s.page_stride;
    const int lanes = 1 << s.lane_bits, word0 = threadIdx.x & (lanes - 1), outer0 = threadIdx.x >> s.lane_bits;
    for (int item = blockIdx.y; item < s.items; item += gridDim.y) {
      const int group = item / s.pieces, first = (item - group * s.pieces) * PIECE;
      const int outer = (group << (8 - s.lane_bits)) + outer0, end = min(s.words, first + PIECE);
      if (outer >= s.outer) continue;
      const V* from_words = reinterpret_cast<const V*>(src + outer * s.outer_stride);
      V* to_words = reinterpret_cast<V*>(dst + outer * s.outer_stride);
      for (int i = first + word0; i < end; i += 8 * lanes) {
        V v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (i + u * lanes < end) v[u] = from_words[i + u * lanes];
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (i + u * lanes < end) to_words[i + u * lanes] = v[u];
      }
    }
  }
}

int steps_of(long long rows, int vocab) {
  // the largest pieces that leave a block for each SM, or the smallest (4 rows of 151,936 values: 8.3 us with two steps, 9.5 with
  // one; 120 of 100,001: 19.7 with eight, 21.9 with two)
  int steps = 8;
  while (steps > 1 && rows * vocab < (long long)SMS * CHUNK_WARPS * steps * STEP * 32) steps /= 2;
  return steps;
}
int chunks_of(long long rows, int vocab) {
  const int c = CHUNK_WARPS * 32 * STEP * steps_of(rows, vocab);
  return (int)((vocab + (long long)c - 1) / c);
}
long long best_bytes(long long rows, int chunks, int beams) { return (rows * chunks * beams * (long long)sizeof(Best) + 15) / 16 * 16; }

}  // namespace

// Bytes of scratch that lse_beam_select needs, in units of 1024 (at most 2^31 - 1 of them).
extern "C" int lse_beam_select_scratch_kb(int requests, int beams, int vocab) {
  if (requests <= 0 || beams <= 0 || vocab <= 0) return 0;
  const long long rows = (long long)requests * beams;
  const int chunks = chunks_of(rows, vocab);
  return (int)((best_bytes(rows, chunks, beams) + rows * chunks * (long long)sizeof(Sum) + 1023) / 1024);
}

// logits float32 [requests * beams, vocab] (rows row_stride apart); scores float32, ended int32 [requests, beams]; the outputs alike.
extern "C" int lse_beam_select(const float* logits, long long row_stride, int requests, int beams, int vocab, const float* scores,
                               const int* ended, int end_token, void* scratch, float* out_scores, int* out_tokens,
                               int* out_parents, int* out_ended, cudaStream_t stream) {
  if (requests <= 0) return 0;
  if (beams < 1 || beams > MAX_BEAMS || vocab < 1 || row_stride < vocab || end_token < 0 || end_token >= vocab || scratch == nullptr ||
      ((uintptr_t)scratch & 15) || ((uintptr_t)logits & 3))
    return LSE_ERR_BAD_ARGUMENT;
  const long long rows = (long long)requests * beams;
  const int chunks = chunks_of(rows, vocab);
  if (rows > 65535 || (long long)chunks * beams * beams > 0x7fffffffLL) return LSE_ERR_TOO_LARGE;
  Best* best = (Best*)scratch;
  Sum* sums = (Sum*)((unsigned char*)scratch + best_bytes(rows, chunks, beams));
  cudaError_t err;
#define LSE_BEAM_CHUNK(STEPS)                                                                                               \
  lse_launch(beam_chunk_kernel<STEPS>, dim3((unsigned)chunks, (unsigned)rows), dim3(CHUNK_WARPS * 32), 0, stream, logits, row_stride, vocab, \
             beams, scores, ended, best, sums)
  const int steps = steps_of(rows, vocab);
  err = steps == 8 ? LSE_BEAM_CHUNK(8) : steps == 4 ? LSE_BEAM_CHUNK(4) : steps == 2 ? LSE_BEAM_CHUNK(2) : LSE_BEAM_CHUNK(1);
#undef LSE_BEAM_CHUNK
  if (err != cudaSuccess) return (int)err;
#define LSE_BEAM_MERGE(THREADS, HELD)                                                                                        \
  lse_launch(beam_merge_kernel<THREADS, HELD>, dim3((unsigned)requests), dim3(THREADS), 0, stream, (const Best*)best, (const Sum*)sums, chunks, \
             beams, scores, ended, end_token, out_scores, out_tokens, out_parents, out_ended)
  err = (long long)chunks * beams * beams <= 256 * 8 ? LSE_BEAM_MERGE(256, 8) : LSE_BEAM_MERGE(1024, 4);
#undef LSE_BEAM_MERGE
  if (err != cudaSuccess) return (int)err;
  LSE_LAUNCH_CHECK();
}

// storages: n of them, each five numbers: address, outer count, bytes between outer parts, bytes between pages, bytes of a page; and
// pages[i].  new_tables may be null (a further group of storages behind the same tables).
extern "C" int lse_beam_reorder(const int* parents, int requests, int beams, const int* tables, int table_stride, int width,
                                const int* lengths, int page_size, int* new_tables, int new_stride, const long long* storages, int n,
                                cudaStream_t stream) {
  if (requests <= 0) return 0;
  if (beams < 1 || beams > MAX_BEAMS || width < 1 || page_size < 1 || n < 0 || n > MAX_STORAGES || (n > 0 && storages == nullptr))
    return LSE_ERR_BAD_ARGUMENT;
  Storages list;
  list.n = n;
  unsigned long long bits = 0;
  for (int i = 0; i < n; ++i) {
    const long long* s = storages + 6 * i;
    if (s[0] == 0 || s[1] < 0 || s[1] > 0x7fffffffLL || s[4] < 0 || s[5] < 0 || s[5] > 0x7fffffffLL) return LSE_ERR_BAD_ARGUMENT;
    bits |= (unsigned long long)(s[0] | s[2] | s[3] | s[4]);
  }
  const int word = (bits & 15) == 0 ? 16 : (bits & 3) == 0 ? 4 : 1;
  int most = 1;
  for (int i = 0; i < n; ++i) {
    const long long* s = storages + 6 * i;
    if (s[4] / word > 0x7fffffffLL - 8 * 256) return LSE_ERR_TOO_LARGE;
    Storage& to = list.s[i];
    to = {(unsigned char*)s[0], s[2], s[3], (int)s[1], (int)s[5], (int)(s[4] / word), 0, 0, 0};
    while (to.lane_bits < 8 && 1 << to.lane_bits < to.words) ++to.lane_bits;
    to.pieces = (to.words + PIECE - 1) / PIECE;
    const long long items = (((long long)to.outer + (1 << (8 - to.lane_bits)) - 1) >> (8 - to.lane_bits)) * to.pieces;
    if (items > 0x7fffffffLL) return LSE_ERR_TOO_LARGE;
    to.items = (int)items;
    if (to.items > most) most = to.items;
  }
  const long long rows = (long long)requests * beams;
  // about eight blocks an SM, two thirds of which find nothing to copy (a child that goes on in its parent's page)
  const long long slices = rows < 8 * SMS ? 8 * SMS / rows : 1;
  const dim3 grid((unsigned)rows, (unsigned)(most > slices ? slices : most));
#define LSE_REORDER(V) lse_launch(beam_reorder_kernel<V>, grid, dim3(256), 0, stream, parents, beams, tables, table_stride, width, lengths, \
                                  page_size, new_tables, new_stride, list)
  const cudaError_t err = word == 16 ? LSE_REORDER(uint4) : word == 4 ? LSE_REORDER(uint32_t) : LSE_REORDER(unsigned char);
#undef LSE_REORDER
  if (err != cudaSuccess) return (int)err;
  LSE_LAUNCH_CHECK();
}

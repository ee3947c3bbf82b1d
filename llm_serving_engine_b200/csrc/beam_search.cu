// Beam search on the device: the choice of the best continuations, and what follows from it for block tables, pages and states.
//
// A request has K beams (at most 32), each with a score (sum of log probabilities).  Beam k offers score_k + logit_kv - lse_k for
// every token v, lse_k = log sum_v exp(logit_kv); a beam that has ended offers itself once more (its end token, its score
// unchanged).  The K best of all K V offers are the next beams, the best first; of equal ones the lower beam, then the lower token.
// A beam whose score is minus infinity, or whose lse is not a number, offers nothing.
//
// Two launches.  chunk: a block takes a piece of a beam's row, once from memory into registers, and leaves its maximum, its sum of
// exponentials and its K best logits (only these can be among the request's K best).  Candidates are found without a sort: 32
// groups of threads give 32 maxima, the K-th largest of them is a bound that at least K values reach, and hardly more than K do.
// merge: a block per request, from the chunks' leavings.  Offers are compared in 64 bits: two beams' offers can be closer than
// float32 tells apart, and lse's error would decide.
// What bounds the choice: the logits are read once, 4 bytes each.
//
// The last kernels of a step: the next step's read its metadata (token ids, block tables) before they wait for the kernels before
// them.  So the kernels here that write metadata never let the next one start early.
#include "common.cuh"

namespace {

constexpr int MAX_BEAMS = 32;
constexpr float LOG2E = 1.4426950408889634f;

struct Best { float value; int token; };
struct Sum { double maximum, sum; };      // of a chunk; the sum relative to the maximum

constexpr int CHUNK_THREADS = 256, GROUPS = 32;
constexpr int LIST = 512;          // candidates above the bound that a block has room for (ties can make them any number)

// The K-th largest of 32 values, one a lane (K <= 32): every lane gets it.
template <typename V> __device__ __forceinline__ V kth_of_lanes(V mine, int k) {
  int rank = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const V other = __shfl_sync(0xffffffffu, mine, i);
    rank += other > mine || (other == mine && i < (int)(threadIdx.x & 31)) ? 1 : 0;
  }
  const unsigned who = __ballot_sync(0xffffffffu, rank == k - 1);
  return __shfl_sync(0xffffffffu, mine, __ffs(who) - 1);
}

template <int VALUES>      // values a thread holds (a multiple of 4)
__global__ void __launch_bounds__(CHUNK_THREADS)
beam_chunk_kernel(const float* __restrict__ logits, long long row_stride, int vocab, int beams, const float* __restrict__ scores,
                  const int* __restrict__ ended, Best* __restrict__ best, Sum* __restrict__ sums) {
  constexpr int CHUNK = CHUNK_THREADS * VALUES;
  __shared__ float group_max[GROUPS], bound_s;
  __shared__ double part[CHUNK_THREADS / 32];
  __shared__ int count;
  __shared__ Best list[LIST];
  pdl_launch_dependents();     // (merge: it waits before it reads anything)
  pdl_wait();
  const int row = blockIdx.y, chunk = blockIdx.x, chunks = gridDim.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (ended[row] != 0 || scores[row] == -INFINITY) return;      // what this beam offers needs no logits
  const float* src = logits + (size_t)row * row_stride;
  // chunks begin at 16-byte boundaries, the first one up to three values before the row (whose length may be odd)
  const int first = chunk * CHUNK - (int)(((uintptr_t)src >> 2) & 3);
  float v[VALUES];
  auto token_of = [&](int j) { return first + (j / 4 * CHUNK_THREADS + tid) * 4 + j % 4; };
#pragma unroll
  for (int j = 0; j < VALUES; j += 4) {
    const int i = token_of(j);
    if (i >= 0 && i + 4 <= vocab) {
      const float4 x = __ldcs(reinterpret_cast<const float4*>(src + i));
      v[j] = x.x; v[j + 1] = x.y; v[j + 2] = x.z; v[j + 3] = x.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j + e] = i + e >= 0 && i + e < vocab ? src[i + e] : -INFINITY;
    }
  }
  if (tid == 0) count = 0;
  float top = v[0];
#pragma unroll
  for (int j = 1; j < VALUES; ++j) top = fmaxf(top, v[j]);
#pragma unroll
  for (int o = 1; o < CHUNK_THREADS / GROUPS; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((tid & (CHUNK_THREADS / GROUPS - 1)) == 0) group_max[tid / (CHUNK_THREADS / GROUPS)] = isnan(top) ? -INFINITY : top;
  __syncthreads();
  const float maximum = warp_max(group_max[lane]);
  if (warp == 0) {
    const float bound = kth_of_lanes(group_max[lane], beams);
    if (lane == 0) bound_s = bound;
  }
  // sum of exponentials relative to the chunk's maximum: float32 inside a thread, 64 bits over the block
  const float zero = maximum == -INFINITY ? 0.f : maximum * LOG2E;
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < VALUES; ++j) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(e) : "f"(fmaf(v[j], LOG2E, -zero)));
    sum += e;
  }
  double total = (double)sum;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    total += __hiloint2double(__shfl_xor_sync(0xffffffffu, __double2hiint(total), o), __shfl_xor_sync(0xffffffffu, __double2loint(total), o));
  if (lane == 0) part[warp] = total;
  __syncthreads();
  if (tid == 0) {
    double all = 0.0;
    for (int w = 0; w < CHUNK_THREADS / 32; ++w) all += part[w];
    sums[(size_t)row * chunks + chunk] = {(double)maximum, all};
  }
  const float bound = bound_s;
#pragma unroll
  for (int j = 0; j < VALUES; ++j) {
    if (v[j] >= bound && v[j] != -INFINITY) {
      const int at = atomicAdd(&count, 1);
      if (at < LIST) list[at] = {v[j], token_of(j)};
    }
  }
  __syncthreads();
  Best* mine = best + ((size_t)row * chunks + chunk) * beams;
  const int found = count;
  if (found <= LIST) {
    for (int i = tid; i < found; i += CHUNK_THREADS) {
      const Best b = list[i];
      int rank = 0;
      for (int k = 0; k < found; ++k) rank += list[k].value > b.value || (list[k].value == b.value && list[k].token < b.token) ? 1 : 0;
      if (rank < beams) mine[rank] = b;
    }
    for (int i = found + tid; i < beams; i += CHUNK_THREADS) mine[i] = {-INFINITY, -1};
    return;
  }
  // More ties than the list has room for: one by one, each the best of what comes after the one before.
  __shared__ float win_v[CHUNK_THREADS / 32];
  __shared__ int win_t[CHUNK_THREADS / 32];
  float last_v = INFINITY;
  int last_t = -1;
  for (int k = 0; k < beams; ++k) {
    float bv = -INFINITY;
    int bt = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < VALUES; ++j) {
      const int token = token_of(j);
      const bool after = v[j] < last_v || (v[j] == last_v && token > last_t);
      if (after && (v[j] > bv || (v[j] == bv && token < bt))) { bv = v[j]; bt = token; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
      const int ot = __shfl_xor_sync(0xffffffffu, bt, o);
      if (ov > bv || (ov == bv && ot < bt)) { bv = ov; bt = ot; }
    }
    __syncthreads();
    if (lane == 0) { win_v[warp] = bv; win_t[warp] = bt; }
    __syncthreads();
    last_v = win_v[0]; last_t = win_t[0];
    for (int w = 1; w < CHUNK_THREADS / 32; ++w)
      if (win_v[w] > last_v || (win_v[w] == last_v && win_t[w] < last_t)) { last_v = win_v[w]; last_t = win_t[w]; }
    if (tid == 0) mine[k] = {last_v, last_v == -INFINITY ? -1 : last_t};
  }
}

constexpr int MERGE_THREADS = 1024;

// One block per request.
__global__ void __launch_bounds__(MERGE_THREADS)
beam_merge_kernel(const Best* __restrict__ best, const Sum* __restrict__ sums, int chunks, int beams, long long vocab,
                  const float* __restrict__ scores, const int* __restrict__ ended, int end_token, float* __restrict__ out_scores,
                  int* __restrict__ out_tokens, int* __restrict__ out_parents, int* __restrict__ out_ended) {
  __shared__ double lse[MAX_BEAMS], warp_top[32], bound_s, list_v[LIST];
  __shared__ long long list_at[LIST];
  __shared__ int over[MAX_BEAMS], count;
  __shared__ float score[MAX_BEAMS];
  pdl_wait();
  const int request = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t row0 = (size_t)request * beams;
  if (tid == 0) count = 0;
  if (warp < beams) {
    const int stopped = ended[row0 + warp] != 0;
    const float before = scores[row0 + warp];
    double sum = 0.0;
    float top = -INFINITY;
    if (!stopped && before != -INFINITY) {
      const Sum* mine = sums + (row0 + warp) * chunks;
      for (int c = lane; c < chunks; c += 32) top = fmaxf(top, (float)mine[c].maximum);
      top = warp_max(top);
      for (int c = lane; c < chunks; c += 32)      // a chunk of nothing but minus infinity has a sum of zero (or not a number)
        sum += mine[c].maximum > -INFINITY ? mine[c].sum * exp(mine[c].maximum - (double)top) : mine[c].sum;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      sum += __hiloint2double(__shfl_xor_sync(0xffffffffu, __double2hiint(sum), o), __shfl_xor_sync(0xffffffffu, __double2loint(sum), o));
    if (lane == 0) { lse[warp] = (double)top + log(sum); over[warp] = stopped; score[warp] = before; }
  }
  __syncthreads();
  // offer number i: of an ended beam its first, of the others all that the chunks left
  const int a_beam = chunks * beams, total = a_beam * beams;
  auto offer = [&](int i, double& value, long long& at) {
    const int beam = i / a_beam, k = i - beam * a_beam;
    value = -INFINITY;
    at = 0x7fffffffffffffffLL;
    if (score[beam] == -INFINITY) return;
    if (over[beam]) {
      if (k == 0) { value = (double)score[beam]; at = beam * vocab + end_token; }
      return;
    }
    const Best b = best[(row0 + beam) * a_beam + k];
    if (b.token < 0) return;
    const double v = (double)score[beam] + ((double)b.value - lse[beam]);
    if (v > -INFINITY) { value = v; at = beam * vocab + b.token; }     // (not a number: nothing)
  };
  double top = -INFINITY;
  for (int i = tid; i < total; i += MERGE_THREADS) {
    double value; long long at;
    offer(i, value, at);
    top = fmax(top, value);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    top = fmax(top, __hiloint2double(__shfl_xor_sync(0xffffffffu, __double2hiint(top), o), __shfl_xor_sync(0xffffffffu, __double2loint(top), o)));
  if (lane == 0) warp_top[warp] = top;
  __syncthreads();
  if (warp == 0) {
    const double bound = kth_of_lanes(warp_top[lane], beams);
    if (lane == 0) bound_s = bound;
  }
  __syncthreads();
  const double bound = bound_s;
  for (int i = tid; i < total; i += MERGE_THREADS) {
    double value; long long at;
    offer(i, value, at);
    if (value >= bound && value > -INFINITY) {
      const int place = atomicAdd(&count, 1);
      if (place < LIST) { list_v[place] = value; list_at[place] = at; }
    }
  }
  __syncthreads();
  auto put = [&](int rank, double value, long long at) {
    const int parent = (int)(at / vocab), token = (int)(at - (long long)parent * vocab);
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
  __shared__ double win_v[32];
  __shared__ long long win_at[32];
  double last_v = INFINITY;
  long long last_at = -1;
  for (int k = 0; k < beams; ++k) {
    double bv = -INFINITY;
    long long ba = 0x7fffffffffffffffLL;
    for (int i = tid; i < total; i += MERGE_THREADS) {
      double value; long long at;
      offer(i, value, at);
      const bool after = value < last_v || (value == last_v && at > last_at);
      if (after && (value > bv || (value == bv && at < ba))) { bv = value; ba = at; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ov = __hiloint2double(__shfl_xor_sync(0xffffffffu, __double2hiint(bv), o), __shfl_xor_sync(0xffffffffu, __double2loint(bv), o));
      const long long oa = __shfl_xor_sync(0xffffffffu, ba, o);
      if (ov > bv || (ov == bv && oa < ba)) { bv = ov; ba = oa; }
    }
    __syncthreads();
    if (lane == 0) { win_v[warp] = bv; win_at[warp] = ba; }
    __syncthreads();
    last_v = win_v[0]; last_at = win_at[0];
    for (int w = 1; w < 32; ++w)
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
constexpr int MAX_STORAGES = 24;
struct Storage { unsigned char* base; long long outer_stride, page_stride, page_bytes; int outer, pages; };
struct Storages { Storage s[MAX_STORAGES]; int n; };

template <typename V>
__global__ void __launch_bounds__(256)
beam_reorder_kernel(const int* __restrict__ parents, int beams, const int* __restrict__ tables, int table_stride, int width,
                    const int* __restrict__ lengths, int page_size, int* __restrict__ new_tables, int new_stride,
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
  const int taken = copies ? (int)__fns(childless, 0, __popc(more & ((1u << beam) - 1u)) + 1) : my_parent;

  const int length = lengths[request], full = length / page_size;
  const bool filling = length > 0 && length % page_size != 0 && full < width;
  const int* from = tables + ((size_t)request * beams + my_parent) * table_stride;
  const int* own = tables + (size_t)row * table_stride;
  const int source = filling ? from[full] : -1, target = filling ? tables[((size_t)request * beams + taken) * table_stride + full] : -1;
  if (blockIdx.y == 0 && new_tables != nullptr)
    for (int i = threadIdx.x; i < width; i += blockDim.x)
      new_tables[(size_t)row * new_stride + i] = i < full ? from[i] : (i == full && filling) ? target : own[i];
  if (!copies || !filling) return;
  for (int k = 0; k < storages.n; ++k) {
    const Storage& s = storages.s[k];
    if (source < 0 || source >= s.pages || target < 0 || target >= s.pages || source == target) continue;
    const long long per = s.page_bytes / (long long)sizeof(V), items = per * s.outer;
    const unsigned char* src = s.base + source * s.page_stride;
    unsigned char* dst = s.base + target * s.page_stride;
    const long long step = (long long)gridDim.y * 256;
    for (long long i0 = (long long)blockIdx.y * 256 + threadIdx.x; i0 < items; i0 += 4 * step) {
      V v[4];
      long long at[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const long long i = i0 + u * step;
        const long long o = i / per;
        at[u] = i < items ? o * s.outer_stride + (i - o * per) * (long long)sizeof(V) : -1;
        if (at[u] >= 0) v[u] = *reinterpret_cast<const V*>(src + at[u]);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (at[u] >= 0) *reinterpret_cast<V*>(dst + at[u]) = v[u];
    }
  }
}

int values_a_thread(long long rows, int vocab) {
  // small chunks while the launch is short of blocks: 4 rows of 151,936 tokens
  return rows * vocab >= 4LL * 148 * CHUNK_THREADS * 32 ? 32 : 8;
}
int chunks_of(long long rows, int vocab) {
  const long long c = CHUNK_THREADS * values_a_thread(rows, vocab);
  return (int)((vocab + 3LL + c - 1) / c);
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
  if (values_a_thread(rows, vocab) == 32)
    err = lse_launch(beam_chunk_kernel<32>, dim3((unsigned)chunks, (unsigned)rows), dim3(CHUNK_THREADS), 0, stream, logits, row_stride, vocab,
                     beams, scores, ended, best, sums);
  else
    err = lse_launch(beam_chunk_kernel<8>, dim3((unsigned)chunks, (unsigned)rows), dim3(CHUNK_THREADS), 0, stream, logits, row_stride, vocab,
                     beams, scores, ended, best, sums);
  if (err != cudaSuccess) return (int)err;
  err = lse_launch(beam_merge_kernel, dim3((unsigned)requests), dim3(MERGE_THREADS), 0, stream, (const Best*)best, (const Sum*)sums, chunks,
                   beams, (long long)vocab, scores, ended, end_token, out_scores, out_tokens, out_parents, out_ended);
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
  long long most = 0;
  unsigned long long bits = 0;
  for (int i = 0; i < n; ++i) {
    const long long* s = storages + 6 * i;
    list.s[i] = {(unsigned char*)s[0], s[2], s[3], s[4], (int)s[1], (int)s[5]};
    if (s[0] == 0 || s[1] < 0 || s[1] > 0x7fffffffLL || s[4] < 0 || s[5] < 0 || s[5] > 0x7fffffffLL) return LSE_ERR_BAD_ARGUMENT;
    bits |= (unsigned long long)(s[0] | s[2] | s[3] | s[4]);
    if (s[1] * s[4] > most) most = s[1] * s[4];
  }
  const long long rows = (long long)requests * beams;
  // about 32 KB a block: eight 16-byte words a thread
  const long long slices = most <= 32768 ? 1 : (most + 32767) / 32768;
  const dim3 grid((unsigned)rows, (unsigned)(slices > 1024 ? 1024 : slices));
#define LSE_REORDER(V) lse_launch(beam_reorder_kernel<V>, grid, dim3(256), 0, stream, parents, beams, tables, table_stride, width, lengths, \
                                  page_size, new_tables, new_stride, list)
  const cudaError_t err = (bits & 15) == 0 ? LSE_REORDER(uint4) : (bits & 3) == 0 ? LSE_REORDER(uint32_t) : LSE_REORDER(unsigned char);
#undef LSE_REORDER
  if (err != cudaSuccess) return (int)err;
  LSE_LAUNCH_CHECK();
}

// What a step's kernels have to know about its rows, made on the device from the requests' lengths: first rows, every row's request,
// position and cache slot, contexts, and block tables padded to a width.  For steps whose requests are known on the device only
// (the beams of a beam search), and for hosts that would rather send a few numbers a request than a few a token.
//
// Request s brings counts[s] tokens behind first[s] earlier ones and owns pages[page_start[s] .. page_start[s + 1]).  Every block
// of the rows adds up all counts itself, 256 at a time (a step holds hundreds of requests at most), and looks its rows up in the
// running sums, so one launch does it: what bounds it is the launch and two dependent loads, not the few hundred KB written.
// The step's kernels read this metadata before they wait for the kernels before them.  So this one never lets the next start early, its
// threads end with a fence, and the beam search puts an ordinary launch between it and the step (visibility is promised behind a
// wait or a complete launch, not behind a fence).
#include "common.cuh"

namespace {

constexpr int THREADS = 256;

__global__ void __launch_bounds__(THREADS)
step_tables_kernel(const int* first, const int* counts, const int* pages,
                   const int* page_start, int requests, int page_size, int tokens, int row_blocks,
                   int* segment_start, int* segment_of_token, int* positions,
                   int* slots, int* contexts, int* tables, int table_stride, int width) {
  __shared__ int ends[THREADS], warp_sums[THREADS / 32];
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if ((int)blockIdx.x >= row_blocks) {       // block tables
    const long long entry = (long long)((int)blockIdx.x - row_blocks) * THREADS + tid;
    const int s = (int)(entry / width), i = (int)(entry - (long long)s * width);
    if (s >= requests) return;
    const int lo = page_start[s], hi = page_start[s + 1];
    tables[(size_t)s * table_stride + i] = i < hi - lo ? pages[lo + i] : -1;
    __threadfence();
    return;
  }
  const int row = (int)blockIdx.x * THREADS + tid;
  int before = 0, seg = -1, start = 0;
  for (int base = 0; base < requests; base += THREADS) {
    const int s = base + tid;
    const int mine = s < requests ? max(counts[s], 0) : 0;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    __syncthreads();                         // (the searches of the chunk before are over)
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    for (int w = 0; w < warp; ++w) sum += warp_sums[w];
    ends[tid] = before + sum;
    if (blockIdx.x == 0 && s < requests) {
      segment_start[s] = before + sum - mine;
      contexts[s] = first[s] + mine;
      if (s == requests - 1) segment_start[requests] = before + sum;
      __threadfence();
    }
    __syncthreads();
    const int last = ends[THREADS - 1];
    if (seg < 0 && row >= before && row < last) {        // the first request whose end lies behind the row
      int lo = 0, hi = THREADS - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] > row) hi = mid; else lo = mid + 1;
      }
      seg = base + lo;
      start = lo > 0 ? ends[lo - 1] : before;
    }
    before = last;
    if (blockIdx.x != 0 && before >= ((int)blockIdx.x + 1) * THREADS) break;      // the same in the whole block
  }
  if (row >= tokens) return;
  int position = 0, slot = -1;
  if (seg >= 0) {
    position = first[seg] + row - start;
    const int lo = page_start[seg], page = position / page_size;
    const int held = page < page_start[seg + 1] - lo && position >= 0 ? pages[lo + page] : -1;
    if (held >= 0) slot = held * page_size + position % page_size;
  }
  segment_of_token[row] = seg;
  positions[row] = position;
  slots[row] = slot;
  __threadfence();
}

}  // namespace

// segment_start int32 [requests + 1]; segment_of_token, positions, slots [tokens] (rows behind the last request: -1, 0, -1);
// contexts [requests]; tables [requests, width] (rows table_stride apart; -1 behind a request's last page).
extern "C" int lse_step_tables(const int* first, const int* counts, const int* pages, const int* page_start, int requests, int page_size,
                               int tokens, int* segment_start, int* segment_of_token, int* positions, int* slots, int* contexts,
                               int* tables, int table_stride, int width, cudaStream_t stream) {
  if (requests <= 0 || tokens < 0 || page_size < 1 || width < 0 || table_stride < width) return LSE_ERR_BAD_ARGUMENT;
  const int row_blocks = tokens > 0 ? (tokens + THREADS - 1) / THREADS : 1;
  const long long table_blocks = ((long long)requests * width + THREADS - 1) / THREADS;
  if (table_blocks + row_blocks > 0x7fffffffLL) return LSE_ERR_TOO_LARGE;
  const cudaError_t err = lse_launch(step_tables_kernel, dim3((unsigned)(row_blocks + table_blocks)), dim3(THREADS), 0, stream, first, counts,
                                     pages, page_start, requests, page_size, tokens, row_blocks, segment_start, segment_of_token,
                                     positions, slots, contexts, tables, table_stride, width > 0 ? width : 1);
  if (err != cudaSuccess) return (int)err;
  LSE_LAUNCH_CHECK();
}

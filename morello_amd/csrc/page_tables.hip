// Lengths of requests -> page tables, slots and positions of a step's new tokens, in one launch.
//
// With n new tokens and c cached ones of a request, starts = the running sum of n, and each request draws
//     max(0, ceil((c + n) / P) - ceil(c / P))
// pages, the first of them behind the running sum of what the requests before it drew.  Every workgroup forms both sums for
// itself (in 64 bits: the lengths are anything) over all requests, 1024 at a time: a second launch, or a wait between
// workgroups, costs more than reading some thousand lengths again.  A workgroup then owns 1024 tokens: the requests that
// have some among them leave a mark at their first, and the largest mark up to a token names its request.  Every page that is
// drawn begins with a new token (the cached ones end in a page before), so the token that opens a page writes its column
// of the table; slots on a page of an earlier step come from the table, whose columns below ceil(c / P) nobody writes.
// What bounds it: the launch, and the trips to memory behind each other (lengths, then pages): 16 requests' single tokens 4.8 us, 67 requests' 11 027 tokens and 171 new pages 6.0 us (with shuffles for the scans 5.3 and 6.4),
// of which an empty launch takes 2 to 3.
#include "paged.h"

namespace mrl {
namespace {

constexpr int THREADS = 256, EACH = 4;   // requests of a pass, and tokens of a workgroup, per thread
constexpr int PASS = THREADS * EACH, WAVES = THREADS / 64;

// x: the sum over the threads before this one; returns the sum over all.
__device__ inline uint64_t scan(uint64_t &x, uint64_t *wave_sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t sum = paged::sums_up_to(x);
  __syncthreads();   // (the sums of the scan before have been read)
  if (lane == 63) wave_sums[wave] = sum;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; w++) {
    if (w < wave) before += wave_sums[w];
    all += wave_sums[w];
  }
  x = before + sum - x;
  return all;
}

__global__ __launch_bounds__(THREADS) void k_page_tables(PageTablesArgs p, FastDiv by_page) {
  // At the place of a request's first token of this workgroup's:
  __shared__ int32_t mark[PASS];          // the place; -1 where no request begins
  __shared__ uint32_t request_of[PASS], start_of[PASS], cached_of[PASS];
  __shared__ uint64_t drawn_of[PASS];     // pages drawn by the requests before it
  __shared__ uint64_t wave_sums[WAVES];
  __shared__ int32_t wave_marks[WAVES];
  const uint32_t tid = threadIdx.x;
  const uint32_t t0 = blockIdx.x * PASS, t1 = min(p.tokens, t0 + PASS);
  const uint64_t free_count = uint64_t(min(max(int64_t(*p.free_count), int64_t(0)), int64_t(p.free_pages)));
  const uint32_t table_tokens = p.width * p.page_size;   // (below 2^31)
  // Columns of the table that n tokens take, of those that there are.
  auto columns = [&](uint64_t n) { return n >= table_tokens ? p.width : n ? by_page.div(uint32_t(n) - 1) + 1 : 0u; };
#pragma unroll
  for (int i = 0; i < EACH; i++) mark[tid + i * THREADS] = -1;
  uint64_t tokens_before = 0, drawn_before = 0;
  for (uint32_t r0 = 0; r0 < p.requests; r0 += PASS) {
    uint32_t cached[EACH], drawn[EACH];
    uint64_t added[EACH], at = 0, page_at = 0;
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const uint32_t r = r0 + tid * EACH + i;
      cached[i] = r < p.requests ? uint32_t(max(p.cached[r], 0)) : 0;
      added[i] = r < p.requests ? uint64_t(max(p.added[r], 0)) : 0;
      at += added[i];
    }
    const uint64_t all_tokens = scan(at, wave_sums);
    at += tokens_before;
    const uint64_t start = min(at, uint64_t(p.tokens));
#pragma unroll
    for (int i = 0; i < EACH; i++) {   // the new tokens that are within `tokens` rows
      const uint64_t from = min(at, uint64_t(p.tokens)), to = min(at + added[i], uint64_t(p.tokens));
      at += added[i];
      added[i] = to - from;
      drawn[i] = columns(cached[i] + added[i]) - columns(cached[i]);
      page_at += drawn[i];
    }
    const uint64_t all_drawn = scan(page_at, wave_sums);   // (its barrier: the marks are set to -1)
    page_at += drawn_before;
    at = start;
    const bool writes = r0 / PASS % gridDim.x == blockIdx.x;
#pragma unroll
    for (int i = 0; i < EACH; i++) {
      const uint32_t r = r0 + tid * EACH + i;
      const uint64_t end = at + added[i];
      if (writes && r < p.requests) {
        if (r == 0) p.starts[0] = 0;
        p.starts[r + 1] = int32_t(end);
        p.lengths[r] = int32_t(min(cached[i] + added[i], uint64_t(0x7fffffff)));
      }
      if (end > max(at, uint64_t(t0)) && at < t1) {
        const uint32_t place = uint32_t(max(at, uint64_t(t0))) - t0;
        mark[place] = int32_t(place);
        request_of[place] = r, start_of[place] = uint32_t(at), cached_of[place] = cached[i], drawn_of[place] = page_at;
      }
      at = end, page_at += drawn[i];
    }
    tokens_before += all_tokens, drawn_before += all_drawn;
  }
  if (blockIdx.x == 0 && tid == 0) {
    p.free_left[0] = int32_t(free_count - min(free_count, drawn_before));
    p.free_left[1] = int32_t(min(drawn_before - min(free_count, drawn_before), uint64_t(0x7fffffff)));
  }
  __syncthreads();
  // The last mark up to each token: of this thread's four, of the lanes before it, of the waves before.
  int32_t own[EACH], last = -1;
#pragma unroll
  for (int i = 0; i < EACH; i++) last = max(last, mark[tid * EACH + i]), own[i] = last;
  const int lane = tid & 63, wave = tid >> 6;
  last = paged::largest_up_to(last, -1);
  if (lane == 63) wave_marks[wave] = last;
  int32_t before = __shfl_up(last, 1);
  if (lane == 0) before = -1;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; w++)
    if (w < wave) before = max(before, wave_marks[w]);
#pragma unroll
  for (int i = 0; i < EACH; i++) {
    const uint32_t t = t0 + tid * EACH + i;
    if (t >= t1) break;
    const int32_t place = max(before, own[i]);
    int32_t slot = -1;
    uint32_t position = 0;
    if (place >= 0 && t < tokens_before) {
      const uint32_t cached = cached_of[place];
      position = cached + (t - start_of[place]);
      if (position < table_tokens) {
        const uint32_t column = by_page.div(position), have = columns(cached), offset = position - column * p.page_size;
        const uint64_t entry = uint64_t(request_of[place]) * p.width + column;
        int32_t page = -1;
        if (column >= have) {
          const uint64_t k = drawn_of[place] + (column - have);
          if (k < free_count) page = p.free_list[free_count - 1 - k];
          if (offset == 0) p.table[entry] = page;
        } else {
          page = p.table[entry];
        }
        if (page >= 0 && uint32_t(page) < p.pages) slot = int32_t(uint32_t(page) * p.page_size + offset);
      }
    }
    p.slots[t] = slot;
    p.positions[t] = int32_t(min(position, 0x7fffffffu));
  }
}

}  // namespace

hipError_t launch_page_tables(const PageTablesArgs &a, hipStream_t stream) {
  plan::work(plan::UNIT_STREAM, 0, 16.0 * a.requests + 8.0 * a.tokens + 8.0 * a.tokens / a.page_size);
  const uint32_t grid = (a.tokens + PASS - 1) / PASS;
  MRL_LAUNCH(k_page_tables, dim3(grid), dim3(THREADS), 0, stream, a, FastDiv(a.page_size));
  return plan::last_error();
}

}  // namespace mrl

// tq_paged_plan.hip -- pages, slots and positions of a serving step from the
// requests' lengths.
//
// Everything is a prefix sum over the requests: the pages that done requests
// give back, the tokens that the others bring, the pages that they need.  One
// workgroup of 16 waves takes 1,024 requests at a time (a DPP scan in each
// wave, the waves' totals through LDS) and carries the sums on, so the free
// list, which every sum goes by, is read and written in order and the step
// needs one launch.  The launch and three dependent reads (lengths, free
// count, pages) bound it: 64 decoding requests take 6.3 us.  The rows of a step
// of more than kApart tokens are a second launch's, a lane a token: 512 requests
// with 87,552 rows take 13.5 + 4.0 us, in one workgroup 36.  (Up to 4,096 rows
// the second launch costs more than it saves: 2,131 rows 12.6 us a call, 4,198
// rows 14.7.)
#include "tq_mfma.h"
#include "tq_paged.h"

namespace {

using namespace tqm;

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kMaxTokens = 1 << 24, kMaxWidth = 1 << 20;
constexpr int kApart = 4096;  // steps of more tokens: their rows by a launch of their own
// A request with at most this many new pages and tokens is written by its own
// lane, a larger one by a wave.
constexpr int kLaneItems = 2;

struct PlanArgs {
  const int *kv_lens, *new_lens;
  int *table, *free_pages;
  const int *free_count;
  long long *slots;
  int *positions, *starts, *appended, *kv_out, *free_out;
  int batch, width, capacity, shift, tokens;
  int apart;  // the tokens' rows are another launch's
};

// Exclusive prefix sum of v over the workgroup's threads, and their total.
__device__ __forceinline__ long long block_prefix(int v, int *s, int lane, int wave, long long &total) {
  const int incl = wave_incl_scan_i(v);
  __syncthreads();  // the totals of the scan before have been read
  if (lane == 63) s[wave] = incl;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; w++) {
    const int t = s[w];
    before += w < wave ? t : 0;
    all += t;
  }
  total = all;
  return before + incl - v;
}

// What a request of the current 1,024 has to write.
struct Item {
  int b, held, need, kv, n, start;
  long long top;  // stack index of its first new page, or of the first that it gives back
};

__device__ __forceinline__ void write_page(const PlanArgs &a, const Item &it, int j) {
  a.table[(long long)it.b * a.width + it.held + j] = a.free_pages[it.top - j];
}
// Token i of the request.  Its page comes from the table or the stack, not
// from the entry that this launch writes.
__device__ __forceinline__ void write_token(const PlanArgs &a, const Item &it, int i) {
  const int pos = it.kv + i, pi = pos >> a.shift;
  const int page = pi < it.held ? a.table[(long long)it.b * a.width + pi] : a.free_pages[it.top - (pi - it.held)];
  a.slots[it.start + i] = page < 0 ? -1 : ((long long)page << a.shift) + (pos & ((1 << a.shift) - 1));
  a.positions[it.start + i] = pos;
}
__device__ __forceinline__ void write_none(const PlanArgs &a, int t) {
  a.slots[t] = -1;
  a.positions[t] = -1;
}

__global__ __launch_bounds__(kThreads) void paged_plan_kernel(PlanArgs a) {
  __shared__ int s_sum[kWaves];
  __shared__ Item s_item[kThreads];
  __shared__ int s_items, s_used;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int page = 1 << a.shift;
  const long long room = (long long)a.width << a.shift;
  const int free0 = min(max(a.free_count[0], 0), a.capacity);
  auto kv_of = [&](int b) { return max(a.kv_lens[b], 0); };
  auto pages_of = [&](long long tokens) { return (int)min((tokens + page - 1) >> a.shift, (long long)a.width); };

  // ---- done requests put their pages on the stack, in order ----
  long long released = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
    const int b = b0 + tid;
    const bool done = b < a.batch && a.new_lens[b] < 0;
    const int back = done ? pages_of(kv_of(b)) : 0;
    if (!__syncthreads_or(back)) continue;
    if (tid == 0) s_items = 0;  // the barrier above: the round before has been read
    long long total;
    const long long at = free0 + released + block_prefix(back, s_sum, lane, wave, total);
    if (back) s_item[atomicAdd(&s_items, 1)] = Item{b, 0, back, 0, 0, 0, at};
    __syncthreads();
    // a wave a request, 256 pages' reads side by side
    const int items = s_items;
    for (int k = wave; k < items; k += kWaves) {
      const Item it = s_item[k];
      const int *row = a.table + (long long)it.b * a.width;
      for (int j0 = lane; j0 < it.need; j0 += 256) {
        int page[4];
#pragma unroll
        for (int u = 0; u < 4; u++) page[u] = j0 + 64 * u < it.need ? row[j0 + 64 * u] : 0;
#pragma unroll
        for (int u = 0; u < 4; u++) {
          const int j = j0 + 64 * u;
          if (j < it.need && it.top + j < a.capacity) a.free_pages[it.top + j] = page[u];
        }
      }
    }
    released += total;
  }
  const long long avail = min(free0 + released, (long long)a.capacity);
  if (tid == 0) s_used = 0;
  __syncthreads();  // the stack is whole before pages are taken from it

  // ---- the others take theirs ----
  long long start0 = 0, taken0 = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
    const int b = b0 + tid;
    const bool live = b < a.batch;
    const int kv = live ? kv_of(b) : 0, raw = live ? a.new_lens[b] : 0;
    const int n = min(max(raw, 0), kMaxTokens + 1);  // one more than any step holds: it does not fit
    long long total, all_need;
    const long long start = start0 + block_prefix(n, s_sum, lane, wave, total);
    start0 += total;
    if (tid == 0) s_items = 0;  // all have passed the scan's barriers, so the round before
    const bool has_room = (long long)kv + n <= room && start + n <= a.tokens;
    const int held = pages_of(kv);
    const int need = has_room ? pages_of((long long)kv + n) - held : 0;
    const long long taken = taken0 + block_prefix(need, s_sum, lane, wave, all_need);
    taken0 += all_need;
    const bool fits = has_room && (need == 0 || taken + need <= avail);
    // the requests that fit and need pages are the first that need any, so what
    // is taken ends with the last of them
    if (fits && need > 0) atomicMax(&s_used, (int)(taken + need));
    if (live) {
      a.starts[b] = (int)min(start, 0x7fffffffll);
      a.appended[b] = fits ? n : 0;
      a.kv_out[b] = raw < 0 ? 0 : (fits ? kv + n : kv);
      const Item it{b, held, fits ? need : 0, kv, fits ? n : 0, (int)min(start, 0x7fffffffll), avail - 1 - taken};
      const int rows = a.apart ? 0 : n;
      if (fits && rows <= kLaneItems && it.need <= kLaneItems) {
        for (int j = 0; j < it.need; j++) write_page(a, it, j);
        for (int i = 0; i < rows; i++) write_token(a, it, i);
      } else if (fits || (rows > 0 && start < a.tokens)) {
        s_item[atomicAdd(&s_items, 1)] = fits ? it : Item{b, -1, 0, 0, (int)min((long long)n, a.tokens - start), (int)start, 0};
      }
    }
    __syncthreads();
    const int items = s_items;
    for (int k = wave; k < items; k += 4 * kWaves) {
      // four requests' first pages, their reads side by side
      int page[4];
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int ku = k + u * kWaves;
        page[u] = ku < items && lane < s_item[ku].need ? a.free_pages[s_item[ku].top - lane] : 0;
      }
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int ku = k + u * kWaves;
        if (ku >= items) break;
        const Item it = s_item[ku];
        if (it.held < 0) {  // it does not fit: its rows hold no tokens
          for (int i = lane; i < it.n; i += 64) write_none(a, it.start + i);
          continue;
        }
        if (lane < it.need) a.table[(long long)it.b * a.width + it.held + lane] = page[u];
        for (int j = 64 + lane; j < it.need; j += 64) write_page(a, it, j);
        if (a.apart) continue;
        for (int i = lane; i < it.n; i += 64) write_token(a, it, i);
      }
    }
  }
  __syncthreads();
  if (tid == 0) {
    a.starts[a.batch] = (int)min(start0, 0x7fffffffll);
    a.free_out[0] = (int)(avail - s_used);
  }
  if (a.apart) return;
  for (long long t = start0 + tid; t < a.tokens; t += kThreads) write_none(a, (int)t);
}

// The rows of a step of many tokens, a lane a token: its request is the last
// that starts at or before it (every kth start in LDS, then at most k more).
constexpr int kStarts = 2048;
__global__ __launch_bounds__(256) void paged_tokens_kernel(PlanArgs a, int k) {
  __shared__ int s_start[kStarts];
  const int n = (a.batch + k - 1) / k;  // <= kStarts
  for (int i = threadIdx.x; i < n; i += 256) s_start[i] = a.starts[i * k];
  __syncthreads();
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= a.tokens) return;
  if (t >= a.starts[a.batch]) return write_none(a, t);
  int lo = 0, hi = n;  // s_start[lo] <= t < s_start[hi]
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (s_start[m] <= t) lo = m;
    else hi = m;
  }
  lo *= k;
  hi = min(lo + k, a.batch);
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (a.starts[m] <= t) lo = m;
    else hi = m;
  }
  const int got = a.appended[lo];
  if (got == 0) return write_none(a, t);
  const int pos = a.kv_out[lo] - got + (t - a.starts[lo]);
  const int page = a.table[(long long)lo * a.width + (pos >> a.shift)];
  a.slots[t] = page < 0 ? -1 : ((long long)page << a.shift) + (pos & ((1 << a.shift) - 1));
  a.positions[t] = pos;
}

}  // namespace

extern "C" int tq_paged_plan(const int *kv_lens, const int *new_lens, int batch, int *block_table, int table_width,
                             int *free_pages, int free_capacity, const int *free_count, int page_size, int num_tokens,
                             long long *slots, int *positions, int *starts, int *appended, int *kv_lens_out,
                             int *free_count_out, hipStream_t stream) {
  const int shift = tqh::page_shift(page_size);
  if (shift < 0)
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "page_size %d is no power of two from 16 to 1024", page_size);
  if (batch < 0 || batch > 65535) return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "batch %d outside 0 to 65,535", batch);
  if (num_tokens < 0 || num_tokens > kMaxTokens)
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "num_tokens %d outside 0 to 2^24", num_tokens);
  if (table_width < 0 || table_width > kMaxWidth || (long long)table_width << shift > 0x7fffffffll)
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "table_width %d: at most 2^20 pages and 2^31 - 1 tokens a request",
                     table_width);
  if (free_capacity < 0) return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "negative free_capacity");
  if (!starts || !free_count || !free_count_out || (free_capacity && !free_pages) ||
      (batch && (!kv_lens || !new_lens || !appended || !kv_lens_out || (table_width && !block_table))) ||
      (num_tokens && (!slots || !positions)))
    return tqh::fail(TQ_ERR_INVALID_ARGUMENT, "null pointer");
  PlanArgs a{kv_lens, new_lens, block_table, free_pages, free_count, slots, positions, starts, appended, kv_lens_out,
             free_count_out, batch, table_width, free_capacity, shift, num_tokens, batch && num_tokens > kApart};
  hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kThreads), 0, stream, a);
  if (a.apart)
    hipLaunchKernelGGL(paged_tokens_kernel, dim3((unsigned)((num_tokens + 255) / 256)), dim3(256), 0, stream, a,
                       (batch + kStarts - 1) / kStarts);
  return tqh::check_launch("paged_plan_kernel");
}

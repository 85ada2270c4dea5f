// Page tables, slots and positions of a step from the requests' lengths (kq_plan_pages), without a look at the lengths on the host.
//
// Request r holds ceil(seen_r / page) pages and takes as many more as seen_r + new_r tokens need (never more than its table row
// holds), from a list of free pages: first_r = taken + sum of what the requests before it take.  Token i of request r stands at
// position seen_r + i, in slot table[r][position / page] * page + position % page.
//
// Bound by latency (a few KB in, 12 bytes per token out): one launch, in which every CTA scans all requests' lengths itself
// (1024 at a time, a thread each) and writes the tokens of its own range.  A fresh page is entered into the table by the
// thread of its first token, which is always a new one; tokens take a fresh page's name from the free list, so that no CTA waits
// for another one's table entries.  64 requests of a decode step take 3.3 us, 500 prompts with 262 500 tokens 5.9 (with one CTA per multiprocessor and
// two tokens per thread 7.3).
#include "kq_common.cuh"

namespace kq {

namespace {

constexpr int PG_THREADS = 1024;
constexpr int PG_TOKENS = 1024;          // tokens of a CTA's range at least

struct PageParams {
  int32_t* table; int64_t table_r; int width;
  const int32_t* seen; const int32_t* fresh; int requests;
  const int32_t* free_pages; int num_free;
  const int32_t* taken;
  int page_size;
  int num_tokens;
  int32_t* total; int32_t* starts; int32_t* positions; int64_t* slots; int32_t* taken_out;
};

__device__ __forceinline__ int to_int(int64_t v) { return (int)min(v, (int64_t)0x7fffffff); }

__device__ __forceinline__ uint32_t pages_of(uint32_t tokens, int page_size) { return tokens / page_size + (tokens % page_size != 0); }

__global__ void __launch_bounds__(PG_THREADS) plan_pages_kernel(const PageParams p, int range) {
  __shared__ int s_start[PG_THREADS + 1];
  __shared__ int2 s_seen[PG_THREADS];                                 // tokens, pages
  __shared__ int64_t s_first[PG_THREADS];
  __shared__ int64_t s_warp[2][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_trigger();
  pdl_wait();
  const int t0 = (int)min((int64_t)blockIdx.x * range, (int64_t)p.num_tokens);
  const int t1 = (int)min((int64_t)t0 + range, (int64_t)p.num_tokens);
  int64_t run_new = 0, run_need = p.taken[0];
  for (int r0 = 0; r0 < p.requests; r0 += PG_THREADS) {
    const int r = r0 + tid;
    int seen = 0, fresh = 0;
    if (r < p.requests) { seen = max(p.seen[r], 0); fresh = max(p.fresh[r], 0); }
    const uint32_t total = (uint32_t)seen + fresh;                    // below 2^32, as every position; divisions in 32 bits
    const int held = pages_of(seen, p.page_size);
    const int64_t need = max((int64_t)0, (int64_t)min(pages_of(total, p.page_size), (uint32_t)p.width) - held);
    int64_t a = fresh, n = need;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t ua = __shfl_up_sync(0xffffffffu, a, d), un = __shfl_up_sync(0xffffffffu, n, d);
      if (lane >= d) { a += ua; n += un; }
    }
    if (lane == 31) { s_warp[0][warp] = a; s_warp[1][warp] = n; }
    __syncthreads();
    if (warp < 2) {
      int64_t v = s_warp[warp][lane];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += u;
      }
      s_warp[warp][lane] = v;
    }
    __syncthreads();
    if (warp > 0) { a += s_warp[0][warp - 1]; n += s_warp[1][warp - 1]; }
    s_start[tid] = to_int(run_new + a - fresh);
    s_seen[tid] = make_int2(seen, held);
    s_first[tid] = run_need + n - need;
    if (tid == PG_THREADS - 1) s_start[PG_THREADS] = to_int(run_new + a);
    if (blockIdx.x == 0 && r < p.requests) {
      p.total[r] = to_int(total);
      p.starts[r] = to_int(run_new + a - fresh);
    }
    run_new += s_warp[0][31];
    run_need += s_warp[1][31];
    __syncthreads();
    // tokens of this CTA's range that belong to these requests
    const int lo = max(t0, s_start[0]), hi = min(t1, s_start[PG_THREADS]);
    for (int t = lo + tid; t < hi; t += PG_THREADS) {
      int a0 = 0, a1 = min(PG_THREADS, p.requests - r0);       // the last request with start <= t: s_start[a0] <= t < s_start[a1]
      while (a1 - a0 > 1) {
        const int mid = (a0 + a1) >> 1;
        if (s_start[mid] <= t) a0 = mid; else a1 = mid;
      }
      const int2 held_by = s_seen[a0];
      const uint32_t pos = (uint32_t)held_by.x + (t - s_start[a0]), at = pos / p.page_size;
      const int have = held_by.y, place = (int)(pos - at * p.page_size);
      int name = -1;
      if (at < (uint32_t)p.width) {
        int32_t* entry = p.table + (int64_t)(r0 + a0) * p.table_r + at;
        if ((int)at < have) {
          name = *entry;
        } else {
          const int64_t from = s_first[a0] + ((int)at - have);
          if (from >= 0 && from < p.num_free) name = p.free_pages[from];
          if (place == 0) *entry = name;
        }
      }
      p.positions[t] = to_int(pos);
      p.slots[t] = name >= 0 ? (int64_t)name * p.page_size + place : -1;
    }
    __syncthreads();
  }
  if (blockIdx.x == 0 && tid == 0) {
    p.starts[p.requests] = to_int(run_new);
    p.taken_out[0] = to_int(run_need);
  }
  for (int t = max(t0, to_int(run_new)) + tid; t < t1; t += PG_THREADS) {   // padding
    p.positions[t] = 0;
    p.slots[t] = -1;
  }
}

}  // namespace

}  // namespace kq

using namespace kq;

extern "C" int kq_plan_pages(int32_t* block_table, int64_t table_stride, int64_t table_width, const int32_t* seq_lens,
                             const int32_t* new_lens, int64_t requests, const int32_t* free_pages, int64_t num_free,
                             const int32_t* taken, int64_t page_size, int64_t num_tokens, int32_t* total_lens, int32_t* starts,
                             int32_t* positions, int64_t* slots, int32_t* taken_out, void* stream) {
  const char* fn = "kq_plan_pages";
  clear_error();
  if (requests < 0 || table_width < 0 || num_free < 0 || num_tokens < 0 || page_size <= 0) { set_error("%s: page_size must be positive, the other sizes not negative", fn); return KQ_EINVAL; }
  if (requests > (1 << 20) || table_width > 0x7fffffff || num_free > 0x7fffffff || num_tokens > 0x7fffffff || page_size > 0x7fffffff) { set_error("%s: size out of range", fn); return KQ_ELIMIT; }
  if (requests > 1 && table_stride < table_width) { set_error("%s: rows of the table overlap", fn); return KQ_EINVAL; }
  if (!taken || !starts || !taken_out || (requests && (!seq_lens || !new_lens || !total_lens)) || (requests && table_width && !block_table) ||
      (num_free && !free_pages) || (num_tokens && (!positions || !slots))) {
    set_error("%s: null pointer", fn);
    return KQ_EINVAL;
  }
  if (((uintptr_t)block_table | (uintptr_t)seq_lens | (uintptr_t)new_lens | (uintptr_t)free_pages | (uintptr_t)taken | (uintptr_t)total_lens | (uintptr_t)starts |
       (uintptr_t)positions | (uintptr_t)taken_out) % 4 || (uintptr_t)slots % 8) {
    set_error("%s: misaligned pointer", fn);
    return KQ_EINVAL;
  }
  // other CTAs may still read what the first one would overwrite
  const void* outs[] = {total_lens, starts, positions, slots, taken_out};
  const void* ins[] = {block_table, seq_lens, new_lens, free_pages, taken};
  for (int i = 0; i < 5; ++i)
    for (int j = 0; j < 5; ++j)
      if (outs[i] && (outs[i] == ins[j] || (j < i && outs[i] == outs[j]))) { set_error("%s: outputs must be neither inputs nor each other", fn); return KQ_EINVAL; }
  if (block_table && (block_table == seq_lens || block_table == new_lens || block_table == free_pages || block_table == taken)) {
    set_error("%s: block_table is written, and must not be another input", fn);
    return KQ_EINVAL;
  }
  PageParams p;
  p.table = block_table; p.table_r = table_stride; p.width = (int)table_width; p.seen = seq_lens; p.fresh = new_lens;
  p.requests = (int)requests; p.free_pages = free_pages; p.num_free = (int)num_free; p.taken = taken; p.page_size = (int)page_size;
  p.num_tokens = (int)num_tokens; p.total = total_lens; p.starts = starts; p.positions = positions; p.slots = slots; p.taken_out = taken_out;
  const int64_t most = 2 * sm_count();     // two CTAs fit
  int64_t ctas = (num_tokens + PG_TOKENS - 1) / PG_TOKENS;
  ctas = ctas < 1 ? 1 : ctas > most ? most : ctas;
  const int64_t range = (num_tokens + ctas - 1) / ctas;
  KQ_CUDA_TRY(launch_pdl(plan_pages_kernel, dim3((unsigned)ctas), dim3(PG_THREADS), (size_t)0, (cudaStream_t)stream, options().pdl != 0, p, (int)range));
  options().launches += 1;
  return KQ_OK;
}

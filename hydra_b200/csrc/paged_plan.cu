// Block tables, slots and positions of a step from the requests' lengths, built on the device in one launch.
//
//   held_b = ceil(context_b / P), want_b = ceil((context_b + new_b) / P); the pages of all requests that want more are dealt
//   out of the free list in request order: table[b][j] = free[start + sum_{a<b}(want_a - held_a) + j - held_b].
//   Token i of request b (new tokens are packed request after request): position context_b + i, slot = page * P + offset.
//
// Bound: launch latency (a decode step moves a few KB; a 64k-token prefill 0.8 MB).  So there is one launch and no
// workspace: every CTA scans all lengths itself (two prefix sums over at most 4096 requests) and writes its part of the
// tokens and of the new table entries.  A token's page comes from the table where the request held it before and
// straight from the free list where it is new, so no CTA reads what another one writes.  64 requests with a new token
// each: 6.0 us of device time, 250 with 64000 between them: 5.6, launch and two dependent reads.
#include "common.cuh"

namespace hb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxBatch = 4096;
constexpr int kTokens = 4;       // consecutive tokens per thread: one search, 16-byte stores

struct PlanParams {
  const int32_t *context, *fresh, *free_pages, *free_start;
  int32_t *table, *kv_lens, *cu, *positions, *start_out, *status;
  int64_t* slots;
  int64_t table_ld, n_free;
  int B, width, page_size, room;
};

__device__ __forceinline__ int sat32(int64_t v) { return v > 0x7fffffff ? 0x7fffffff : (int)v; }

// Inclusive-to-exclusive scan of two 64-bit sums over the CTA (thread order).
__device__ __forceinline__ void scan2(int64_t& a, int64_t& b, int64_t& ta, int64_t& tb, int64_t (*buf)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t ia = a, ib = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t xa = __shfl_up_sync(0xffffffffu, ia, o), xb = __shfl_up_sync(0xffffffffu, ib, o);
    if (lane >= o) { ia += xa; ib += xb; }
  }
  if (lane == 31) { buf[warp][0] = ia; buf[warp][1] = ib; }
  __syncthreads();
  int64_t oa = 0, ob = 0;
  ta = tb = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w == warp) { oa = ta; ob = tb; }
    ta += buf[w][0];
    tb += buf[w][1];
  }
  a = oa + ia - a;
  b = ob + ib - b;
}

__global__ void __launch_bounds__(kThreads) paged_plan_kernel(const PlanParams p) {
  __shared__ int32_t s_cu[kMaxBatch + 1];      // new tokens before each request
  __shared__ int32_t s_first[kMaxBatch];       // pages dealt out before each request
  __shared__ int64_t s_buf[kThreads / 32][2];
  __shared__ int s_flags;
  const int tid = threadIdx.x;
  const bool writer = blockIdx.x == 0;
  if (tid == 0) s_flags = 0;
  const int64_t start = p.free_start ? (int64_t)*p.free_start : 0;

  struct Lengths { int64_t context, total; int held, want; int flags; };
  auto lengths = [&](int b) {
    Lengths r;
    int64_t c = p.context[b], n = p.fresh[b];
    r.flags = (c < 0 || n < 0) ? HB200_PLAN_BAD_LENGTH : 0;
    c = c < 0 ? 0 : c;
    n = n < 0 ? 0 : n;
    if (c + n > 0x7fffffff) { n = 0x7fffffff - c; r.flags = HB200_PLAN_BAD_LENGTH; }
    r.context = c;
    r.total = c + n;
    const int64_t held = (c + p.page_size - 1) / p.page_size, want = (r.total + p.page_size - 1) / p.page_size;
    if (want > p.width) r.flags |= HB200_PLAN_TABLE_FULL;
    r.held = (int)(held < p.width ? held : p.width);
    r.want = (int)(want < p.width ? want : p.width);
    return r;
  };

  const int per = (p.B + kThreads - 1) / kThreads, b0 = tid * per;
  int64_t tokens = 0, pages = 0;
  int flags = 0;
  for (int i = 0; i < per && b0 + i < p.B; ++i) {
    const Lengths r = lengths(b0 + i);
    tokens += r.total - r.context;
    pages += r.want - r.held;
    flags |= r.flags;
  }
  int64_t all_tokens, all_pages;
  scan2(tokens, pages, all_tokens, all_pages, s_buf);   // its barrier also orders s_flags = 0
  if (flags) atomicOr(&s_flags, flags);
  for (int i = 0; i < per && b0 + i < p.B; ++i) {
    const Lengths r = lengths(b0 + i);
    s_cu[b0 + i] = sat32(tokens);
    s_first[b0 + i] = sat32(pages);
    if (writer) {
      p.kv_lens[b0 + i] = (int32_t)r.total;
      p.cu[b0 + i] = sat32(tokens);
    }
    tokens += r.total - r.context;
    pages += r.want - r.held;
  }
  if (tid == 0) s_cu[p.B] = sat32(all_tokens);
  __syncthreads();
  if (writer && tid == 0) {
    p.cu[p.B] = sat32(all_tokens);
    const bool out = all_pages > 0 && (start < 0 || start + all_pages > p.n_free);
    p.start_out[0] = (int32_t)(out ? (start > p.n_free ? start : p.n_free) : start + all_pages);
    p.status[0] = s_flags | (out ? HB200_PLAN_OUT_OF_PAGES : 0) | (all_tokens > p.room ? HB200_PLAN_OUT_OF_ROOM : 0);
  }

  auto dealt = [&](int64_t i) {   // the i-th page that this call deals out
    const int64_t at = start + i;
    return at >= 0 && at < p.n_free ? p.free_pages[at] : -1;
  };
  // new table entries: a warp per request
  const int lane = tid & 31, nwarps = gridDim.x * (kThreads / 32);
  for (int b = blockIdx.x * (kThreads / 32) + (tid >> 5); b < p.B; b += nwarps) {
    const Lengths r = lengths(b);
    for (int j = r.held + lane; j < r.want; j += 32) p.table[(int64_t)b * p.table_ld + j] = dealt((int64_t)s_first[b] + j - r.held);
  }
  // tokens
  for (int64_t i0 = ((int64_t)blockIdx.x * kThreads + tid) * kTokens; i0 < p.room; i0 += (int64_t)gridDim.x * kThreads * kTokens) {
    int32_t pos[kTokens];
    int64_t slot[kTokens];
    int b = -1, next = 0, page_of = -1, page = -1;
    Lengths r = {};
    if (i0 < s_cu[p.B]) {
      int lo = 0, hi = p.B;         // s_cu[lo] <= i0 < s_cu[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cu[mid] <= i0) lo = mid; else hi = mid;
      }
      b = lo;
      next = s_cu[b + 1];
      r = lengths(b);
    }
#pragma unroll
    for (int k = 0; k < kTokens; ++k) {
      const int64_t i = i0 + k;
      pos[k] = -1;
      slot[k] = -1;
      if (i < s_cu[p.B] && i < p.room) {
        if (i >= next) {
          do { ++b; } while (s_cu[b + 1] <= i);
          next = s_cu[b + 1];
          r = lengths(b);
          page_of = -1;
        }
        pos[k] = (int32_t)(r.context + (i - s_cu[b]));
        const int j = pos[k] / p.page_size;
        if (j != page_of) {
          page_of = j;
          page = j >= p.width ? -1 : (j < r.held ? p.table[(int64_t)b * p.table_ld + j] : dealt((int64_t)s_first[b] + j - r.held));
        }
        if (page >= 0) slot[k] = (int64_t)page * p.page_size + (pos[k] - j * p.page_size);
      }
    }
    if (i0 + kTokens <= p.room) {   // 16-byte stores: the arrays are 16-byte aligned and i0 is a multiple of 4
      *reinterpret_cast<int4*>(p.positions + i0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<longlong2*>(p.slots + i0) = make_longlong2(slot[0], slot[1]);
      *reinterpret_cast<longlong2*>(p.slots + i0 + 2) = make_longlong2(slot[2], slot[3]);
    } else {
#pragma unroll
      for (int k = 0; k < kTokens; ++k)
        if (i0 + k < p.room) { p.positions[i0 + k] = pos[k]; p.slots[i0 + k] = slot[k]; }
    }
  }
}

}  // namespace
}  // namespace hb200

using namespace hb200;

extern "C" int hb200_paged_plan(const int32_t* context_lens, const int32_t* new_lens, int B, int32_t* block_tables,
                                int64_t table_ld, int table_width, int page_size, const int32_t* free_pages, int64_t n_free,
                                const int32_t* free_start, int32_t* kv_lens, int32_t* cu_new, int32_t* positions,
                                int64_t* slots, int max_new, int32_t* free_start_out, int32_t* status, void* stream) {
  HB_REQUIRE(B >= 0 && table_width >= 0 && table_ld >= table_width && page_size >= 1 && n_free >= 0 && max_new >= 0,
             HB200_ERR_INVALID, "paged_plan: bad shape B=%d width=%d page_size=%d n_free=%lld max_new=%d", B, table_width,
             page_size, (long long)n_free, max_new);
  HB_REQUIRE(B <= kMaxBatch, HB200_ERR_UNSUPPORTED, "paged_plan: %d requests (up to %d in one call)", B, kMaxBatch);
  HB_REQUIRE(n_free <= 0x7fffffff, HB200_ERR_UNSUPPORTED, "paged_plan: a free list of %lld pages", (long long)n_free);
  HB_REQUIRE(cu_new && free_start_out && status && (B == 0 || (context_lens && new_lens && kv_lens)) &&
                 (B == 0 || table_width == 0 || block_tables) && (n_free == 0 || free_pages) && (max_new == 0 || (positions && slots)),
             HB200_ERR_INVALID, "paged_plan: null pointer");
  HB_REQUIRE(aligned16(positions) && aligned16(slots), HB200_ERR_INVALID, "paged_plan: positions and slots must be 16-byte aligned");
  // Every CTA reads all lengths while others store.
  const int64_t each = (int64_t)B * 4;
  const Reach read[] = {reach_of(context_lens, each), reach_of(new_lens, each), reach_of(free_pages, n_free * 4), reach_of(free_start, free_start ? 4 : 0)};
  const Reach written[] = {reach_of(block_tables, (int64_t)table_width * 4, {{B, table_ld * 4}}), reach_of(kv_lens, each), reach_of(cu_new, each + 4),
                           reach_of(positions, (int64_t)max_new * 4), reach_of(slots, (int64_t)max_new * 8), reach_of(free_start_out, 4), reach_of(status, 4)};
  for (const Reach& w : written) {
    for (const Reach& r : read)
      HB_REQUIRE(!overlap(w, r), HB200_ERR_INVALID, "paged_plan: block_tables and the results must not overlap the lengths or the free list");
    for (const Reach* other = written; other != &w; ++other)
      HB_REQUIRE(!overlap(w, *other), HB200_ERR_INVALID, "paged_plan: block_tables and the results must not overlap one another");
  }
  PlanParams p = {};
  p.context = context_lens; p.fresh = new_lens; p.free_pages = free_pages; p.free_start = free_start;
  p.table = block_tables; p.kv_lens = kv_lens; p.cu = cu_new; p.positions = positions; p.start_out = free_start_out;
  p.status = status; p.slots = slots; p.table_ld = table_ld; p.n_free = n_free;
  p.B = B; p.width = table_width; p.page_size = page_size; p.room = max_new;
  const int64_t by_tokens = ceil_div64(max_new, kThreads * kTokens), by_rows = ceil_div64(B, kThreads / 32);
  int64_t grid = by_tokens > by_rows ? by_tokens : by_rows;
  grid = grid < 1 ? 1 : (grid > 256 ? 256 : grid);
  paged_plan_kernel<<<(unsigned)grid, kThreads, 0, (cudaStream_t)stream>>>(p);
  HB_LAUNCH_CHECK();
  return 0;
}

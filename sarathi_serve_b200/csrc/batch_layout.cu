// Block tables and index arrays of a serving step, made on the GPU from the lengths of its requests, so that a step
// that is replayed from a CUDA graph needs nothing from the host but those lengths.
//
// Counterpart in the reference: the block manager's lists and the host loops of the attention wrapper's begin_forward
// (sarathi/core/block_space_manager, sarathi/model_executor/attention/flashinfer_attention_wrapper.py), which walk the
// sequences in Python every step.
//
// Both kernels are bound by latency (their floor is well below a microsecond for a step of a few hundred requests; the layout
// of 212 requests with 1997 tokens takes 5.6 us), so each is ONE launch: every CTA computes the prefix sums over the requests for
// itself, into shared memory, and the items (pages, tokens) are then dealt out flat -- an item finds its request by binary search --
// so that one request with thousands of pages takes no longer than thousands of requests with one.
#include "common.cuh"
#include "sm100_ptx.cuh"

namespace sb200 {

constexpr int kMaxRequests = SB200_MAX_REQUESTS;
constexpr int kLayoutThreads = 512;

// Exclusive prefix sum over the CTA of one value per thread; *total = their sum.  `red` needs 33 words.
__device__ __forceinline__ long long block_exclusive_scan(long long v, long long* red, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the last use of `red` is over
  if (lane == 31) red[warp] = x;
  __syncthreads();
  if (warp == 0) {
    long long s = lane < warps ? red[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    red[lane] = s;
  }
  __syncthreads();
  *total = red[warps - 1];
  return x - v + (warp ? red[warp - 1] : 0);
}

// The request that item e belongs to: p[r] <= e < p[r + 1] (p: exclusive prefix sums, p[n] = their total > e).
__device__ __forceinline__ int owner_of(const int* p, int n, int e) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p[mid] <= e) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

struct TablesArgs {
  int32_t* tables; int64_t ld;
  int32_t* num_blocks;
  const int32_t* seq_lens;
  int32_t* free_blocks;
  int32_t* num_free;
  int32_t* granted;
  int n, width, capacity, page_size;
};

// Pages a request must have; more than the table holds: width + 1.
__device__ __forceinline__ int pages_wanted(int len, int page, int width) {
  const int w = len / page + (len % page != 0);
  return w > width ? width + 1 : w;
}

// One CTA, or a cluster of them when many pages may move.  Given-back pages are pushed in request order and grants pop in
// request order; a grant that reaches into the pages just pushed reads them from the table they come from, so that the two
// halves need no barrier between them -- only the counters, which every CTA reads, are written behind one.  A page is a search
// in shared memory, a load and a store after one another, about 1.3 us: a thread has four of them under way.
// 128 requests of which a few start a page: 4.3 us; 512 requests with 74000 pages to move: 15 us (one page at a time: 24.6; a cluster of
// four: 25).
constexpr int kTablesThreads = 1024;

__global__ void __launch_bounds__(kTablesThreads)
resize_tables_kernel(const TablesArgs a) {
  grid_dependency_begin();
  extern __shared__ int smem_i[];
  __shared__ long long red[33];
  int* give = smem_i;              // exclusive prefix sums of the pages given back, and of the pages asked for
  int* take = smem_i + a.n + 1;
  int* owned = smem_i + 2 * (a.n + 1);   // pages that every request has, and wants
  int* wanted = owned + a.n;
  const int per = (a.n + kTablesThreads - 1) / kTablesThreads, r0 = min(a.n, (int)threadIdx.x * per), r1 = min(a.n, r0 + per);
  const int ctas = gridDim.x, cta = blockIdx.x;

  auto both = [&](int r, int* have, int* want) {  // (a negative length: the request is left alone)
    *have = clampi(a.num_blocks[r], 0, a.width);
    const int len = a.seq_lens[r];
    *want = len < 0 ? *have : pages_wanted(len, a.page_size, a.width);
  };
  long long g = 0, t = 0;
  for (int r = r0; r < r1; ++r) {
    int have, want;
    both(r, &have, &want);
    owned[r] = have;
    wanted[r] = want;
    if (want < have) g += have - want;
    else if (want <= a.width) t += want - have;
  }
  long long all_give, all_take;
  long long gp = block_exclusive_scan(g, red, &all_give);
  long long tp = block_exclusive_scan(t, red, &all_take);
  const int n0 = clampi(*a.num_free, 0, a.capacity);
  for (int r = r0; r < r1; ++r) {
    const int have = owned[r], want = wanted[r];
    give[r] = (int)gp;
    take[r] = (int)tp;
    if (want < have) gp += have - want;
    else if (want <= a.width) tp += want - have;
  }
  if (threadIdx.x == 0) { give[a.n] = (int)all_give; take[a.n] = (int)all_take; }
  __syncthreads();
  // what fits: requests up to the first whose share would pass the end of the stack (never, if the pool is consistent) ...
  const int room = a.capacity - n0;
  const int given = all_give <= room ? (int)all_give : give[owner_of(give, a.n, room)];
  const int avail = n0 + given;
  // ... or the pages there are
  const int taken = all_take <= avail ? (int)all_take : take[owner_of(take, a.n, avail)];

  auto given_page = [&](int e) {
    const int r = owner_of(give, a.n, e);
    return a.tables[r * a.ld + wanted[r] + (e - give[r])];
  };
  const int first = cta * kTablesThreads + threadIdx.x, step = ctas * kTablesThreads;
  constexpr int kAhead = 4;
  for (int e0 = first; e0 < given; e0 += kAhead * step) {
    int page[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (e0 + i * step < given) page[i] = given_page(e0 + i * step);
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (e0 + i * step < given) a.free_blocks[n0 + e0 + i * step] = page[i];
  }
  for (int e0 = first; e0 < taken; e0 += kAhead * step) {
    int page[kAhead];
    int32_t* to[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int e = e0 + i * step, at = avail - 1 - e;
      if (e >= taken) continue;
      const int r = owner_of(take, a.n, e);
      page[i] = at >= n0 ? given_page(at - n0) : a.free_blocks[at];
      to[i] = a.tables + (r * a.ld + owned[r] + (e - take[r]));
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (e0 + i * step < taken) *to[i] = page[i];
  }
  if (ctas > 1) ptx::cluster_sync_all();
  else __syncthreads();
  if (cta == 0) {
    for (int r = threadIdx.x; r < a.n; r += kTablesThreads) {
      const int have = owned[r], want = wanted[r];
      const bool ok = want < have ? give[r + 1] <= given : want == have || (want <= a.width && take[r + 1] <= taken);
      a.granted[r] = ok ? 1 : 0;
      a.num_blocks[r] = ok ? want : have;
    }
    if (threadIdx.x == 0) *a.num_free = avail - taken;
  }
}

struct LayoutArgs {
  const int32_t *query_lens, *context_lens, *tables; int64_t ld;
  int32_t *qo_indptr, *kv_lens, *kv_indptr, *kv_indices, *last_page_len, *batch_indices;
  int64_t *positions, *kv_slots;
  int n, width, page_size, num_pages, num_tokens;
  int64_t capacity;  // entries of kv_indices
};

__global__ void __launch_bounds__(kLayoutThreads)
batch_layout_kernel(const LayoutArgs a) {
  grid_dependency_begin();
  extern __shared__ int smem_i[];
  __shared__ long long red[33];
  int* rows = smem_i;              // first row of every request, and first entry of its page list
  int* pages = smem_i + a.n + 1;
  const int per = (a.n + kLayoutThreads - 1) / kLayoutThreads, r0 = min(a.n, (int)threadIdx.x * per), r1 = min(a.n, r0 + per);
  const int most = (int)min((long long)a.width * a.page_size, (long long)INT32_MAX);  // tokens that a block table has room for
  auto context = [&](int r) { return clampi(a.context_lens[r], 0, most); };
  auto query = [&](int r) { return clampi(a.query_lens[r], 0, most - context(r)); };

  long long s = 0, total;
  for (int r = r0; r < r1; ++r) s += query(r);
  long long p = block_exclusive_scan(s, red, &total);
  for (int r = r0; r < r1; ++r) {
    rows[r] = (int)min(p, (long long)a.num_tokens);
    p += query(r);
  }
  if (threadIdx.x == 0) rows[a.n] = (int)min(total, (long long)a.num_tokens);
  __syncthreads();
  auto length = [&](int r) { return context(r) + rows[r + 1] - rows[r]; };
  auto pages_of = [&](int len) { return len / a.page_size + (len % a.page_size != 0); };
  s = 0;
  for (int r = r0; r < r1; ++r) s += pages_of(length(r));
  p = block_exclusive_scan(s, red, &total);
  for (int r = r0; r < r1; ++r) {
    pages[r] = (int)p;
    p += pages_of(length(r));
  }
  if (threadIdx.x == 0) pages[a.n] = (int)total;
  __syncthreads();

  const int first = blockIdx.x * kLayoutThreads + threadIdx.x, step = gridDim.x * kLayoutThreads;
  for (int r = first; r <= a.n; r += step) {
    a.qo_indptr[r] = rows[r];
    a.kv_indptr[r] = pages[r];
    if (r < a.n) {
      const int len = length(r);
      a.kv_lens[r] = len;
      a.last_page_len[r] = len ? len - (pages_of(len) - 1) * a.page_size : 0;
    }
  }
  const int used = rows[a.n];
  for (int t = first; t < a.num_tokens; t += step) {
    int req = -1, pos = 0;
    int64_t slot = -1;
    if (t < used) {
      req = owner_of(rows, a.n, t);
      pos = context(req) + t - rows[req];
      const int page = a.tables[req * a.ld + pos / a.page_size];
      if (page >= 0 && page < a.num_pages) slot = (int64_t)page * 2 * a.page_size + pos % a.page_size;
    }
    a.batch_indices[t] = req;
    a.positions[t] = pos;
    a.kv_slots[t] = slot;
  }
  const int listed = pages[a.n];
  for (int64_t e = first; e < a.capacity; e += step) {
    int32_t v = -1;
    if (e < listed) {
      const int r = owner_of(pages, a.n, (int)e);
      v = a.tables[r * a.ld + (e - pages[r])];
    }
    a.kv_indices[e] = v;
  }
}

}  // namespace sb200

using namespace sb200;

// A range of memory that a call reads or writes.
struct Range {
  const void* at;
  uint64_t bytes;
};

// Does any of the written ranges meet another one of them, or one of those that are read?
template <int W, int R> static bool any_meet(const Range (&written)[W], const Range (&read)[R]) {
  for (int i = 0; i < W; ++i) {
    for (int j = i + 1; j < W; ++j)
      if (ranges_meet(written[i].at, written[i].bytes, written[j].at, written[j].bytes)) return true;
    for (int j = 0; j < R; ++j)
      if (ranges_meet(written[i].at, written[i].bytes, read[j].at, read[j].bytes)) return true;
  }
  return false;
}

// (Each kernel is allowed what kMaxRequests need, once: the limit without that counts its static shared memory too, and a limit that
// follows each call's own size would be lowered under another thread's launch.)
static size_t layout_smem(int n, int arrays) { return (size_t)arrays * (n + 1) * sizeof(int); }

extern "C" int sb200_resize_block_tables(int32_t* block_tables, int64_t ld, int32_t* num_blocks, const int32_t* seq_lens,
                                         int32_t* free_blocks, int32_t* num_free, int32_t* granted, int num_requests, int width,
                                         int64_t capacity, int page_size, sb200_stream_t stream) {
  SB_CHECK_ARG(num_requests >= 0 && width >= 0 && capacity >= 0 && page_size > 0 && ld >= width && width < INT32_MAX &&
                   capacity <= INT32_MAX && (int64_t)num_requests * width <= INT32_MAX / 2,
               "resize_block_tables: bad sizes (%d requests, %d blocks each, %lld free)", num_requests, width, (long long)capacity);
  if (num_requests > kMaxRequests) {
    set_error("resize_block_tables: %d requests, at most %d are supported", num_requests, kMaxRequests);
    return SB200_ERR_UNSUPPORTED;
  }
  if (num_requests == 0) return SB200_OK;
  SB_CHECK_ARG((block_tables || width == 0) && num_blocks && seq_lens && (free_blocks || capacity == 0) && num_free && granted,
               "resize_block_tables: null pointer");
  const uint64_t n = num_requests;
  const Range written[] = {{block_tables, width ? ((n - 1) * ld + width) * 4 : 0}, {num_blocks, n * 4}, {free_blocks, (uint64_t)capacity * 4},
                           {num_free, 4}, {granted, n * 4}};
  const Range read[] = {{seq_lens, n * 4}};
  SB_CHECK_ARG(!any_meet(written, read), "resize_block_tables: the arrays must not overlap");
  TablesArgs a = {block_tables, ld, num_blocks, seq_lens, free_blocks, num_free, granted, num_requests, width, (int)capacity, page_size};
  // Eight CTAs where the tables could hold so many pages that a prompt's worth of them may move in one step.
  const int ctas = (int64_t)num_requests * width > 16384 ? 8 : 1;
  const size_t smem = layout_smem(num_requests, 4);
  static std::atomic<uint64_t> allowed{0};
  SB_CUDA(allow_smem(reinterpret_cast<const void*>(resize_tables_kernel), (int)layout_smem(kMaxRequests, 4), &allowed));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kTablesThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  SB_CUDA(cudaLaunchKernelEx(&cfg, resize_tables_kernel, a));
  return SB200_OK;
}

extern "C" int sb200_batch_layout(const int32_t* query_lens, const int32_t* context_lens, const int32_t* block_tables, int64_t ld,
                                  int num_requests, int width, int page_size, int64_t num_pages, int64_t num_tokens,
                                  int32_t* qo_indptr, int32_t* kv_lens, int32_t* kv_indptr, int32_t* kv_indices,
                                  int64_t kv_capacity, int32_t* last_page_len, int32_t* batch_indices, int64_t* positions,
                                  int64_t* kv_slots, sb200_stream_t stream) {
  SB_CHECK_ARG(num_requests >= 0 && width >= 0 && page_size > 0 && ld >= width && num_pages >= 0 && num_pages <= INT32_MAX &&
                   num_tokens >= 0 && num_tokens <= INT32_MAX / 2 && (int64_t)num_requests * width <= INT32_MAX,
               "batch_layout: bad sizes (%d requests, %d blocks each, %lld tokens)", num_requests, width, (long long)num_tokens);
  if (num_requests > kMaxRequests) {
    set_error("batch_layout: %d requests, at most %d are supported", num_requests, kMaxRequests);
    return SB200_ERR_UNSUPPORTED;
  }
  SB_CHECK_ARG(kv_capacity >= (int64_t)num_requests * width, "batch_layout: kv_indices must hold %lld entries",
               (long long)num_requests * width);
  SB_CHECK_ARG(qo_indptr && kv_indptr && (num_requests == 0 || (query_lens && context_lens && kv_lens && last_page_len)) &&
                   (kv_capacity == 0 || kv_indices) && ((int64_t)num_requests * width == 0 || block_tables) &&
                   (num_tokens == 0 || (batch_indices && positions && kv_slots)),
               "batch_layout: null pointer");
  // (every CTA reads the lengths for itself while others may have written theirs: last step's kv_lens, say, must be copied first)
  const uint64_t n = num_requests, t = num_tokens;
  const Range written[] = {{qo_indptr, (n + 1) * 4}, {kv_lens, n * 4}, {kv_indptr, (n + 1) * 4}, {kv_indices, (uint64_t)kv_capacity * 4},
                           {last_page_len, n * 4}, {batch_indices, t * 4}, {positions, t * 8}, {kv_slots, t * 8}};
  const Range read[] = {{query_lens, n * 4}, {context_lens, n * 4}, {block_tables, n && width ? ((n - 1) * ld + width) * 4 : 0}};
  SB_CHECK_ARG(!any_meet(written, read), "batch_layout: the arrays it writes must not overlap each other or those it reads");
  LayoutArgs a = {query_lens, context_lens, block_tables, ld, qo_indptr, kv_lens, kv_indptr, kv_indices, last_page_len, batch_indices,
                  positions, kv_slots, num_requests, width, page_size, (int)num_pages, (int)num_tokens, kv_capacity};
  // One item a thread, up to a CTA per SM: the prefix sums that each CTA makes cost as much as a few items.
  int64_t items = kv_capacity > num_tokens ? kv_capacity : num_tokens;
  if (items < num_requests + 1) items = num_requests + 1;
  int64_t ctas = (items + kLayoutThreads - 1) / kLayoutThreads;
  if (ctas > sm_count()) ctas = sm_count();
  const size_t smem = layout_smem(num_requests, 2);
  static std::atomic<uint64_t> allowed{0};
  SB_CUDA(allow_smem(reinterpret_cast<const void*>(batch_layout_kernel), (int)layout_smem(kMaxRequests, 2), &allowed));
  SB_CUDA(launch_dependent(batch_layout_kernel, dim3((unsigned)ctas), dim3(kLayoutThreads), smem, (cudaStream_t)stream, a));
  return SB200_OK;
}

// Attention of a step's new tokens over the paged KV cache: the plan kernel, the join of cut units, the C entry points.
// attention.cuh has the division of the work, attention_simt.cu the fp32 kernel, attention_tc.cu the tensor-core kernel.
//
// Replaces the flashinfer calls of the reference's attention wrapper
// (sarathi/model_executor/attention/flashinfer_attention_wrapper.py:240-299: one paged prefill wrapper for prompt chunks
// and decodes, planned once a step in begin_forward and run by every layer).
#include "attention.cuh"

namespace sb200 {

constexpr int kPlanThreads = 1024;
constexpr int kNearTiles = 1024;
constexpr int kJoinThreads = 256, kJoinValues = 4 * kJoinThreads;

struct PlanArgs {
  AttnPlanView plan;
  const int32_t *qo_indptr, *kv_lens, *kv_indptr;
  int64_t num_kv_indices;
  int n, workers, max_tokens;
  AttnShape sh;
};

// What a block of keys, and a unit apart from its blocks, costs a CTA, in hundredths of a microsecond, and the least blocks of a
// piece.  Fitted to when the CTAs ended in 17 steps, most of them mixed, their keys in HBM: 0.2 us a block more for many rows than where
// every SM does them, a window's masks at both ends 2 us a unit.  Few rows count at the share of HBM that an SM has when all of them
// stream (3 % less than fitted then, as a unit starts faster since: 512 rows with 100 decodes 187 -> 182 us).
__device__ __forceinline__ void unit_cost(const AttnShape& sh, int kind, int nrows, int* block, int* fixed, int* least) {
  const bool wide = sh.head_dim > 64;
  if (sh.dtype == SB200_F32) {
    *block = (kind == ATTN_MANY ? 1200 : 150) * sh.head_dim / 64;
    *fixed = kind == ATTN_MANY ? 350 : 200;
    *least = 1;
  } else if (kind == ATTN_MANY) {
    *block = nrows > 128 ? (wide ? 192 : 170) : (wide ? 170 : 150);
    *fixed = (wide ? 508 : 480) + (sh.window > 0 ? 200 : 0);
    *least = 2;
  } else {
    *block = sh.head_dim == 256 ? 290 : wide ? 145 : 97;
    *fixed = wide ? 250 : 215;
    *least = 2;
  }
}

// A unit as a whole.  fp32 tiles of many rows go 64 keys (or 32) at a time: a half of the first or last block that no row sees is not
// done.  (A chunk of 256 tokens with 32 decodes: the last worker done after 37 us, most of them after 27, with whole blocks.)
__device__ __forceinline__ long long unit_time(const AttnShape& sh, const AttnTile& d, int block, int fixed, int* lead) {
  *lead = 0;
  long long t = (long long)d.nblk * block + fixed;
  if (sh.dtype == SB200_F32 && d.kind == ATTN_MANY && d.nblk > 0) {
    const int tok0 = d.row0 / sh.group, tok1 = (d.row0 + d.nrows - 1) / sh.group;
    const int hi = max(0, d.pos0 + tok1 + 1), lo = sh.window > 0 ? max(0, d.pos0 + tok0 + 1 - sh.window) : 0;
    if (lo - d.blk_lo * kAttnBlock >= kAttnBlock / 2) *lead = block / 2;
    t -= *lead;
    if ((d.blk_lo + d.nblk) * kAttnBlock - hi >= kAttnBlock / 2) t -= block / 2;
  }
  return t;
}

constexpr long long kShareMany = 200, kShareFew = 150, kJoinMany = 500, kJoinFew = 250;

__device__ __forceinline__ long long scan_block(long long v, long long* red, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) red[warp] = x;
  __syncthreads();
  if (warp == 0) {
    long long s = red[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    red[lane] = s;
  }
  __syncthreads();
  *total = red[31];
  return x - v + (warp ? red[warp - 1] : 0);
}

// One CTA: tiles per request (prefix sum over the requests), then the tiles and their costs (prefix sum over the tiles,
// 1024 at a time), then the start of every worker's share (binary search).  Made once a step, read by every layer; 8 us, bound by
// latency (three block-wide sums, a search in shared memory, the tile it finds).
__global__ void __launch_bounds__(kPlanThreads)
attn_plan_kernel(const PlanArgs a) {
  grid_dependency_begin();
  extern __shared__ int smem_i[];
  int* first = smem_i;               // [n + 1] first tile of every request that has tiles of many rows,
  int* few = smem_i + a.n + 1;       // and of those with few: these come behind all others
  __shared__ long long red[33];
  __shared__ long long near[kNearTiles];  // costs of the first tiles: the search below reads them one after the other
  const AttnShape& sh = a.sh;
  const int per = (a.n + kPlanThreads - 1) / kPlanThreads, r0 = min(a.n, (int)threadIdx.x * per), r1 = min(a.n, r0 + per);
  auto span = [&](int r, int* q0) {
    const int b = max(0, min(a.qo_indptr[r], a.max_tokens)), e = max(0, min(a.qo_indptr[r + 1], a.max_tokens));
    *q0 = b;
    return max(0, e - b);
  };
  auto kind_of = [&](int qlen, int* rows) {
    const long long all = (long long)qlen * sh.group;
    if (all <= sh.few_limit) { *rows = sh.rows_few; return (int)ATTN_FEW; }
    *rows = sh.rows_many;
    return (int)ATTN_MANY;
  };
  auto tiles_of = [&](int r, bool want_few) {
    int q0, rows;
    const int q = span(r, &q0);
    const bool is_few = kind_of(q, &rows) == ATTN_FEW;
    return is_few == want_few ? ((long long)q * sh.group + rows - 1) / rows : 0;
  };
  long long total, many_total = 0;
  for (int kind = 0; kind < 2; ++kind) {
    int* at = kind ? few : first;
    long long s = 0;
    for (int r = r0; r < r1; ++r) s += tiles_of(r, kind);
    long long p = scan_block(s, red, &total) + many_total;
    for (int r = r0; r < r1; ++r) {
      at[r] = (int)min(p, (long long)a.plan.tiles_cap);
      p += tiles_of(r, kind);
    }
    total += many_total;
    if (threadIdx.x == 0) at[a.n] = (int)min(total, (long long)a.plan.tiles_cap);
    if (!kind) many_total = total;
  }
  const int tiles = (int)min(total, (long long)a.plan.tiles_cap), tiles_many = (int)min(many_total, (long long)a.plan.tiles_cap);
  __syncthreads();

  long long carry = 0;
  for (int base = 0; base < tiles; base += kPlanThreads) {
    const int t = base + threadIdx.x;
    long long c = 0;
    if (t < tiles) {
      const int* begin = t < tiles_many ? first : few;
      int lo = 0, hi = a.n;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (begin[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      AttnTile d;
      int rows;
      const int q = span(lo, &d.q_row);
      d.kind = kind_of(q, &rows);
      d.row0 = (t - begin[lo]) * rows;
      d.nrows = (int)min((long long)rows, (long long)q * sh.group - d.row0);
      // no more tokens than the listed pages have room for, whatever the length says
      const long long at0 = min((long long)max(0, a.kv_indptr[lo]), (long long)a.num_kv_indices);
      const long long at1 = min((long long)max(0, a.kv_indptr[lo + 1]), (long long)a.num_kv_indices);
      const long long room = min(max(0ll, at1 - at0) * sh.page_size, (long long)kAttnMaxKeys);
      const int len = (int)min((long long)max(0, a.kv_lens[lo]), room);
      d.pos0 = len - q;
      d.page_at = (int)at0;
      const int tok0 = d.row0 / sh.group, tok1 = (d.row0 + d.nrows - 1) / sh.group;
      const int seen_hi = max(0, d.pos0 + tok1 + 1);
      const int seen_lo = sh.window > 0 ? max(0, d.pos0 + tok0 + 1 - sh.window) : 0;
      d.blk_lo = seen_lo / kAttnBlock;
      d.nblk = max(0, (seen_hi + kAttnBlock - 1) / kAttnBlock - d.blk_lo);
      int4* dst = reinterpret_cast<int4*>(a.plan.tiles + t);
      dst[0] = make_int4(d.q_row, d.row0, d.nrows, d.kind);
      dst[1] = make_int4(d.pos0, d.page_at, d.blk_lo, d.nblk);
      int block, fixed, least;
      unit_cost(sh, d.kind, d.nrows, &block, &fixed, &least);
      int lead;
      c = unit_time(sh, d, block, fixed, &lead) * sh.kv_heads;
    }
    const long long at = carry + scan_block(c, red, &total);
    if (t < tiles) {
      a.plan.cost[t] = at;
      if (t < kNearTiles) near[t] = at;
    }
    carry += total;
  }
  __shared__ int4 at[kAttnMaxWorkers + 1];
  if (threadIdx.x == 0) a.plan.cost[tiles] = carry;
  __syncthreads();
  // No more workers than have a share worth starting for (in hundredths of a microsecond, as unit_cost): a piece more is a start, a
  // store of its part and a load in the join.
  const long long busy = max(1ll, min((long long)a.workers, carry / (tiles_many ? kShareMany : kShareFew)));
  // No more units than workers: every unit can have workers of its own, each with one piece of it.  That saves a worker the second
  // start and store that a share across a cut costs, but the pieces are no longer equal: warp k looks at shares of at most
  // 1 + k / 10 times the equal one, and the least that suffices is taken if it is not beyond the equal share with a unit's fixed cost.
  // Nothing is cut at all where that costs less than the join does.  (Heads of 64, 16 on 4, chunks of 333, 326 and 319 tokens at 1500,
  // 1000 and 500: 31.7 -> 26.0 us, 37 decodes with a window of 1000 tokens: 17.4 -> 12.6.)
  __shared__ int near_blocks[kAttnMaxWorkers], near_cost[kAttnMaxWorkers], near_fixed[kAttnMaxWorkers];
  __shared__ unsigned suffices;
  __shared__ int largest;
  bool aligned = false;
  if (tiles > 0 && (long long)tiles * sh.kv_heads <= a.workers) {
    if (threadIdx.x == 0) { suffices = 0; largest = 0; }
    __syncthreads();
    if ((int)threadIdx.x < tiles) {
      const AttnTile d = a.plan.tiles[threadIdx.x];
      int block, fixed, least;
      unit_cost(sh, d.kind, d.nrows, &block, &fixed, &least);
      near_blocks[threadIdx.x] = d.nblk;
      near_cost[threadIdx.x] = block;
      near_fixed[threadIdx.x] = fixed;
      int lead;
      atomicMax(&largest, (int)min(unit_time(sh, d, block, fixed, &lead), 1ll << 30));
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
    const long long equal = carry / busy;
    auto pieces_of = [&](int t, int factor) {  // of a unit, where no piece may take longer than equal (1 + factor / 10)
      const long long room = max(equal + equal * factor / 10 - near_fixed[t], (long long)near_cost[t]) / near_cost[t];
      return (int)max(1ll, min((near_blocks[t] + room - 1) / room, (long long)a.workers));
    };
    int sum = 0;
    for (int t = lane; t < tiles; t += 32) sum += pieces_of(t, k);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0 && (long long)sum * sh.kv_heads <= busy) atomicOr(&suffices, 1u << k);
    __syncthreads();
    const int factor = suffices ? __ffs(suffices) - 1 : 32;
    aligned = factor < 32 && equal * factor / 10 <= near_fixed[0];
    const bool whole = largest <= equal + (aligned ? equal * factor / 10 : near_fixed[0]) + (tiles_many ? kJoinMany : kJoinFew);
    aligned = aligned || whole;
    if (aligned) {
      const int own = (int)threadIdx.x >= tiles ? 0 : whole ? 1 : pieces_of(threadIdx.x, factor);
      const int from = (int)scan_block((long long)own * sh.kv_heads, red, &total);
      for (int h = 0; h < sh.kv_heads && own; ++h)
        for (int i = 0; i < own; ++i)
          at[from + h * own + i] = make_int4((int)threadIdx.x, h, (int)((long long)near_blocks[threadIdx.x] * i / own), 0);
      for (int w = (int)total + threadIdx.x; w <= a.workers; w += kPlanThreads) at[w] = make_int4(tiles, 0, 0, 0);
    }
  }
  // A share that begins inside a unit has a start more than the line says, a dearer one among the units of many rows: the workers
  // that do those get as much less to do.  (In units of 1/1024 worker.  512 rows with 64 decodes of 512 to 8192 tokens: the last
  // worker done after 221 us, half of them after 182, without this and with the costs of a step of many rows only.)
  const long long line_many = tiles_many < tiles ? a.plan.cost[tiles_many] : carry, line_few = carry - line_many;
  long long workers_many = 0;
  if (line_many > 0) {
    int block, fixed_many, fixed_few, least;
    unit_cost(sh, ATTN_MANY, sh.rows_many, &block, &fixed_many, &least);
    unit_cost(sh, ATTN_FEW, sh.rows_few, &block, &fixed_few, &least);
    const long long equal = carry / busy, own = max(equal - line_few * max(0, fixed_many - fixed_few) / carry, equal / 2 + 1);
    workers_many = line_few == 0 ? busy * 1024 : min(line_many * 1024 / own, busy * 1024 - 1);
  }
  for (int w = aligned ? a.workers + 1 : (int)threadIdx.x; w <= a.workers; w += kPlanThreads) {
    int4 out = make_int4(tiles, 0, 0, 0);
    if (w < busy && tiles > 0) {
      const long long x = w * 1024 <= workers_many ? line_many * (w * 1024) / max(workers_many, 1ll)
                                                   : line_many + line_few * (w * 1024 - workers_many) / (busy * 1024 - workers_many);
      int lo = 0, hi = tiles - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((mid < kNearTiles ? near[mid] : a.plan.cost[mid]) <= x) lo = mid;
        else hi = mid - 1;
      }
      const AttnTile d = a.plan.tiles[lo];
      int block, fixed, least;
      unit_cost(sh, d.kind, d.nrows, &block, &fixed, &least);
      int lead;
      const long long unit = unit_time(sh, d, block, fixed, &lead), rem = x - (lo < kNearTiles ? near[lo] : a.plan.cost[lo]);
      int head = (int)(rem / unit);
      const long long in = rem - head * unit + lead;
      int blk = in <= fixed / 2 ? 0 : (int)min((in - fixed / 2 + block / 2) / block, (long long)d.nblk);
      // no piece of less than `least` blocks: the cut moves to the end of the unit it is near to
      if (blk < least) blk = 0;
      else if (d.nblk - blk < least) { blk = 0; ++head; }
      out = head < sh.kv_heads ? make_int4(lo, head, blk, 0) : make_int4(lo + 1, 0, 0, 0);
    }
    at[w] = out;
  }
  __syncthreads();
  // One thread per worker from here on (workers < threads).
  const int w = threadIdx.x;
  auto same = [&](int x, int y) { return at[x].x == at[y].x && at[x].y == at[y].y; };
  auto empty = [&](int x) { return same(x, x + 1) && at[x].z == at[x + 1].z; };
  int own = 0;  // pieces of this worker that are not whole units: one that begins inside a unit, one that ends inside one
  if (w < a.workers && !empty(w)) own = (at[w].z > 0) + (at[w + 1].z > 0 && !(at[w].z > 0 && same(w, w + 1)));
  const int slot = (int)scan_block(own, red, &total);
  const bool first_in = w > 0 && w < a.workers && at[w].z > 0 && !(at[w - 1].z > 0 && same(w - 1, w));
  const AttnTile d = w <= a.workers && at[min(w, a.workers)].x < tiles ? a.plan.tiles[at[min(w, a.workers)].x] : AttnTile{};
  const long long unit = scan_block(first_in ? 1 : 0, red, &total);
  const int units = (int)total;
  const int groups = first_in ? (d.nrows * sh.head_dim + kJoinValues - 1) / kJoinValues : 0;
  const int group0 = (int)scan_block(groups, red, &total);
  if (first_in) {  // (the slot before this worker's first holds the piece before it)
    int pieces = 1;
    for (int v = w; v < a.workers && same(v, w); ++v) pieces += !empty(v);
    a.plan.cuts[unit] = AttnCut{d.q_row, d.row0, d.nrows, d.pos0, at[w].y, slot - 1, pieces, 0};
    a.plan.cut_first[unit] = group0;
  }
  if (w == 0) a.plan.cut_first[units] = (int)total;
  if (w <= a.workers) {
    AttnStart s;
    s.at = at[w];
    s.tile = d;
    s.many = tiles_many;
    s.slot = slot;
    s.rows = a.n ? max(0, min(a.qo_indptr[w == 1 ? 0 : a.n], a.max_tokens)) : 0;
    s.units = units;
    const int4* src = reinterpret_cast<const int4*>(&s);
    int4* dst = reinterpret_cast<int4*>(a.plan.starts + w);
    for (int i = 0; i < 4; ++i) dst[i] = src[i];
  }
}

// Joins the pieces of cut units: o = sum_p 2^(l_p - m) o_p / sum_p 2^(l_p - m) with l_p the log2 of piece p's sum, in the
// order of the keys.  The cut units' rows are dealt out in groups of 1024 values, four a thread: neighbouring lanes have neighbouring
// rows, which is how the slots are laid out.  Also clears the rows that belong to no request, when asked to.  Bound by
// latency: the groups' prefix sums, the unit and its pieces (sums and outputs of four at a time) are three loads after one another:
// 2 to 4 us for decodes, 20 with a cut unit of 256 rows on every SM.
// What it reads of the plan it reads ahead of its wait: the attention kernel lets it start only when its own wait is over, and the plan
// was complete then.
template <typename T, int HD>
__global__ void __launch_bounds__(kJoinThreads, 5)
attn_join_kernel(const AttnArgs a) {
  constexpr int kRows = kJoinValues / HD, kBatch = 4;
  __shared__ int first[kAttnMaxWorkers + 1];
  T* out = reinterpret_cast<T*>(a.out);
  const int units = attn_clamp(__ldcg(&a.plan.starts[0].units), 0, a.workers);  // (what comes from the plan: see attn_piece)
  for (int i = threadIdx.x; i <= a.workers; i += kJoinThreads) first[i] = __ldcg(a.plan.cut_first + i);  // (behind `units`: anything)
  __syncthreads();
  const int groups = min(first[units], a.workers * (a.slot_rows * HD / kJoinValues));
  int lo = 0;
  int4 u, v;  // the cut unit of group g
  auto look_up = [&](int g) {
    int hi = units - 1;
    lo = 0;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= g) lo = mid;
      else hi = mid - 1;
    }
    const int4* rec = reinterpret_cast<const int4*>(a.plan.cuts + lo);
    u = __ldcg(rec);
    v = __ldcg(rec + 1);
  };
  if ((int)blockIdx.x < groups) look_up(blockIdx.x);
  grid_dependency_begin();
  if (a.zero_behind) {
    const int ahead = attn_clamp(a.plan.starts[1].rows, 0, a.num_tokens);
    const int behind = attn_clamp(a.plan.starts[0].rows, ahead, a.num_tokens), per_row = a.kv_heads * a.group * HD;
    for (int row = blockIdx.x; row < ahead + a.num_tokens - behind; row += gridDim.x) {
      const int t = row < ahead ? row : row - ahead + behind;
      for (int i = threadIdx.x; i < per_row; i += kJoinThreads) out[t * a.ldo + i] = DT<T>::from_f(0.f);
      if (a.lse)
        for (int i = threadIdx.x; i < a.kv_heads * a.group; i += kJoinThreads)
          a.lse[(int64_t)t * (a.kv_heads * a.group) + i] = -INFINITY;
    }
  }
  for (int g = blockIdx.x; g < groups; g += gridDim.x) {
    if (g != (int)blockIdx.x) look_up(g);
    const AttnCut c = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
    const int r = (g - first[lo]) * kRows + threadIdx.x % kRows, col4 = threadIdx.x / kRows;
    const bool fine = (unsigned)c.q_row <= (unsigned)a.num_tokens && (unsigned)c.row0 <= (unsigned)(a.num_tokens * a.group) &&
                      (unsigned)c.nrows <= (unsigned)a.slot_rows && (unsigned)c.head < (unsigned)a.kv_heads &&
                      (unsigned)c.slot <= (unsigned)(2 * a.workers) && (unsigned)c.pieces <= (unsigned)(2 * a.workers - c.slot);
    if (!fine || (unsigned)r >= (unsigned)min(c.nrows, max(0, (a.num_tokens - c.q_row) * a.group - c.row0))) continue;
    float m = -INFINITY, base = 0.f, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < c.pieces; i += kBatch) {
      float l[kBatch];
      float4 o[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int slot = c.slot + min(i + k, c.pieces - 1);
        l[k] = i + k < c.pieces ? a.part_l[(int64_t)slot * a.slot_rows + r] : -INFINITY;
        o[k] = *attn_part(a, HD, slot, c.nrows, r, col4);
      }
      float top = m;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) top = fmaxf(top, l[k]);
      base = top == -INFINITY ? 0.f : top;
      const float keep = m == -INFINITY ? 0.f : exp2f(m - base);  // (a further batch: what there is comes to the new maximum)
      m = top;
      sum *= keep;
      acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const float wt = exp2f(l[k] - base);
        sum += wt;
        if (i + k < c.pieces) {  // (a piece that this row sees nothing of holds zeros; one that it sees counts, however small its weight)
          acc.x += wt * o[k].x; acc.y += wt * o[k].y; acc.z += wt * o[k].z; acc.w += wt * o[k].w;
        }
      }
    }
    const int row = c.row0 + r, tok = a.by_group.div(row);
    const int token = c.q_row + tok, head = c.head * a.group + (row - tok * a.group);
    const float inv = attn_inverse(sum, c.pos0 + tok);
    T* dst = out + token * a.ldo + head * HD + col4 * 4;
    dst[0] = DT<T>::from_f(acc.x * inv); dst[1] = DT<T>::from_f(acc.y * inv);
    dst[2] = DT<T>::from_f(acc.z * inv); dst[3] = DT<T>::from_f(acc.w * inv);
    if (a.lse && col4 == 0) a.lse[(int64_t)token * (a.kv_heads * a.group) + head] = (base + log2f(sum)) * 0.69314718055994531f;
  }
}

// ------------------------------------------------------------------ host
static int attn_shape(const sb200_attention_shape* s, AttnShape* sh, const char* what) {
  SB_CHECK_ARG(s, "%s: null shape", what);
  SB_CHECK_ARG(s->num_heads > 0 && s->num_kv_heads > 0 && s->num_heads % s->num_kv_heads == 0,
               "%s: %d heads cannot share %d kv heads evenly", what, s->num_heads, s->num_kv_heads);
  SB_CHECK_ARG(s->page_size > 0 && s->page_size <= (1 << 20) && s->window >= 0 && s->max_requests >= 0 && s->max_tokens >= 0 &&
                   s->max_tokens <= (1 << 28) && s->num_heads <= (1 << 16) &&
                   (int64_t)s->max_tokens * (s->num_heads / s->num_kv_heads) <= (1 << 30),
               "%s: bad sizes", what);
  if (s->head_dim != 64 && s->head_dim != 128 && s->head_dim != 256) {
    set_error("%s: head size %d is not supported (64, 128 or 256)", what, s->head_dim);
    return SB200_ERR_UNSUPPORTED;
  }
  if (s->max_requests > SB200_MAX_REQUESTS) {
    set_error("%s: %d requests, at most %d are supported", what, s->max_requests, SB200_MAX_REQUESTS);
    return SB200_ERR_UNSUPPORTED;
  }
  if (s->dtype != SB200_F32 && s->dtype != SB200_F16 && s->dtype != SB200_BF16) {
    set_error("%s: unsupported dtype id %d", what, s->dtype);
    return SB200_ERR_UNSUPPORTED;
  }
  sh->heads = s->num_heads;
  sh->kv_heads = s->num_kv_heads;
  sh->group = s->num_heads / s->num_kv_heads;
  sh->head_dim = s->head_dim;
  sh->page_size = s->page_size;
  sh->dtype = s->dtype;
  sh->window = s->window < kAttnMaxKeys ? s->window : 0;  // (a wider one hides nothing; position - window stays within 32 bits)
  // Tiles of 256 rows on tcgen05 fetch keys in boxes of whole swizzle atoms (8 rows), and hold scores and outputs of two halves in TMEM.
  // Pages that are no multiple of 8, and heads of 256, of which TMEM has room for one half (128 + 256 columns) only, stay with tiles of
  // 16 rows: a tenth of the rate in long chunks (2000 tokens at 8000, 32 heads on 8: 266 us with heads of 128 and pages of 16, 2232 with pages of
  // 12, 4754 with heads of 256).
  const bool many = s->dtype != SB200_F32 && s->head_dim <= 128 && s->page_size % 8 == 0;
  const bool f32 = s->dtype == SB200_F32;
  sh->rows_many = f32 ? 64 : many ? 256 : 16;
  sh->rows_few = f32 ? 4 : 16;
  sh->few_limit = f32 ? 8 : many ? 16 : INT32_MAX;
  return SB200_OK;
}

// Tiles of at most `rows` rows: every request may end in a partial one.
static int64_t tiles_cap(const AttnShape& sh, const sb200_attention_shape* s) {
  const int64_t few = sh.few_limit < INT32_MAX ? (sh.few_limit + sh.rows_few - 1) / sh.rows_few : 1;
  return (int64_t)s->max_tokens * sh.group / sh.rows_many + few * s->max_requests + 1;
}

static size_t align16(size_t v) { return (v + 15) & ~size_t(15); }

static size_t plan_view(void* base, int64_t cap, AttnPlanView* v) {
  uint8_t* p = reinterpret_cast<uint8_t*>(base);
  size_t at = 0;
  v->starts = reinterpret_cast<AttnStart*>(p + at);
  at += (kAttnMaxWorkers + 1) * sizeof(AttnStart);
  v->cuts = reinterpret_cast<AttnCut*>(p + at);
  at += kAttnMaxWorkers * sizeof(AttnCut);
  v->cut_first = reinterpret_cast<int*>(p + at);
  at += align16((kAttnMaxWorkers + 1) * sizeof(int));
  v->cost = reinterpret_cast<long long*>(p + at);
  at += align16((size_t)(cap + 1) * sizeof(long long));
  v->tiles = reinterpret_cast<AttnTile*>(p + at);
  at += (size_t)cap * sizeof(AttnTile);
  v->tiles_cap = (int)cap;
  return at;
}

static int attn_workers() {
  const int n = sm_count();
  return n < kAttnMaxWorkers ? n : kAttnMaxWorkers;
}

// Do `rows` rows of `row` bytes each, ldx and ldy bytes apart, meet anywhere?  (Columns of one buffer interleave without meeting.)
static bool rows_meet(const void* x, uint64_t ldx, const void* y, uint64_t ldy, uint64_t rows, uint64_t row) {
  if (!ranges_meet(x, (rows - 1) * ldx + row, y, (rows - 1) * ldy + row)) return false;
  if (ldx != ldy || rows == 1) return true;
  const uint64_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y), apart = (a < b ? b - a : a - b) % ldx;
  return apart < row || apart > ldx - row;
}

// Does a range meet any of `rows` rows of `row` bytes, ldx bytes apart?  (The gaps between them may hold it.)
static bool range_meets_rows(const void* r, uint64_t n, const void* x, uint64_t ldx, uint64_t rows, uint64_t row) {
  const uint64_t a = reinterpret_cast<uintptr_t>(r), b = reinterpret_cast<uintptr_t>(x);
  const uint64_t i = a < b + row ? 0 : (a - b - row) / ldx + 1;  // the first row that ends behind the range's start
  return i < rows && b + i * ldx < a + n;
}

static int slot_rows(const AttnShape& sh) { return sh.rows_many > sh.rows_few ? sh.rows_many : sh.rows_few; }

template <typename T>
static cudaError_t launch_join(int head_dim, const AttnArgs& a, dim3 grid, cudaStream_t s) {
  auto kern = head_dim == 64 ? attn_join_kernel<T, 64> : head_dim == 128 ? attn_join_kernel<T, 128> : attn_join_kernel<T, 256>;
  return launch_dependent(kern, grid, dim3(kJoinThreads), 0, s, a);
}

}  // namespace sb200

using namespace sb200;

extern "C" int64_t sb200_attention_plan_bytes(const sb200_attention_shape* shape) {
  AttnShape sh;
  if (attn_shape(shape, &sh, "attention_plan_bytes")) return -1;
  AttnPlanView v;
  return (int64_t)plan_view(nullptr, tiles_cap(sh, shape), &v);
}

extern "C" int64_t sb200_attention_workspace_bytes(const sb200_attention_shape* shape) {
  AttnShape sh;
  if (attn_shape(shape, &sh, "attention_workspace_bytes")) return -1;
  return (int64_t)2 * attn_workers() * slot_rows(sh) * (sh.head_dim + 1) * sizeof(float);
}

extern "C" int sb200_attention_plan(void* plan, int64_t plan_bytes, const sb200_attention_shape* shape, const int32_t* qo_indptr,
                                    const int32_t* kv_lens, const int32_t* kv_indptr, int num_requests, int64_t num_kv_indices,
                                    sb200_stream_t stream) {
  AttnShape sh;
  if (int rc = attn_shape(shape, &sh, "attention_plan")) return rc;
  SB_CHECK_ARG(num_requests >= 0 && num_requests <= shape->max_requests, "attention_plan: %d requests, made for at most %d",
               num_requests, shape->max_requests);
  PlanArgs a;
  const size_t need = plan_view(plan, tiles_cap(sh, shape), &a.plan);
  SB_CHECK_ARG(plan && aligned16(plan) && plan_bytes >= (int64_t)need, "attention_plan: the plan buffer must be 16-byte aligned and hold %lld bytes",
               (long long)need);
  SB_CHECK_ARG(qo_indptr && (num_requests == 0 || (kv_lens && kv_indptr)) && num_kv_indices >= 0 && num_kv_indices <= INT32_MAX,
               "attention_plan: null pointer or bad number of page entries");
  a.qo_indptr = qo_indptr;
  a.kv_lens = kv_lens;
  a.kv_indptr = kv_indptr;
  a.num_kv_indices = num_kv_indices;
  a.n = num_requests;
  a.workers = attn_workers();
  a.max_tokens = shape->max_tokens;
  a.sh = sh;
  const size_t smem = 2 * (size_t)(num_requests + 1) * sizeof(int);
  // (What the most requests need, once: the limit without it is on this and the kernel's static 16 KB together, and a limit that
  // follows each call's own size would be lowered under another thread's launch.)
  static std::atomic<uint64_t> allowed{0};
  SB_CUDA(allow_smem(reinterpret_cast<const void*>(attn_plan_kernel), 2 * (SB200_MAX_REQUESTS + 1) * (int)sizeof(int), &allowed));
  SB_CUDA(launch_dependent(attn_plan_kernel, dim3(1), dim3(kPlanThreads), smem, (cudaStream_t)stream, a));
  return SB200_OK;
}

extern "C" int sb200_paged_attention(void* out, int64_t ldo, float* lse, const void* q, int64_t ldq, int64_t num_tokens,
                                     const void* cache, int64_t num_pages, const void* plan, const sb200_attention_shape* shape,
                                     const int32_t* kv_indices, int64_t num_kv_indices, float scale, int zero_rows_behind,
                                     void* workspace, int64_t workspace_bytes, uint32_t* status, sb200_stream_t stream) {
  AttnShape sh;
  if (int rc = attn_shape(shape, &sh, "paged_attention")) return rc;
  SB_CHECK_ARG(num_tokens >= 0 && num_tokens <= shape->max_tokens, "paged_attention: %lld tokens, the plan is made for at most %d",
               (long long)num_tokens, shape->max_tokens);
  if (num_tokens == 0) return SB200_OK;
  const int64_t row = (int64_t)sh.heads * sh.head_dim;
  const int64_t es = (int64_t)dtype_size(sh.dtype);
  SB_CHECK_ARG(out && q && plan && cache && (kv_indices || num_kv_indices == 0), "paged_attention: null pointer");
  SB_CHECK_ARG(ldq >= row && ldo >= row && aligned16(q) && aligned16(out) && aligned16(cache) && (ldq * es) % 16 == 0 && (ldo * es) % 16 == 0,
               "paged_attention: rows of q and out must be 16-byte aligned and at least %lld elements apart", (long long)row);
  // (the kernels address the rows of q by 32-bit numbers of 16 bytes, the last of which stands for no row)
  SB_CHECK_ARG(ldq <= (int64_t)((uint64_t)UINT32_MAX * 16 / es) / num_tokens && ldo <= INT64_MAX / es / num_tokens,
               "paged_attention: %lld rows of q or out are too far apart (%lld, %lld)", (long long)num_tokens, (long long)ldq, (long long)ldo);
  SB_CHECK_ARG(num_pages > 0 && num_kv_indices >= 0 && num_pages * 2 * sh.page_size <= INT32_MAX, "paged_attention: bad cache of %lld pages",
               (long long)num_pages);
  SB_CHECK_ARG(workspace && aligned16(workspace) && workspace_bytes >= sb200_attention_workspace_bytes(shape),
               "paged_attention: the workspace must be 16-byte aligned and hold %lld bytes", (long long)sb200_attention_workspace_bytes(shape));
  SB_CHECK_ARG(isfinite(scale), "paged_attention: the scale is not a finite number");
  const uint64_t out_bytes = (uint64_t)((num_tokens - 1) * ldo + row) * es;
  const uint64_t cache_bytes = (uint64_t)num_pages * 2 * sh.page_size * sh.kv_heads * sh.head_dim * es;
  SB_CHECK_ARG(!rows_meet(q, ldq * es, out, ldo * es, num_tokens, row * es) && !ranges_meet(out, out_bytes, cache, cache_bytes),
               "paged_attention: out must not overlap q or the cache");
  const uint64_t lse_bytes = (uint64_t)num_tokens * sh.heads * sizeof(float);
  SB_CHECK_ARG(!lse || (!range_meets_rows(lse, lse_bytes, out, ldo * es, num_tokens, row * es) &&
                        !range_meets_rows(lse, lse_bytes, q, ldq * es, num_tokens, row * es) &&
                        !ranges_meet(lse, lse_bytes, cache, cache_bytes)),
               "paged_attention: lse must not overlap out, q or the cache");
  AttnArgs a = {};
  plan_view(const_cast<void*>(plan), tiles_cap(sh, shape), &a.plan);
  a.q = q; a.ldq = ldq; a.out = out; a.ldo = ldo; a.lse = lse; a.cache = cache;
  a.kv_indices = kv_indices;
  a.num_kv_indices = num_kv_indices;
  a.num_pages = (int)num_pages;
  a.num_tokens = (int)num_tokens;
  a.kv_heads = sh.kv_heads;
  a.group = sh.group;
  a.page_size = sh.page_size;
  a.by_group = FastDiv::of(sh.group);
  a.by_page = FastDiv::of(sh.page_size);
  a.window = sh.window;
  a.slot_rows = slot_rows(sh);
  a.part_o = reinterpret_cast<float*>(workspace);
  a.part_l = a.part_o + (size_t)2 * attn_workers() * a.slot_rows * sh.head_dim;
  a.status = status;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.zero_behind = zero_rows_behind;
  const int workers = a.workers = attn_workers();
  a.rows_many = sh.rows_many;
  a.rows_few = sh.rows_few;
  a.many_cap = sh.few_limit < INT32_MAX ? a.plan.tiles_cap : 0;
  const int64_t listed = min(num_kv_indices * sh.page_size, (int64_t)kAttnMaxKeys);
  a.blocks = (int)((listed + kAttnBlock - 1) / kAttnBlock);
  cudaStream_t s = (cudaStream_t)stream;
  if (int rc = sh.dtype == SB200_F32 ? run_attn_simt(sh.head_dim, a, workers, s)
                                     : run_attn_tc(sh.dtype, sh.head_dim, a, sh, workers, s))
    return rc;
  const dim3 grid((unsigned)(workers * 5));  // as many as are resident
  SB_DISPATCH_FLOAT(sh.dtype, SB_CUDA(launch_join<scalar_t>(sh.head_dim, a, grid, s)));
  return SB200_OK;
}

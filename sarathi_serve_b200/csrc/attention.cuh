// What the attention kernels share: the plan of a step (which CTA does which rows against which keys), the addressing of
// the paged cache, and where a piece of work leaves its result.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i . k_j - m_i),   j <= pos_i  (and j > pos_i - window)
//
// A query row is a (token, q head) pair.  The `group` q heads that share a kv head also share its keys and values, so
// the rows of a request for one kv head are (token, head of the group) pairs, token-major, and a TILE is a run of them.  A
// UNIT is a tile for one kv head; its keys come in blocks of 128.  Units are laid end to end, tile by tile and head by
// head, weighted by what a block costs, and every CTA (one per SM) gets an equal share of that line: long contexts are cut
// wherever a share ends, short ones are not cut at all.  A PIECE is the part of a unit that one CTA does.  A piece that is
// a whole unit writes the output; the others leave (o / l, log2-sum) in fp32 in a workspace, and a second kernel joins the
// pieces of each cut unit in the order of their keys.  A CTA has at most two such pieces, its first and its last, so
// the workspace has two slots per CTA, and the result does not depend on timing.
#pragma once

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace sb200 {

constexpr int kAttnBlock = 128;       // keys of a block
constexpr int kAttnMaxKeys = 1 << 30; // of a request; positions are below
constexpr int kAttnMaxWorkers = 256;  // (B200: 148 SMs)

// How the rows of a tile are computed.
enum { ATTN_FEW = 1, ATTN_MANY = 2 };

struct AttnTile {
  int q_row;    // first row of the request's tokens in q
  int row0;     // first (token, head of the group) row of the tile
  int nrows;
  int kind;
  int pos0;     // position of the request's first new token (negative: more new tokens than the cache is said to hold)
  int page_at;  // first entry of the request's pages in kv_indices
  int blk_lo, nblk;  // blocks of keys that some row sees
};

// Where a worker's share begins, with the tile it begins in, in one line of memory: what a CTA needs before its first load of
// keys is one load away.
struct alignas(16) AttnStart {
  int4 at;        // (tile, head, block); (tiles, 0, 0) behind the last
  AttnTile tile;  // of `at`
  int many;       // tiles of many rows (they come before the others)
  int slot;       // of its first piece that is not a whole unit; slots of one unit follow one another in the order of the keys
  int rows;       // of the first worker: the row of q behind the last request's; of the second: the first request's first row
  int units;      // cut units
};

// A unit that is cut, for the join.
struct alignas(16) AttnCut {
  int q_row, row0, nrows, pos0;  // as in its tile
  int head, slot, pieces, pad;   // its pieces are in the slots from `slot` on
};

struct AttnPlanView {
  AttnStart* starts; // [workers + 1]
  AttnCut* cuts;     // [workers]
  int* cut_first;    // [workers + 1] first group of rows of every cut unit (see attn_join_kernel); the last entry: their number
  long long* cost;   // [tiles + 1] start of every tile on the line
  AttnTile* tiles;
  int tiles_cap;
};

struct AttnShape {
  int heads, kv_heads, group, head_dim, page_size, dtype, window;
  int rows_many;   // rows of a tile, and up to how many rows a request takes the kernel for few rows
  int rows_few;
  int few_limit;   // INT32_MAX: all
};

// n / d for 0 <= n < 2^31 as a product: with 2^(s - 1) < d <= 2^s and m = floor(2^(31 + s) / d) + 1, m d exceeds 2^(31 + s) by at
// most d <= 2^s, so n m / 2^(31 + s) exceeds n / d by less than 1 / d.  A division takes some 40 instructions instead, and the
// kernels make one for every row and every page they address.
struct FastDiv {
  uint32_t mul, shift, d;
  __host__ static FastDiv of(int d) {
    uint32_t s = 0;
    while ((1ll << s) < d) ++s;
    return FastDiv{(uint32_t)((1ull << (31 + s)) / (uint32_t)d + 1), 31 + s, (uint32_t)d};
  }
  __host__ __device__ __forceinline__ int div(int n) const { return (int)(((uint64_t)(uint32_t)n * mul) >> shift); }
};

struct AttnArgs {
  AttnPlanView plan;
  const void* q; int64_t ldq;
  void* out; int64_t ldo;
  float* lse;
  const void* cache;
  const int32_t* kv_indices;
  float* part_o;       // [2 workers] slots of [slot_rows x head_dim], see attn_part
  float* part_l;       // [2 workers][slot_rows]
  uint32_t* status;
  int64_t num_kv_indices;
  int num_pages, num_tokens;
  int workers;
  int rows_many, rows_few;  // of a tile, at most
  int many_cap;             // tiles of many rows, at most (0: this shape has none)
  int blocks;               // of a request, at most: no more than all listed pages hold
  int kv_heads, group, page_size, window, slot_rows;
  FastDiv by_group, by_page;
  float scale_log2;    // scale * log2(e): scores in powers of two
  int zero_behind;
};

struct AttnPiece {
  AttnTile t;
  int head, b0, b1;   // blocks [b0, b1) of the tile's nblk
  int slot;           // -1: the whole unit
  int lo, hi;         // keys [lo, hi) that some row of the tile sees
  int stride;         // rows of the tile as planned: what a slot is laid out by
};

// A slot holds [4 columns][row][4] floats: threads with a row each store 16 bytes side by side.
__device__ __forceinline__ float4* attn_part(const AttnArgs& a, int head_dim, int slot, int stride, int row, int col4) {
  return reinterpret_cast<float4*>(a.part_o + (int64_t)slot * a.slot_rows * head_dim) + (col4 * stride + row);
}

__host__ __device__ __forceinline__ int attn_min(int a, int b) { return a < b ? a : b; }
__host__ __device__ __forceinline__ int attn_max(int a, int b) { return a > b ? a : b; }
__host__ __device__ __forceinline__ int attn_clamp(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// The piece of tile t that begins at `cur`, in a share that ends at `end`; `most`: rows of its kind of tile, `slot`: of the share's next
// piece that is not a whole unit.
// What comes from the plan is held to what the call's own arguments allow.  Calls that share a plan follow one another, and then
// nothing changes here; if a caller lets them overlap all the same (graphs on two streams, the C interface), or hands over the plan of
// another shape, the numbers are wrong but no address is: rows are rows of q, there are no more steps than keys listed, and the page of
// a key, wherever its number comes from, is looked up within the list and checked.  (Only what addresses need: this code is in six
// places, and what it costs is fetching it.  With a clamp for each number three chunks of 1500 take 2 us of 88 more.)
__host__ __device__ __forceinline__ AttnPiece attn_piece(const AttnArgs& a, const AttnTile& t, int4 cur, int4 end, int most, int* slot) {
  AttnPiece p;
  const bool tail_cut = cur.x == end.x && cur.y == end.y;
  p.t = t;
  p.head = cur.y;
  p.b0 = cur.z;
  p.b1 = attn_max(cur.z, attn_min(tail_cut ? end.z : t.nblk, cur.z + a.blocks));
  p.slot = tail_cut || cur.z > 0 ? (*slot)++ : -1;
  p.stride = attn_min(t.nrows, most);
  // q may have fewer rows than the plan was made for (tokens x group stays below 2^30)
  const bool rows = (unsigned)t.q_row <= (unsigned)a.num_tokens && (unsigned)t.row0 <= (1u << 30);
  p.t.nrows = rows ? attn_max(0, attn_min(p.stride, (a.num_tokens - t.q_row) * a.group - t.row0)) : 0;
  const int first = a.by_group.div(t.row0), last = a.by_group.div(t.row0 + attn_max(p.t.nrows, 1) - 1);
  p.hi = attn_max(0, t.pos0 + last + 1);
  p.lo = a.window > 0 ? attn_min(attn_max(0, t.pos0 + first + 1 - a.window), kAttnMaxKeys) : 0;
  return p;
}

// Walks a worker's share of the line.  How many pieces it finds follows from the share's two ends alone, which all warps of a CTA have
// from one copy in shared memory; a piece's tile is the same for all lanes of a warp.  So waits for each other hold up even where the
// plan changes meanwhile (see attn_piece).
struct AttnWalk {
  int4 cur, end;
  int word;  // lane i, i + 8, ...: the i-th number of the tile at `cur`, asked for when the one before was taken
  int many, slot, most;
  // s: the worker's AttnStart and the first 16 bytes of the next one (attn_share)
  __device__ __forceinline__ AttnWalk(const AttnArgs& a, const int4* s) {
    cur = s[0];
    end = s[4];
    // (as attn_piece: these hold the tile, the head, the block and the two slots of a share)
    cur = make_int4(max(cur.x, 0), attn_clamp(cur.y, 0, a.kv_heads - 1), attn_clamp(cur.z, 0, kAttnMaxKeys / kAttnBlock), 0);
    if (end.x >= a.plan.tiles_cap) end = make_int4(a.plan.tiles_cap, 0, 0, 0);
    many = attn_clamp(s[3].x, 0, a.many_cap);
    slot = attn_clamp(s[3].y, 0, 2 * a.workers - 2);
    word = reinterpret_cast<const int*>(s + 1)[threadIdx.x & 7];
    most = 0;
  }
  __device__ __forceinline__ void fetch(const AttnArgs& a) {
    if (more()) word = reinterpret_cast<const int*>(a.plan.tiles + cur.x)[threadIdx.x & 7];
  }
  // Only the tiles of many rows, or the others.
  __device__ __forceinline__ void only_many(const AttnArgs& a) {
    most = a.rows_many;
    if (end.x >= many) end = make_int4(many, 0, 0, 0);
  }
  __device__ __forceinline__ void only_few(const AttnArgs& a) {
    most = a.rows_few;
    if (cur.x < many) {
      // pieces that are passed over keep their slots: the first, and the last if the share ends among them
      if (more() && cur.z > 0) ++slot;
      cur = make_int4(many, 0, 0, 0);
      fetch(a);
    }
  }
  __device__ __forceinline__ bool more() const {
    return cur.x < end.x || (cur.x == end.x && (cur.y < end.y || (cur.y == end.y && cur.z < end.z)));
  }
  // Called by whole warps.
  __device__ __forceinline__ bool next(const AttnArgs& a, AttnPiece* p) {
    if (!more()) return false;
    AttnTile t;
    t.q_row = __shfl_sync(0xffffffffu, word, 0);
    t.row0 = __shfl_sync(0xffffffffu, word, 1);
    t.nrows = __shfl_sync(0xffffffffu, word, 2);
    t.kind = 0;  // (the walk goes over one kind only)
    t.pos0 = __shfl_sync(0xffffffffu, word, 4);
    t.page_at = __shfl_sync(0xffffffffu, word, 5);
    t.blk_lo = __shfl_sync(0xffffffffu, word, 6);
    t.nblk = __shfl_sync(0xffffffffu, word, 7);
    *p = attn_piece(a, t, cur, end, most, &slot);
    if (cur.y + 1 < a.kv_heads) {
      cur = make_int4(cur.x, cur.y + 1, 0, 0);
    } else {
      cur = make_int4(cur.x + 1, 0, 0, 0);
      fetch(a);  // (in good time for the next call)
    }
    return true;
  }
};

// The CTA's share: five times 16 bytes of the plan, read once for all of its threads.
__device__ __forceinline__ void attn_share(const AttnArgs& a, int4* to) {
  if (threadIdx.x < 5) to[threadIdx.x] = reinterpret_cast<const int4*>(a.plan.starts + blockIdx.x)[threadIdx.x];
  __syncthreads();
}

// Cache row (of kv_heads * head_dim elements) of a key, or -1 where its page is not one of the cache's: such a page reads
// as zeros, so that a bad table cannot reach outside.  The value is page_size rows further.
__device__ __forceinline__ int attn_key_row(const AttnArgs& a, int page_at, int key) {
  const int p = a.by_page.div(key);
  const long long at = (long long)page_at + p;
  const int page = at >= 0 && at < a.num_kv_indices ? a.kv_indices[at] : -1;
  return (unsigned)page < (unsigned)a.num_pages ? page * 2 * a.page_size + (key - p * a.page_size) : -1;
}

// The same in two halves, for loads that run ahead: the entry of kv_indices is asked for now (whatever it says is looked at
// later, so that nothing waits for it), the row is made when its turn comes.
struct AttnAhead {
  int page, slot;  // slot < 0: a key that no row sees
  __device__ __forceinline__ void ask(const AttnArgs& a, int page_at, int key, bool seen) {
    const int p = a.by_page.div(max(key, 0));
    const long long at = (long long)page_at + p;
    seen = seen && at >= 0 && at < a.num_kv_indices;
    page = seen ? a.kv_indices[at] : -1;
    slot = seen ? key - p * a.page_size : -1;
  }
  __device__ __forceinline__ int row(const AttnArgs& a) const {
    return slot >= 0 && (unsigned)page < (unsigned)a.num_pages ? page * 2 * a.page_size + slot : -1;
  }
};

// Where row r of a piece's tile goes: (token row, q head).
__host__ __device__ __forceinline__ void attn_row(const AttnArgs& a, const AttnPiece& p, int r, int* token, int* head, int* pos) {
  const int row = p.t.row0 + r, tok = a.by_group.div(row);
  *token = p.t.q_row + tok;
  *head = p.head * a.group + (row - tok * a.group);
  *pos = p.t.pos0 + tok;
}

// Of a sum that came out as zero: nothing to see gives zeros, keys with scores of minus infinity only are 0 / 0.
__device__ __forceinline__ float attn_inverse(float l, int pos) {
  if (l > 0.f || l != l) return 1.f / l;
  return pos < 0 ? 0.f : __int_as_float(0x7fc00000);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

int run_attn_simt(int head_dim, const AttnArgs& a, int workers, cudaStream_t s);
int run_attn_tc(int dtype, int head_dim, const AttnArgs& a, const AttnShape& sh, int workers, cudaStream_t s);

}  // namespace sb200

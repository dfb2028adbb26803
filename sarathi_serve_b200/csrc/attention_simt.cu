// Attention on the FMA pipes: fp32 throughout (the parity configuration wants more than tf32 products).
//
// Many rows: a CTA of 256 threads holds a tile of 64 query rows and walks the keys of its piece 64 (heads of 256: 32) at a time:
// keys and values through shared memory, asked for one step ahead; a thread has 4 rows x 4 keys of the scores and 4 rows x
// HD / 16 columns of the output, so that a load of 16 bytes from shared memory feeds 8 multiply-adds or more (with 1 x 4
// the kernel was bound by those loads: 19 us for 128 keys x 32 rows with heads of 64).
//
// Few rows (a request of up to 8 rows, 4 a unit): bound by HBM.  As in attention_tc.cu the eight warps stream keys in turn, each
// through a ring of its own that asynchronous copies fill; a key belongs to HD / 8 lanes, which hold 8 columns of queries and
// outputs of all four rows in registers, so that a warp works on 1 to 4 keys at a time and reads each byte once.
// (32 decodes of 256 to 2048 tokens and a chunk of 256, heads of 64: 39 us, with tiles of 32 rows only 250.  What bounds it now are the
// chunk's tiles: 6.1 us for 64 rows and 64 keys, a third of the FMA rate.)
#include "attention.cuh"

namespace sb200 {

constexpr int kSimtRows = 64, kSimtThreads = 256;
constexpr int kFew32Rows = 4, kFew32Warps = kSimtThreads / 32, kFew32Stages = 3;

template <int HD> struct Few32 {
  static constexpr int KEYS = 1024 / HD;              // of a step: 4 KB of keys, then their values
  static constexpr int HALF = KEYS * HD * 4;
  static constexpr int RING = kFew32Warps * kFew32Stages * 2 * HALF;
  static constexpr int JOIN = kFew32Warps * kFew32Rows * HD * 4;
  static constexpr int SMEM = RING + JOIN + 2 * kFew32Warps * kFew32Rows * 4;
};

template <int HD> struct Many32 {
  static constexpr int KEYS = HD == 256 ? 32 : 64;
  static constexpr int LD = HD + 4, LDP = kSimtRows + 4;
  static constexpr int SMEM = (kSimtRows * LD + KEYS * LD + KEYS * HD + KEYS * LDP) * 4;
};

template <int HD> constexpr size_t simt_smem() {
  return Many32<HD>::SMEM > Few32<HD>::SMEM ? Many32<HD>::SMEM : Few32<HD>::SMEM;
}

// Writes N (2, 4 or 8) neighbouring columns, from `col` on, of row r of a piece: sums o made with the maximum `base`, l their sum.
template <int HD, int N>
__device__ __forceinline__ void simt_store(const AttnArgs& a, const AttnPiece& p, int r, int col, const float* o, float base, float l, bool first) {
  int token, head, pos;
  attn_row(a, p, r, &token, &head, &pos);
  const bool some = l > 0.f || l != l;
  const float inv = p.slot < 0 ? attn_inverse(l, pos) : some ? 1.f / l : 0.f;
  float* dst = p.slot < 0 ? reinterpret_cast<float*>(a.out) + token * a.ldo + head * HD + col : nullptr;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (p.slot < 0) dst[j] = o[j] * inv;
    else reinterpret_cast<float*>(attn_part(a, HD, p.slot, p.stride, r, (col + j) >> 2))[(col + j) & 3] = o[j] * inv;
  }
  if (first) {
    if (p.slot >= 0) a.part_l[(int64_t)p.slot * a.slot_rows + r] = some ? base + log2f(l) : -INFINITY;
    else if (a.lse) a.lse[(int64_t)token * (a.kv_heads * a.group) + head] = (base + log2f(l)) * 0.69314718055994531f;
  }
}

template <int HD>
__device__ void simt_many(const AttnArgs& a, float* smem, AttnWalk walk) {
  using M = Many32<HD>;
  constexpr int VPR = HD / 4, PER = M::KEYS * VPR / kSimtThreads, KT = M::KEYS / 16, CT = HD / 64;
  float* sq = smem;                        // [64][LD]
  float* sk = sq + kSimtRows * M::LD;      // [KEYS][LD]
  float* sv = sk + M::KEYS * M::LD;        // [KEYS][HD]
  float* sp = sv + M::KEYS * HD;           // [KEYS][LDP]: probabilities, rows side by side
  const int tid = threadIdx.x, rg = tid >> 4, cg = tid & 15;  // rows 4 rg .. + 3; keys cg + 16 i, columns 4 cg + 64 i
  const float* q = reinterpret_cast<const float*>(a.q);
  const float* cache = reinterpret_cast<const float*>(a.cache);
  const int64_t ldc = (int64_t)a.kv_heads * HD;
  // The keys of a piece, as its first warp sees them: every step below waits for all warps (two pieces' in turn: the next one's
  // are written when not all may have read these).
  __shared__ int2 ends[2];
  int turn = 0;
  AttnPiece p;
  while (walk.next(a, &p)) {
    if (tid == 0)
      ends[turn] = make_int2(max(p.lo, (p.t.blk_lo + p.b0) * kAttnBlock) & ~(M::KEYS - 1), min(p.hi, (p.t.blk_lo + p.b1) * kAttnBlock));
    __syncthreads();  // the previous piece has been read
    const int k0 = ends[turn].x, k1 = ends[turn].y;
    turn ^= 1;
    for (int i = tid; i < kSimtRows * VPR; i += kSimtThreads) {
      const int r = i / VPR, v = i - r * VPR;
      int token, head, pos;
      attn_row(a, p, r, &token, &head, &pos);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < p.t.nrows) x = *reinterpret_cast<const float4*>(q + token * a.ldq + head * HD + v * 4);
      *reinterpret_cast<float4*>(sq + r * M::LD + v * 4) = x;
    }
    float m[4], l[4];
    int pos[4];
    float4 acc[4][CT];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int token, head;
      attn_row(a, p, min(rg * 4 + j, max(p.t.nrows - 1, 0)), &token, &head, &pos[j]);
      m[j] = -INFINITY;
      l[j] = 0.f;
#pragma unroll
      for (int i = 0; i < CT; ++i) acc[j][i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const int pos_first = p.t.pos0 + a.by_group.div(p.t.row0), pos_last = p.hi - 1;
    const int warp_lo = __shfl_sync(0xffffffffu, pos[0], 0), warp_hi = __shfl_sync(0xffffffffu, pos[3], 31);  // of the warp's rows
    // Lane l knows the pages of keys l, l + 32 of the step after the next, so that the loads of the next one (this thread's share:
    // next_k, next_v; real: whether its i-th row is one) wait for nothing.
    AttnAhead ahead[M::KEYS / 32];
    float4 next_k[PER], next_v[PER];
    uint32_t real = 0;
    auto look_up = [&](int kb) {
#pragma unroll
      for (int h = 0; h < M::KEYS / 32; ++h) {
        const int key = kb + h * 32 + (tid & 31);
        ahead[h].ask(a, p.t.page_at, key, key >= p.lo && key < k1);
      }
    };
    auto ask = [&]() {
      int rows[M::KEYS / 32];
#pragma unroll
      for (int h = 0; h < M::KEYS / 32; ++h) rows[h] = ahead[h].row(a);
      real = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int j = i * kSimtThreads + tid, r = j / VPR, v = j - r * VPR;
        static_assert(32 % (kSimtThreads / VPR) == 0, "the rows of one i are in one half");
        const int at = __shfl_sync(0xffffffffu, rows[i * (kSimtThreads / VPR) / 32], r & 31);
        if (at >= 0) real |= 1u << i;
        const float* src = cache + (int64_t)max(at, 0) * ldc + p.head * HD + v * 4;
        next_k[i] = *reinterpret_cast<const float4*>(src);
        next_v[i] = *reinterpret_cast<const float4*>(src + a.page_size * ldc);
      }
    };
    if (k0 < k1) {
      look_up(k0);
      ask();
      look_up(k0 + M::KEYS);
    }
    for (int kb = k0; kb < k1; kb += M::KEYS) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int j = i * kSimtThreads + tid, r = j / VPR, v = j - r * VPR;
        const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
        *reinterpret_cast<float4*>(sk + r * M::LD + v * 4) = (real >> i) & 1u ? next_k[i] : none;
        *reinterpret_cast<float4*>(sv + r * HD + v * 4) = (real >> i) & 1u ? next_v[i] : none;
      }
      __syncthreads();
      if (kb + M::KEYS < k1) {
        ask();
        look_up(kb + 2 * M::KEYS);
      }
      float s[4][KT] = {};
#pragma unroll 4
      for (int c = 0; c < HD; c += 4) {
        float4 x[4], y[KT];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const float4*>(sq + (rg * 4 + j) * M::LD + c);
#pragma unroll
        for (int i = 0; i < KT; ++i) y[i] = *reinterpret_cast<const float4*>(sk + (cg + 16 * i) * M::LD + c);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < KT; ++i) s[j][i] += x[j].x * y[i].x + x[j].y * y[i].y + x[j].z * y[i].z + x[j].w * y[i].w;
      }
      const bool all = kb + M::KEYS - 1 <= pos_first && (a.window == 0 || kb > pos_last - a.window);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float top = m[j];
#pragma unroll
        for (int i = 0; i < KT; ++i) {
          const int key = kb + cg + 16 * i;
          s[j][i] *= a.scale_log2;
          if (!all && (key > pos[j] || (a.window > 0 && key <= pos[j] - a.window))) s[j][i] = -INFINITY;
          top = fmaxf(top, s[j][i]);
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float base = top == -INFINITY ? 0.f : top, keep = exp2f(m[j] - base);
        m[j] = top;
        l[j] *= keep;
#pragma unroll
        for (int i = 0; i < KT; ++i) {
          s[j][i] = exp2f(s[j][i] - base);
          l[j] += s[j][i];
        }
#pragma unroll
        for (int i = 0; i < CT; ++i) { acc[j][i].x *= keep; acc[j][i].y *= keep; acc[j][i].z *= keep; acc[j][i].w *= keep; }
      }
#pragma unroll
      for (int i = 0; i < KT; ++i)
        *reinterpret_cast<float4*>(sp + (cg + 16 * i) * M::LDP + rg * 4) = make_float4(s[0][i], s[1][i], s[2][i], s[3][i]);
      __syncwarp();  // the rows of a warp are its own
      // Keys that all rows of the warp see, and around them those that only some see: such a key contributes nothing to the others,
      // whatever its value holds.  (Not: whose probability is 0.  A value that is not finite reaches every row that sees it.)
      // (One by one through every step that has any: the chunk of 256 and 32 decodes of above took 43 us then, not 39.  Eight keys of
      // the middle at a time, not four: 1000 tokens at 2000 447 -> 404 us.)
      const int see = min(M::KEYS, max(0, warp_hi + 1 - kb)), see_lo = a.window > 0 ? min(see, max(0, warp_lo - a.window + 1 - kb)) : 0;
      const int mid = a.window > 0 ? min(see, max(see_lo, warp_hi - a.window + 1 - kb)) : 0, mid_end = min(see, max(mid, warp_lo + 1 - kb));
      const unsigned reach = a.window > 0 ? a.window : 1u << 31;  // a row sees so many keys, from its own on back
      auto one_by_one = [&](int k, int end) {
#pragma unroll 1
        for (; k < end; ++k) {
          const float* w = sp + k * M::LDP + rg * 4;
#pragma unroll
          for (int i = 0; i < CT; ++i) {
            const float4 v = *reinterpret_cast<const float4*>(sv + k * HD + cg * 4 + 64 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float x = w[j];
              if ((unsigned)(pos[j] - kb - k) < reach) { acc[j][i].x += x * v.x; acc[j][i].y += x * v.y; acc[j][i].z += x * v.z; acc[j][i].w += x * v.w; }
            }
          }
        }
      };
      one_by_one(see_lo, mid);
#pragma unroll 8
      for (int k = mid; k < mid_end; ++k) {
        const float4 w = *reinterpret_cast<const float4*>(sp + k * M::LDP + rg * 4);
#pragma unroll
        for (int i = 0; i < CT; ++i) {
          const float4 v = *reinterpret_cast<const float4*>(sv + k * HD + cg * 4 + 64 * i);
          acc[0][i].x += w.x * v.x; acc[0][i].y += w.x * v.y; acc[0][i].z += w.x * v.z; acc[0][i].w += w.x * v.w;
          acc[1][i].x += w.y * v.x; acc[1][i].y += w.y * v.y; acc[1][i].z += w.y * v.z; acc[1][i].w += w.y * v.w;
          acc[2][i].x += w.z * v.x; acc[2][i].y += w.z * v.y; acc[2][i].z += w.z * v.z; acc[2][i].w += w.z * v.w;
          acc[3][i].x += w.w * v.x; acc[3][i].y += w.w * v.y; acc[3][i].z += w.w * v.z; acc[3][i].w += w.w * v.w;
        }
      }
      one_by_one(mid_end, see);
      __syncwarp();
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], o);
      const int r = rg * 4 + j;
      if (r < p.t.nrows)
#pragma unroll
        for (int i = 0; i < CT; ++i)
          simt_store<HD, 4>(a, p, r, i * 64 + cg * 4, reinterpret_cast<const float*>(&acc[j][i]), m[j] == -INFINITY ? 0.f : m[j], l[j], i == 0 && cg == 0);
    }
  }
}

// The steps of a warp, for the loads and for the sums alike.
template <int HD> struct Few32Steps {
  AttnWalk walk;
  AttnPiece p;
  int key, end;
  __device__ __forceinline__ explicit Few32Steps(const AttnWalk& w) : walk(w), key(0), end(0) {}
  __device__ __forceinline__ bool next_piece(const AttnArgs& a, int warp) {
    if (!walk.next(a, &p)) return false;
    constexpr int K = Few32<HD>::KEYS;
    key = (max(p.lo, (p.t.blk_lo + p.b0) * kAttnBlock) & ~(K - 1)) + warp * K;
    end = min(p.hi, (p.t.blk_lo + p.b1) * kAttnBlock);
    return true;
  }
};

template <int HD>
__device__ void simt_few(const AttnArgs& a, float* smem, const AttnWalk& walk) {
  using F = Few32<HD>;
  constexpr int R = kFew32Rows, LPK = HD / 8, KPW = 32 / LPK, CPR = HD / 4, kStep = kFew32Warps * F::KEYS;
  static_assert(F::KEYS == 4 * KPW, "a step is four turns of the warp");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % LPK, mine = lane / LPK;
  uint8_t* bytes = reinterpret_cast<uint8_t*>(smem);
  float* ring = reinterpret_cast<float*>(bytes + warp * (kFew32Stages * 2 * F::HALF));
  float* join = reinterpret_cast<float*>(bytes + F::RING);                // [warp][row][HD]
  float* stat_m = reinterpret_cast<float*>(bytes + F::RING + F::JOIN);    // [warp][row]
  float* stat_l = stat_m + kFew32Warps * R;
  const float* cache = reinterpret_cast<const float*>(a.cache);
  const int64_t ldc = (int64_t)a.kv_heads * HD;

  Few32Steps<HD> ld(walk);
  bool more = true;
  AttnAhead next;
  int head_next = 0, put = 0;
  auto look_up = [&]() {  // lane i: the page of key i of the step after the next
    while (more && ld.key >= ld.end) more = ld.next_piece(a, warp);
    if (!more) return;
    const int key = ld.key + lane % F::KEYS;
    next.ask(a, ld.p.t.page_at, key, key >= ld.p.lo && key < ld.p.hi);
    head_next = ld.p.head;
    ld.key += kStep;
  };
  auto load = [&]() {
    if (more) {
      const int rows = next.row(a), head = head_next;
      const uint32_t dst = ptx::smem_u32(ring) + put * (2 * F::HALF);
#pragma unroll
      for (int i = 0; i < F::KEYS * CPR / 32; ++i) {
        const int c = i * 32 + lane, k = c / CPR, row = __shfl_sync(0xffffffffu, rows, k);
        const float* src = cache + (int64_t)max(row, 0) * ldc + head * HD + (c % CPR) * 4;
        cp_async16(dst + c * 16, src, row >= 0);
        cp_async16(dst + F::HALF + c * 16, src + (row >= 0 ? a.page_size * ldc : 0), row >= 0);
      }
      if (++put == kFew32Stages) put = 0;
      look_up();
    }
    cp_async_commit();
  };
  look_up();
#pragma unroll 1
  for (int i = 0; i < kFew32Stages - 1; ++i) load();

  Few32Steps<HD> st(walk);
  int get = 0;
  while (st.next_piece(a, warp)) {
    const AttnPiece& p = st.p;
    float4 q[R][2], o[R][2];
    float m[R], l[R];
    int pos[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      int token, head;
      attn_row(a, p, min(r, max(p.t.nrows - 1, 0)), &token, &head, &pos[r]);
      const float* src = reinterpret_cast<const float*>(a.q) + token * a.ldq + head * HD + sub * 4;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        q[r][h] = o[r][h] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < p.t.nrows) q[r][h] = *reinterpret_cast<const float4*>(src + h * (HD / 2));
      }
      m[r] = -INFINITY;
      l[r] = 0.f;
    }
    const int pos_first = p.t.pos0 + a.by_group.div(p.t.row0), pos_last = p.hi - 1;
    for (; st.key < st.end; st.key += kStep) {
      load();
      cp_async_wait<kFew32Stages - 1>();
      __syncwarp();
      const float* sk = ring + get * (2 * F::HALF / 4) + mine * HD + sub * 4;
      const float* sv = sk + F::HALF / 4;
      if (++get == kFew32Stages) get = 0;
      const bool all = st.key + F::KEYS - 1 <= pos_first && (a.window == 0 || st.key > pos_last - a.window);
      float s[4][R];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float4 x = *reinterpret_cast<const float4*>(sk + t * KPW * HD), y = *reinterpret_cast<const float4*>(sk + t * KPW * HD + HD / 2);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float d = q[r][0].x * x.x + q[r][0].y * x.y + q[r][0].z * x.z + q[r][0].w * x.w;
          d += q[r][1].x * y.x + q[r][1].y * y.y + q[r][1].z * y.z + q[r][1].w * y.w;
          s[t][r] = d;
        }
      }
#pragma unroll
      for (int x = 1; x < LPK; x <<= 1)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int r = 0; r < R; ++r) s[t][r] += __shfl_xor_sync(0xffffffffu, s[t][r], x);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float top = m[r];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          s[t][r] *= a.scale_log2;
          const int key = st.key + t * KPW + mine;
          if (!all && (key > pos[r] || (a.window > 0 && key <= pos[r] - a.window))) s[t][r] = -INFINITY;
          top = fmaxf(top, s[t][r]);
        }
        const float base = top == -INFINITY ? 0.f : top, keep = exp2f(m[r] - base);
        m[r] = top;
        l[r] *= keep;
#pragma unroll
        for (int h = 0; h < 2; ++h) { o[r][h].x *= keep; o[r][h].y *= keep; o[r][h].z *= keep; o[r][h].w *= keep; }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          s[t][r] = exp2f(s[t][r] - base);
          l[r] += s[t][r];
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float4 x = *reinterpret_cast<const float4*>(sv + t * KPW * HD), y = *reinterpret_cast<const float4*>(sv + t * KPW * HD + HD / 2);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float w = s[t][r];
          const int key = st.key + t * KPW + mine;
          if (all || (key <= pos[r] && (a.window == 0 || key > pos[r] - a.window))) {  // a key that the row does not see contributes nothing, whatever its value holds
            o[r][0].x += w * x.x; o[r][0].y += w * x.y; o[r][0].z += w * x.z; o[r][0].w += w * x.w;
            o[r][1].x += w * y.x; o[r][1].y += w * y.y; o[r][1].z += w * y.z; o[r][1].w += w * y.w;
          }
        }
      }
      __syncwarp();  // the stage may be filled again
    }
    // ---- join: the lanes of a warp that have the same columns, then the warps
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = m[r];
#pragma unroll
      for (int x = LPK; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float keep = m[r] == -INFINITY ? 0.f : exp2f(m[r] - top);
      m[r] = top;
      l[r] *= keep;
      float* v[8] = {&o[r][0].x, &o[r][0].y, &o[r][0].z, &o[r][0].w, &o[r][1].x, &o[r][1].y, &o[r][1].z, &o[r][1].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) *v[e] *= keep;
#pragma unroll
      for (int x = LPK; x < 32; x <<= 1) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) *v[e] += __shfl_xor_sync(0xffffffffu, *v[e], x);
      }
      if (mine == 0) {
        *reinterpret_cast<float4*>(join + (warp * R + r) * HD + sub * 4) = o[r][0];
        *reinterpret_cast<float4*>(join + (warp * R + r) * HD + HD / 2 + sub * 4) = o[r][1];
      }
      if (lane == 0) { stat_m[warp * R + r] = m[r]; stat_l[warp * R + r] = l[r]; }
    }
    __syncthreads();
    if (warp < p.t.nrows) {
      constexpr int N = HD / 32;
      float top = -INFINITY, sum = 0.f, acc[N] = {};
#pragma unroll
      for (int w = 0; w < kFew32Warps; ++w) top = fmaxf(top, stat_m[w * R + warp]);
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int w = 0; w < kFew32Warps; ++w) {
        const float mw = stat_m[w * R + warp], f = mw == -INFINITY ? 0.f : exp2f(mw - base);
        sum += f * stat_l[w * R + warp];
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] += f * join[(w * R + warp) * HD + lane * N + j];
      }
      simt_store<HD, N>(a, p, warp, lane * N, acc, base, sum, lane == 0);
    }
    __syncthreads();
  }
  cp_async_wait<0>();
}

// One CTA per SM: its share's tiles of many rows first, then those of few.
template <int HD>
__global__ void __launch_bounds__(kSimtThreads, 1)
attn_simt_kernel(const __grid_constant__ AttnArgs a) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();  // (the join reads the plan at once)
  extern __shared__ float smem_f[];
  __shared__ int4 share[5];
  attn_share(a, share);
  AttnWalk walk(a, share), few = walk;
  walk.only_many(a);
  simt_many<HD>(a, smem_f, walk);
  __syncthreads();
  few.only_few(a);
  simt_few<HD>(a, smem_f, few);
}

template <int HD>
static int launch_simt(const AttnArgs& a, int workers, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  SB_CUDA(allow_smem(reinterpret_cast<const void*>(attn_simt_kernel<HD>), (int)simt_smem<HD>(), &allowed));
  auto kern = attn_simt_kernel<HD>;  // (waits for its predecessor by hand)
  SB_CUDA(launch_dependent(kern, dim3((unsigned)workers), dim3(kSimtThreads), simt_smem<HD>(), s, a));
  return SB200_OK;
}

int run_attn_simt(int head_dim, const AttnArgs& a, int workers, cudaStream_t s) {
  return head_dim == 64 ? launch_simt<64>(a, workers, s) : head_dim == 128 ? launch_simt<128>(a, workers, s) : launch_simt<256>(a, workers, s);
}

}  // namespace sb200

// Attention of fp16 / bf16 steps on the tensor cores.
//
// Few rows (a decoded token of a group of heads, a chunk of a handful of tokens: up to 16 rows a unit).  Every key and
// value is read once for at most 16 rows, 4 FLOP a byte and row: bound by HBM, far below what any tensor instruction asks
// for, so the products are warp-wide m16n8k16 with the rows as M, and everything is arranged for loads in flight.  The
// eight warps of a CTA take 16 keys each in turn and own a ring of three steps apiece in shared memory, filled by
// 16-byte asynchronous copies: no barrier between them while they stream, and 128 to 192 KB in flight per SM.  A warp keeps
// its own running maximum, sum and output; they are joined once a piece.  Its loads run ahead into the next piece.
//
// Many rows (prompt chunks): tiles of 256 rows on tcgen05, see "many rows" below.
#include "attention.cuh"
#include "gemm_host.cuh"

namespace sb200 {

constexpr int kFewRows = 16, kFewKeys = 16;

template <int HD> struct Few {
  static constexpr int WARPS = HD == 256 ? 4 : 8;
  static constexpr int STAGES = HD == 64 ? 6 : 3;
  static constexpr int ROW = HD * 2;                    // bytes of a key
  static constexpr int HALF = kFewKeys * ROW;           // the keys of a step; its values follow
  static constexpr int RING = WARPS * STAGES * 2 * HALF;
  static constexpr int JOIN_ROWS = 8;                   // rows that the warps hand over at a time
  static constexpr int JOIN = WARPS * JOIN_ROWS * HD * 4;
  static constexpr int STATS = 2 * WARPS * kFewRows * 4;
  static constexpr int SMEM = RING + JOIN + STATS;
};

// ------------------------------------------------------------------ warp-wide pieces
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// `ex2.approx`: relative error 2^-22, 2^-inf = 0.
__device__ __forceinline__ float pow2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (DT<T>::id == SB200_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// N times four 8 x 8 matrices; addr(i) is this lane's row address of load i.
template <int N, bool TRANS, typename F> __device__ __forceinline__ void load_matrices(uint32_t (&r)[N][4], F addr) {
  __syncwarp();
#define SB_LDMATRIX(KIND) "ldmatrix.sync.aligned.m8n8.x4" KIND ".shared.b16 {%0, %1, %2, %3}, [%4];"
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (TRANS)
      asm volatile(SB_LDMATRIX(".trans") : "=r"(r[i][0]), "=r"(r[i][1]), "=r"(r[i][2]), "=r"(r[i][3]) : "r"(addr(i)) : "memory");
    else
      asm volatile(SB_LDMATRIX("") : "=r"(r[i][0]), "=r"(r[i][1]), "=r"(r[i][2]), "=r"(r[i][3]) : "r"(addr(i)) : "memory");
  }
#undef SB_LDMATRIX
}

// c(i) += a(i) * b(i) for N products of 16 x 16 by 16 x 8: `step(i, &c, &a, &b)` names the registers of product i.
template <typename T, int N, typename F> __device__ __forceinline__ void multiply(F step) {
  __syncwarp();
#define SB_MMA(TY) "mma.sync.aligned.m16n8k16.row.col.f32." TY "." TY ".f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float* c;
    const uint32_t *a, *b;
    step(i, &c, &a, &b);
    if constexpr (DT<T>::id == SB200_BF16)
      asm volatile(SB_MMA("bf16") : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                   : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
    else
      asm volatile(SB_MMA("f16") : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                   : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  }
#undef SB_MMA
}

// Barrier of the warps that compute.
__device__ __forceinline__ void few_barrier(int threads) {
  __syncwarp();
  asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
}

// A maximum is replaced only when the new one is this much larger (in powers of two): until then probabilities grow to at most
// 2^8, which 16 bits hold as well as numbers below 1, and the output need not be rescaled.
constexpr float kLazy = 8.f;

// One row's output recomputed key by key: what a product with P = 0 cannot do is to leave out a value that is not finite.
// Called by a warp for a row whose output came out not finite; m is the maximum that the row's sum l was made with.
template <typename T, int HD>
__device__ __noinline__ void attn_repair_row(const AttnArgs& a, const AttnPiece& p, int r, float m, float* o) {
  constexpr int N = HD / 32;
  const int lane = threadIdx.x & 31;
  int token, head, pos;
  attn_row(a, p, r, &token, &head, &pos);
  const T* q = reinterpret_cast<const T*>(a.q) + token * a.ldq + head * HD + lane * N;
  const T* cache = reinterpret_cast<const T*>(a.cache) + p.head * HD + lane * N;
  const int64_t ldc = (int64_t)a.kv_heads * HD;
  float x[N];
#pragma unroll
  for (int j = 0; j < N; ++j) { x[j] = DT<T>::to_f(q[j]); o[j] = 0.f; }
  const int k0 = max(a.window > 0 ? max(0, pos + 1 - a.window) : 0, (p.t.blk_lo + p.b0) * kAttnBlock);
  const int k1 = min(pos + 1, (p.t.blk_lo + p.b1) * kAttnBlock);
  for (int key = k0; key < k1; ++key) {
    const int at = attn_key_row(a, p.t.page_at, key);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) s += at >= 0 ? x[j] * DT<T>::to_f(cache[at * ldc + j]) : x[j] * 0.f;
    s = warp_sum(s);
    const float pr = DT<T>::to_f(DT<T>::from_f(pow2(s * a.scale_log2 - m)));
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] += pr * (at >= 0 ? DT<T>::to_f(cache[(at + a.page_size) * ldc + j]) : 0.f);
  }
}

// The steps of 16 keys that a warp loads (or computes) for the pieces of its CTA's share, one after the other.
template <int HD> struct FewSteps {
  AttnWalk walk;
  AttnPiece p;
  int key, end;   // next step of the current piece, and where it ends
  __device__ __forceinline__ FewSteps(const AttnArgs& a, int worker) : walk(a, worker), key(0), end(0) { walk.from(a.plan.header[3]); }
  __device__ __forceinline__ bool next_piece(const AttnArgs& a, int warp) {
    if (!walk.next(a, &p)) return false;
    key = (max(p.lo, (p.t.blk_lo + p.b0) * kAttnBlock) & ~(kFewKeys - 1)) + warp * kFewKeys;
    end = min(p.hi, (p.t.blk_lo + p.b1) * kAttnBlock);
    return true;
  }
};

template <typename T, int HD>
__device__ void few_share(const AttnArgs& a, uint8_t* smem, int worker) {
  using F = Few<HD>;
  constexpr int CPR = HD / 8;              // 16-byte pieces of a key
  constexpr int KPI = 32 / CPR > 0 ? 32 / CPR : 1;  // keys that one copy instruction of the warp covers
  constexpr int IPK = CPR > 32 ? CPR / 32 : 1;
  static_assert(IPK == 1, "a key is at most 32 pieces");
  constexpr int KS = HD / 16, NT = HD / 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const uint32_t ring = ptx::smem_u32(smem) + warp * (F::STAGES * 2 * F::HALF);
  float* join = reinterpret_cast<float*>(smem + F::RING);               // [warp][row of a pass][HD]
  float* stat_m = reinterpret_cast<float*>(smem + F::RING + F::JOIN);   // [warp][16]
  float* stat_l = stat_m + F::WARPS * kFewRows;
  const T* cache = reinterpret_cast<const T*>(a.cache);
  const int64_t ldc = (int64_t)a.kv_heads * HD;
  constexpr int kStep = F::WARPS * kFewKeys;

  // loads: one step ahead of the copies runs the look-up of the keys' rows (lane i: key i of the step)
  FewSteps<HD> ld(a, worker);
  bool more = true;
  int row_next = -1, head_next = 0;
  auto look_up = [&]() {
    while (more && ld.key >= ld.end) more = ld.next_piece(a, warp);
    if (!more) return;
    const int key = ld.key + (lane & 15);
    row_next = key >= ld.p.lo && key < ld.p.hi ? attn_key_row(a, ld.p.t.page_at, key) : -1;
    head_next = ld.p.head;
    ld.key += kStep;
  };
  int put = 0;
  auto load = [&]() {
    if (more) {
      const int rows = row_next, head = head_next;
      const uint32_t dst = ring + put * (2 * F::HALF);
      const int sub = lane / CPR, chunk = lane % CPR;
#pragma unroll
      for (int i = 0; i < kFewKeys / KPI; ++i) {
        const int k = i * KPI + sub, row = __shfl_sync(0xffffffffu, rows, k);
        const T* src = cache + (int64_t)max(row, 0) * ldc + head * HD + chunk * 8;
        const uint32_t at = dst + k * F::ROW + ((chunk ^ (k & 7)) << 4);
        cp_async16(at, src, row >= 0);
        cp_async16(at + F::HALF, src + (row >= 0 ? a.page_size * ldc : 0), row >= 0);
      }
      if (++put == F::STAGES) put = 0;
      look_up();
    }
    cp_async_commit();
  };
  look_up();
#pragma unroll 1
  for (int i = 0; i < F::STAGES - 1; ++i) load();

  FewSteps<HD> st(a, worker);
  int get = 0;
  while (st.next_piece(a, warp)) {
    const AttnPiece& p = st.p;
    // query rows as the A operand: rows g and g + 8, columns 2 t and 2 t + 8 of every 16
    uint32_t qf[KS][4];
    int pos_lo, pos_hi;
    {
      int token, head;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = g + 8 * half;
        attn_row(a, p, min(r, max(p.t.nrows - 1, 0)), &token, &head, half ? &pos_hi : &pos_lo);
        const T* src = reinterpret_cast<const T*>(a.q) + token * a.ldq + head * HD + 2 * t4;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            qf[k][half + 2 * c] = r < p.t.nrows ? *reinterpret_cast<const uint32_t*>(src + k * 16 + c * 8) : 0u;
      }
    }
    const int pos_first = p.t.pos0 + p.t.row0 / a.group, pos_last = p.hi - 1;
    float o[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) { o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f; }
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;  // rows g and g + 8
    for (; st.key < st.end; st.key += kStep) {
      load();
      cp_async_wait<F::STAGES - 1>();
      __syncwarp();
      const uint32_t sk = ring + get * (2 * F::HALF), sv = sk + F::HALF;
      if (++get == F::STAGES) get = 0;
      float s[2][4] = {};
      {
        const int r = ((lane >> 4) << 3) + (lane & 7), c = (lane >> 3) & 1;
#pragma unroll
        for (int k0 = 0; k0 < KS; k0 += 4) {
          constexpr int KB = 4;
          uint32_t kf[KB][4];
          load_matrices<KB, false>(kf, [&](int k) { return sk + r * F::ROW + ((((k0 + k) * 2 + c) ^ (r & 7)) << 4); });
          multiply<T, 2 * KB>([&](int i, float** cc, const uint32_t** aa, const uint32_t** bb) {
            *cc = s[i & 1]; *aa = qf[k0 + (i >> 1)]; *bb = &kf[i >> 1][2 * (i & 1)];
          });
        }
      }
      const int key = st.key + 2 * t4;
      const bool all = st.key + kFewKeys - 1 <= pos_first && (a.window == 0 || st.key > pos_last - a.window);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[n][e] *= a.scale_log2;
          s[n][2 + e] *= a.scale_log2;
          if (!all) {
            const int j = key + n * 8 + e;
            if (j > pos_lo || (a.window > 0 && j <= pos_lo - a.window)) s[n][e] = -INFINITY;
            if (j > pos_hi || (a.window > 0 && j <= pos_hi - a.window)) s[n][2 + e] = -INFINITY;
          }
        }
      float t0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
      float t1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
#pragma unroll
      for (int x = 1; x < 4; x <<= 1) {
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, x));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, x));
      }
      const bool grow = t0 > m0 + kLazy || t1 > m1 + kLazy || (m0 == -INFINITY && t0 > m0) || (m1 == -INFINITY && t1 > m1);
      if (__any_sync(0xffffffffu, grow)) {
        const float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1);
        const float f0 = m0 == -INFINITY ? 0.f : pow2(m0 - n0), f1 = m1 == -INFINITY ? 0.f : pow2(m1 - n1);
        m0 = n0; m1 = n1;
        l0 *= f0; l1 *= f1;
#pragma unroll
        for (int i = 0; i < NT; ++i) { o[i][0] *= f0; o[i][1] *= f0; o[i][2] *= f1; o[i][3] *= f1; }
      }
      const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
      uint32_t pf[4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float x0 = pow2(s[n][0] - b0), x1 = pow2(s[n][1] - b0), x2 = pow2(s[n][2] - b1), x3 = pow2(s[n][3] - b1);
        l0 += x0 + x1;
        l1 += x2 + x3;
        pf[2 * n] = pack2<T>(x0, x1);
        pf[2 * n + 1] = pack2<T>(x2, x3);
      }
      {
        const int r = (((lane >> 3) & 1) << 3) + (lane & 7), c = lane >> 4;
#pragma unroll
        for (int n0 = 0; n0 < NT; n0 += 8) {
          constexpr int NB = 8;
          uint32_t vf[NB / 2][4];
          load_matrices<NB / 2, true>(vf, [&](int n) { return sv + r * F::ROW + (((n0 + n * 2 + c) ^ (r & 7)) << 4); });
          multiply<T, NB>([&](int i, float** cc, const uint32_t** aa, const uint32_t** bb) {
            *cc = o[n0 + i]; *aa = pf; *bb = &vf[i >> 1][2 * (i & 1)];
          });
        }
      }
      __syncwarp();  // the stage may be filled again
    }
    // ---------------------------------------------------------------- join the warps
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, x);
      l1 += __shfl_xor_sync(0xffffffffu, l1, x);
    }
    if (t4 == 0) {
      stat_m[warp * kFewRows + g] = m0; stat_m[warp * kFewRows + g + 8] = m1;
      stat_l[warp * kFewRows + g] = l0; stat_l[warp * kFewRows + g + 8] = l1;
    }
    static_assert(F::JOIN_ROWS == 8, "rows g, then rows g + 8");
    for (int pass = 0; pass * 8 < max(p.t.nrows, 1); ++pass) {
      if (pass * 8 + g < p.t.nrows) {
        float* dst = join + (warp * 8 + g) * HD + 2 * t4;
#pragma unroll
        for (int i = 0; i < NT; ++i)
          *reinterpret_cast<float2*>(dst + i * 8) = pass ? make_float2(o[i][2], o[i][3]) : make_float2(o[i][0], o[i][1]);
      }
      few_barrier(F::WARPS * 32);
      const int rows = min(8, p.t.nrows - pass * 8);
      constexpr int N = HD / 32;
      for (int rr = warp; rr < rows; rr += F::WARPS) {  // a warp per row, N columns a lane
        const int r = pass * 8 + rr;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < F::WARPS; ++w) m = fmaxf(m, stat_m[w * kFewRows + r]);
        const float base = m == -INFINITY ? 0.f : m;
        float l = 0.f, acc[N] = {};
#pragma unroll
        for (int w = 0; w < F::WARPS; ++w) {
          const float mw = stat_m[w * kFewRows + r];
          if (mw == -INFINITY) { l += stat_l[w * kFewRows + r]; continue; }
          const float f = pow2(mw - base);
          l += f * stat_l[w * kFewRows + r];
#pragma unroll
          for (int j = 0; j < N; ++j) acc[j] += f * join[(w * 8 + rr) * HD + lane * N + j];
        }
        bool fine = true;
#pragma unroll
        for (int j = 0; j < N; ++j) fine = fine && fabsf(acc[j]) < INFINITY;
        if (!__all_sync(0xffffffffu, fine)) attn_repair_row<T, HD>(a, p, r, base, acc);
        int token, head, pos;
        attn_row(a, p, r, &token, &head, &pos);
        if (p.slot < 0) {
          const float inv = attn_inverse(l, pos);
          T* dst = reinterpret_cast<T*>(a.out) + token * a.ldo + head * HD + lane * N;
#pragma unroll
          for (int j = 0; j < N; j += 2) *reinterpret_cast<uint32_t*>(dst + j) = pack2<T>(acc[j] * inv, acc[j + 1] * inv);
          if (a.lse && lane == 0) a.lse[(int64_t)token * (a.kv_heads * a.group) + head] = (base + log2f(l)) * 0.69314718055994531f;
        } else {
          const bool some = l > 0.f || l != l;
          const float inv = some ? 1.f / l : 0.f;
          const int64_t at = (int64_t)p.slot * a.slot_rows + r;
#pragma unroll
          for (int j = 0; j < N; ++j) a.part_o[at * HD + lane * N + j] = acc[j] * inv;
          if (lane == 0) a.part_l[at] = some ? base + log2f(l) : -INFINITY;
        }
      }
      few_barrier(F::WARPS * 32);  // the rows (and the statistics) may be written again
    }
  }
  cp_async_wait<0>();
}

// ------------------------------------------------------------------ many rows
// A tile of 256 query rows in two halves A and B of 128, keys in blocks of 128, both products on tcgen05:
//   S = Q K^T     both operands in shared memory, K-major
//   O += P V      P (16 bits) in TMEM where S was, V in shared memory as it lies in the cache (its rows are the K side)
// TMEM holds S / P of both halves (2 x 128 columns) and O of both (2 x HD).  Warps 0-3 make the probabilities of half A,
// warps 4-7 those of B, a row per thread; warp 8 issues the products, warp 9 the loads.  While the tensor pipe works for one
// half, the other half's warps turn S into P; products of one half are issued back to back (P V of a block, then S of the
// next), so that S needs no second buffer.  The maximum moves only when it has grown by 2^8 (kLazy), so O is hardly ever rescaled,
// and then by the warps that found out: S of a block is complete after O of the one before it.
// Bound: 4 HD FLOP and one exponential a (row, key): 1024 + 1024 clocks of the tensor pipe a block of both halves with
// HD = 128, and 2048 of the exponential unit (16 a clock and SM), side by side.
// Keys and values come a page per box (128-byte swizzle), whatever the page: 8 rows and up.  Pages outside the cache
// are fetched from behind its end, which fills zeros.  Values of keys that no row of the tile sees (behind the last, before the
// window) are cleared in shared memory, as 0 x NaN is not 0; rows that meet one all the same are recomputed (attn_repair_row).
template <int HD> struct Many {
  static constexpr int HALVES = HD / 64;
  static constexpr int BOX = 128 * 128;             // bytes of 128 rows x 64 columns
  static constexpr int TILE = HALVES * BOX;         // 128 rows
  static constexpr int STAGES = HD == 128 ? 5 : 8;  // blocks of keys or values
  static constexpr int SMEM = (2 + STAGES) * TILE;
};

struct ManySync {
  uint64_t full[8], empty[8], q_full[2], s_full[2], p_full[2], o_full[2], drain;
  uint32_t tmem;
  int abort_word;
};

template <int HD>
__device__ __forceinline__ void many_load(const AttnArgs& a, const CUtensorMap* map, uint8_t* smem, ManySync& sy, AttnWalk walk) {
  using M = Many<HD>;
  const int lane = threadIdx.x & 31;
  volatile int* abort_flag = &sy.abort_word;
  const int box = min(a.page_size, kAttnBlock), boxes = kAttnBlock / box;
  const int none = a.num_pages * 2 * a.page_size;  // the first row behind the cache
  int stage = 0, filled = 0;
  uint32_t phase = 0;
  bool ok = true;
  AttnPiece p;
  while (ok && walk.next(a, &p)) {
    for (int b = p.b0; ok && b < p.b1; ++b) {
      const int key0 = (p.t.blk_lo + b) * kAttnBlock;
      const int key = key0 + lane * box;   // lane i: box i of the block
      const bool want = lane < boxes && key < p.hi && key + box > p.lo;
      int row = -1;
      if (want) row = attn_key_row(a, p.t.page_at, key);
      const uint32_t mask = __ballot_sync(0xffffffffu, want);
#pragma unroll 1
      for (int v = 0; ok && v < 2; ++v) {
        ok = ptx::mbar_wait_warp(&sy.empty[stage], phase ^ 1u, abort_flag);
        if (!ok) break;
        uint8_t* dst = smem + (2 + stage) * M::TILE;
        const int at = row < 0 ? none : row + v * a.page_size;
        if (ptx::elect_one()) ptx::mbar_expect_tx(&sy.full[stage], (uint32_t)(__popc(mask) * box * HD * 2));
        __syncwarp();
        for (int i = 0; i < boxes; ++i) {
          const int r = __shfl_sync(0xffffffffu, at, i);
          if ((mask >> i) & 1u) {
            if (ptx::elect_one()) {
#pragma unroll
              for (int h = 0; h < M::HALVES; ++h)
                ptx::tma_load_2d(dst + h * M::BOX + i * box * 128, map, &sy.full[stage], p.head * HD + h * 64, r);
            }
            __syncwarp();
          }
        }
        ++filled;
        if (++stage == M::STAGES) { stage = 0; phase ^= 1u; }
      }
    }
  }
  if (!ok) {
    // given up: wait (with a limit) for the copies that are still on their way before the CTA may end
    __shared__ int never;
    if (lane == 0) never = 0;
    __syncwarp();
    for (int i = max(0, filled - M::STAGES); i < filled; ++i) ptx::mbar_wait_warp(&sy.full[i % M::STAGES], (uint32_t)(i / M::STAGES) & 1u, &never);
  }
}

template <typename T, int HD>
__device__ __forceinline__ void many_multiply(const AttnArgs& a, uint8_t* smem, ManySync& sy, AttnWalk walk) {
  using M = Many<HD>;
  const int lane = threadIdx.x & 31;
  volatile int* abort_flag = &sy.abort_word;
  constexpr int fmt = DT<T>::id == SB200_BF16 ? 1 : 0;
  const uint32_t id_s = ptx::make_idesc(fmt, 128), id_o = ptx::make_idesc(fmt, HD) | ptx::kIdescBRows;
  const uint32_t tmem = sy.tmem, sq = ptx::smem_u32(smem), kv = sq + 2 * M::TILE;
  auto scores = [&](int sub, int stage) {  // S of half `sub` with the keys in `stage`
    if (ptx::elect_one()) {
      const uint64_t dq = ptx::make_smem_desc_sw128(sq + sub * M::TILE), dk = ptx::make_smem_desc_sw128(kv + stage * M::TILE);
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        const uint64_t off = (uint64_t)((k >> 2) * (M::BOX >> 4) + (k & 3) * 2);
        ptx::umma_f16(tmem + sub * 128, dq + off, dk + off, id_s, k > 0 ? 1u : 0u);
      }
      ptx::umma_commit(&sy.s_full[sub]);
    }
    __syncwarp();
  };
  auto output = [&](int sub, int stage, bool first) {
    if (ptx::elect_one()) {
      const uint64_t dv = ptx::make_smem_desc_rows_sw128(kv + stage * M::TILE, M::BOX);
#pragma unroll
      for (int k = 0; k < kAttnBlock / 16; ++k)
        ptx::umma_f16_ts(tmem + 256 + sub * HD, tmem + sub * 128 + k * 8, dv + (uint64_t)(k * (16 * 128 >> 4)), id_o, !first || k > 0 ? 1u : 0u);
    }
    __syncwarp();
  };
  auto release = [&](int stage) {
    if (ptx::elect_one()) ptx::umma_commit(&sy.empty[stage]);
    __syncwarp();
  };
  int stage = 0;
  uint32_t phase = 0, pieces[2] = {0, 0}, blocks[2] = {0, 0};
  auto wait_full = [&]() {
    const bool ok = ptx::mbar_wait_warp(&sy.full[stage], phase, abort_flag);
    ptx::tc_fence_after();
    return ok;
  };
  auto advance = [&]() { if (++stage == M::STAGES) { stage = 0; phase ^= 1u; } };
  bool ok = true;
  AttnPiece p;
  while (ok && walk.next(a, &p)) {
    if (p.b0 >= p.b1) continue;
    const int subs = p.t.nrows > 128 ? 2 : 1;
    ok = wait_full();
    for (int s = 0; ok && s < subs; ++s) {
      ok = ptx::mbar_wait_warp(&sy.q_full[s], pieces[s]++ & 1u, abort_flag);
      ptx::tc_fence_after();
      if (ok) scores(s, stage);
    }
    if (!ok) break;
    release(stage);
    advance();
    for (int b = p.b0; ok && b < p.b1; ++b) {
      const int vs = stage;
      int ks = vs;
      for (int s = 0; ok && s < subs; ++s) {
        if (s == 0) {
          ok = wait_full();
          if (!ok) break;
          // values that no row sees
          const int key0 = (p.t.blk_lo + b) * kAttnBlock, lo = max(0, min(128, p.lo - key0)), hi = max(0, min(128, p.hi - key0));
          if (lo > 0 || hi < 128) {
            uint8_t* v = smem + (2 + vs) * M::TILE;
            for (int i = lane; i < 128 * 8; i += 32) {
              const int r = i >> 3;
              if (r < lo || r >= hi)
#pragma unroll
                for (int h = 0; h < M::HALVES; ++h) *reinterpret_cast<uint4*>(v + h * M::BOX + i * 16) = make_uint4(0, 0, 0, 0);
            }
            ptx::fence_proxy_async_smem();
            __syncwarp();
          }
          advance();
        }
        ok = ptx::mbar_wait_warp(&sy.p_full[s], blocks[s]++ & 1u, abort_flag);
        if (!ok) break;
        ptx::tc_fence_after();
        output(s, vs, b == p.b0);
        if (b + 1 < p.b1) {
          if (s == 0) {
            ok = wait_full();
            if (!ok) break;
            ks = stage;
            advance();
          }
          scores(s, ks);
        } else {
          if (ptx::elect_one()) ptx::umma_commit(&sy.o_full[s]);
          __syncwarp();
        }
      }
      if (!ok) break;
      release(vs);
      if (b + 1 < p.b1) release(ks);
    }
  }
  if (!ok) {  // given up: what has been issued may still read shared memory and write TMEM
    __shared__ int never;
    if (lane == 0) never = 0;
    __syncwarp();
    if (ptx::elect_one()) ptx::umma_commit(&sy.drain);
    ptx::mbar_wait_warp(&sy.drain, 0u, &never);
  }
}

template <typename T, int HD>
__device__ __forceinline__ void many_softmax(const AttnArgs& a, uint8_t* smem, ManySync& sy, AttnWalk walk) {
  using M = Many<HD>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp >> 2, quarter = warp & 3;
  const int r = sub * 128 + quarter * 32 + lane;  // this thread's row of the tile
  volatile int* abort_flag = &sy.abort_word;
  const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
  const uint32_t t_s = sy.tmem + sub * 128 + lanes, t_o = sy.tmem + 256 + sub * HD + lanes;
  // the maximum is taken before the scaling and masked scores are -inf, so the sign of the scale (or its being 0) goes into q
  const float scale = a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2);
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u, keep = a.scale_log2 == 0.f ? 0u : ~0u;
  uint32_t pieces = 0, blocks = 0;
  AttnPiece p;
  while (walk.next(a, &p)) {
    if (sub == 1 && p.t.nrows <= 128) continue;
    int token, head, pos;
    attn_row(a, p, min(r, max(p.t.nrows - 1, 0)), &token, &head, &pos);
    float m = -INFINITY, l = 0.f;
    const bool any = p.b0 < p.b1;
    if (any) {
      // ---- the warp's 32 query rows to shared memory
      constexpr int CPR = HD / 8, RPI = 32 / CPR;
      const int chunk = lane % CPR, c = chunk & 7;
      uint8_t* dst = smem + sub * M::TILE + (chunk >> 3) * M::BOX;
#pragma unroll
      for (int i0 = 0; i0 < 32 / RPI; i0 += 8) {
        uint4 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int rr = quarter * 32 + (i0 + i) * RPI + lane / CPR, row = sub * 128 + rr;
          x[i] = make_uint4(0, 0, 0, 0);
          if (row < p.t.nrows) {
            int tk, hd, ps;
            attn_row(a, p, row, &tk, &hd, &ps);
            x[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + tk * a.ldq + hd * HD + chunk * 8);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int rr = quarter * 32 + (i0 + i) * RPI + lane / CPR;
          x[i] = make_uint4((x[i].x ^ flip) & keep, (x[i].y ^ flip) & keep, (x[i].z ^ flip) & keep, (x[i].w ^ flip) & keep);
          *reinterpret_cast<uint4*>(dst + rr * 128 + ((c ^ (rr & 7)) << 4)) = x[i];
        }
      }
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&sy.q_full[sub]);
    }
    // keys that all rows of this half see need no mask
    const int pos_first = p.t.pos0 + (p.t.row0 + sub * 128) / a.group, pos_last = p.hi - 1;
    for (int b = p.b0; b < p.b1; ++b) {
      if (!ptx::mbar_wait_warp(&sy.s_full[sub], blocks++ & 1u, abort_flag)) return;
      ptx::tc_fence_after();
      uint32_t raw[128];
      ptx::tmem_ld_32x64(t_s, raw);
      ptx::tmem_ld_32x64(t_s + 64, raw + 64);
      const int key0 = (p.t.blk_lo + b) * kAttnBlock;
      if (!(key0 + kAttnBlock - 1 <= pos_first && (a.window == 0 || key0 > pos_last - a.window))) {
        const int hi = pos - key0, lo = a.window > 0 ? hi - a.window : -1;
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (i > hi || (a.window > 0 && i <= lo)) raw[i] = 0xff800000u;
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 128; ++i) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(raw[i]));
      const float now = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      const bool grow = (now - m) * scale > kLazy || (m == -INFINITY && now > m);
      if (__any_sync(0xffffffffu, grow)) {
        const float next = fmaxf(m, now), f = m == -INFINITY ? 0.f : pow2((m - next) * scale);
        m = next;
        l *= f;
        if (b > p.b0) {
#pragma unroll
          for (int i = 0; i < HD / 32; ++i) {
            uint32_t o[32];
            ptx::tmem_ld_32x32(t_o + i * 32, o);
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
            ptx::tmem_st_32x32(t_o + i * 32, o);
          }
        }
      }
      const float base = m == -INFINITY ? 0.f : -m * scale;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 64; ++i) {
        const float x = pow2(fmaf(__uint_as_float(raw[2 * i]), scale, base)), y = pow2(fmaf(__uint_as_float(raw[2 * i + 1]), scale, base));
        sum[i & 1] += x;
        sum[2 + (i & 1)] += y;
        raw[i] = pack2<T>(x, y);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      ptx::tmem_st_32x32(t_s, raw);
      ptx::tmem_st_32x32(t_s + 32, raw + 32);
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&sy.p_full[sub]);
    }
    if (any) {
      if (!ptx::mbar_wait_warp(&sy.o_full[sub], pieces++ & 1u, abort_flag)) return;
      ptx::tc_fence_after();
    }
    // ---- a row per thread
    const bool real = r < p.t.nrows;
    const bool some = l > 0.f || l != l;
    const float inv = p.slot < 0 ? attn_inverse(l, pos) : some ? 1.f / l : 0.f;
    const int64_t at = (int64_t)p.slot * a.slot_rows + r;
    const float base2 = m == -INFINITY ? 0.f : m * scale;
    bool fine = true;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      uint32_t o[32];
      if (any) ptx::tmem_ld_32x32(t_o + i * 32, o);
      else
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j] = 0u;
      float big = 0.f;
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const float v = __uint_as_float(o[j]);
        big = fmaxf(big, fabsf(v));
        fine = fine && v == v;
        o[j] = __float_as_uint(v * inv);
      }
      fine = fine && big < INFINITY;
      if (real) {
        if (p.slot < 0) {
          T* dst = reinterpret_cast<T*>(a.out) + token * a.ldo + head * HD + i * 32;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint4 v;
            v.x = pack2<T>(__uint_as_float(o[8 * j]), __uint_as_float(o[8 * j + 1]));
            v.y = pack2<T>(__uint_as_float(o[8 * j + 2]), __uint_as_float(o[8 * j + 3]));
            v.z = pack2<T>(__uint_as_float(o[8 * j + 4]), __uint_as_float(o[8 * j + 5]));
            v.w = pack2<T>(__uint_as_float(o[8 * j + 6]), __uint_as_float(o[8 * j + 7]));
            reinterpret_cast<uint4*>(dst)[j] = v;
          }
        } else {
          uint4* dst = reinterpret_cast<uint4*>(a.part_o + at * HD + i * 32);
#pragma unroll
          for (int j = 0; j < 8; ++j) dst[j] = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
        }
      }
    }
    if (real) {
      if (p.slot >= 0) a.part_l[at] = some ? base2 + log2f(l) : -INFINITY;
      else if (a.lse) a.lse[(int64_t)token * (a.kv_heads * a.group) + head] = (base2 + log2f(l)) * 0.69314718055994531f;
    }
    uint32_t bad = __ballot_sync(0xffffffffu, real && !fine);
    while (bad) {
      const int who = __ffs(bad) - 1;
      bad &= bad - 1;
      constexpr int N = HD / 32;
      float o[N];
      const int row = sub * 128 + quarter * 32 + who;
      const float f = __shfl_sync(0xffffffffu, inv, who);
      attn_repair_row<T, HD>(a, p, row, __shfl_sync(0xffffffffu, base2, who), o);
      int tk, hd, ps;
      attn_row(a, p, row, &tk, &hd, &ps);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (p.slot < 0) reinterpret_cast<T*>(a.out)[tk * a.ldo + hd * HD + lane * N + j] = DT<T>::from_f(o[j] * f);
        else a.part_o[((int64_t)p.slot * a.slot_rows + row) * HD + lane * N + j] = o[j] * f;
      }
    }
    ptx::tc_fence_before();  // O and S may be written again once the next q_full / p_full is seen
    __syncwarp();
  }
}

template <int HD> constexpr int tc_threads() { return HD == 256 ? Few<HD>::WARPS * 32 : 384; }
template <int HD> constexpr int tc_smem() {
  if constexpr (HD == 256) return Few<HD>::SMEM;
  else return (Few<HD>::SMEM > Many<HD>::SMEM ? Few<HD>::SMEM : Many<HD>::SMEM) + 1024;
}

// One CTA per SM: its share's tiles of many rows first, then those of few.
// 384 threads x 168 registers, dealt out again: 8 warps that compute x 216, and 72 for the four of which two issue products
// and loads.  (256 x 216 + 128 x 72 = 384 x 168.)
template <typename T, int HD>
__global__ void __launch_bounds__(tc_threads<HD>(), 1)
attn_tc_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap map) {
  extern __shared__ uint8_t smem_tc[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_tc) + 1023) & ~uintptr_t(1023));
  ptx::grid_dependency_wait();
  if ((int)blockIdx.x >= a.plan.header[1]) return;
  if constexpr (HD == 256) {
    ptx::grid_launch_dependents();
    few_share<T, HD>(a, smem, blockIdx.x);
  } else {
    __shared__ __align__(8) ManySync sy;
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
    AttnWalk walk(a, blockIdx.x);
    walk.until(a.plan.header[3]);
    const bool many = walk.more();  // the same for the whole CTA
    if (many) {
      if (threadIdx.x == 0) {
        for (int i = 0; i < Many<HD>::STAGES; ++i) { ptx::mbar_init(&sy.full[i], 1); ptx::mbar_init(&sy.empty[i], 1); }
        for (int i = 0; i < 2; ++i) {
          ptx::mbar_init(&sy.q_full[i], 4); ptx::mbar_init(&sy.s_full[i], 1);
          ptx::mbar_init(&sy.p_full[i], 4); ptx::mbar_init(&sy.o_full[i], 1);
        }
        ptx::mbar_init(&sy.drain, 1);
        sy.abort_word = 0;
        ptx::mbar_fence_init();
        ptx::prefetch_tensormap(&map);
      }
      if (warp == 8) { ptx::tmem_alloc(&sy.tmem, 512); ptx::tmem_relinquish(); }
      ptx::tc_fence_before();
      __syncthreads();
      ptx::tc_fence_after();
    }
    ptx::grid_launch_dependents();  // the TMEM is ours
    __syncwarp();
    if (warp >= 8) {
      ptx::registers_shrink<72>();
      if (!many) return;
      if (warp == 9) many_load<HD>(a, &map, smem, sy, walk);
      else if (warp == 8) many_multiply<T, HD>(a, smem, sy, walk);
      __syncwarp();
      ptx::tc_fence_before();
      __syncthreads();
      if (warp == 8) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(sy.tmem, 512);
      }
    } else {
      ptx::registers_grow<216>();
      if (many) {
        many_softmax<T, HD>(a, smem, sy, walk);
        __syncwarp();
        ptx::tc_fence_before();
        __syncthreads();
        if (sy.abort_word && threadIdx.x == 0 && a.status) atomicCAS(a.status, 0u, (uint32_t)CS_TIMEOUT_MBARRIER);
      }
      few_share<T, HD>(a, smem, blockIdx.x);
    }
  }
}

template <typename T, int HD>
static int launch_tc(const AttnArgs& a, bool many, int workers, cudaStream_t s) {
  constexpr int smem = tc_smem<HD>();
  CUtensorMap map = {};
  if (many) {
    const int rc = make_tmap_2d(&map, DT<T>::id, a.cache, (int64_t)a.num_pages * 2 * a.page_size, (int64_t)a.kv_heads * HD,
                                (int64_t)a.kv_heads * HD, a.page_size < kAttnBlock ? a.page_size : kAttnBlock, 64);
    if (rc) return rc;
  }
  SB_CUDA(cudaFuncSetAttribute(attn_tc_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  auto kern = attn_tc_kernel<T, HD>;  // (waits for its predecessor by hand)
  SB_CUDA(launch_dependent(kern, dim3((unsigned)workers), dim3(tc_threads<HD>()), smem, s, a, map));
  return SB200_OK;
}

int run_attn_tc(int dtype, int head_dim, const AttnArgs& a, const AttnShape& sh, int workers, cudaStream_t s) {
  const bool many = sh.few_limit < INT32_MAX;
  if (dtype == SB200_BF16)
    return head_dim == 64    ? launch_tc<__nv_bfloat16, 64>(a, many, workers, s)
           : head_dim == 128 ? launch_tc<__nv_bfloat16, 128>(a, many, workers, s)
                             : launch_tc<__nv_bfloat16, 256>(a, many, workers, s);
  return head_dim == 64    ? launch_tc<__half, 64>(a, many, workers, s)
         : head_dim == 128 ? launch_tc<__half, 128>(a, many, workers, s)
                           : launch_tc<__half, 256>(a, many, workers, s);
}

}  // namespace sb200

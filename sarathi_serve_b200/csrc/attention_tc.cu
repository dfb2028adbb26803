// Attention of fp16 / bf16 steps on the tensor cores.
//
// Few rows (a decoded token of a group of heads, a chunk of a handful of tokens: up to 16 rows a unit).  Every key and
// value is read once for at most 16 rows, 4 FLOP a byte and row: bound by HBM, far below what any tensor instruction asks
// for, so the products are warp-wide m16n8k16 with the rows as M, and everything is arranged for loads in flight.  The
// eight warps of a CTA take 16 keys each in turn and own a ring of three steps apiece in shared memory, filled by
// 16-byte asynchronous copies: no barrier between them while they stream, and 128 to 192 KB in flight per SM.  A warp keeps
// its own running maximum, sum and output; they are joined once a piece.  Its loads run ahead into the next piece.
// 209 decodes of 512 to 8192 tokens, 32 heads on 8 of 128: 612 us for 3.95 GB, 6.4 TB/s; a block of 128 keys and values takes an SM
// 1.4 us then (heads of 64: 0.8), a unit 2.6 us besides.  8 decodes of up to 2048 tokens: 16 us, bound by latency.
//
// Many rows (prompt chunks): tiles of 256 rows on tcgen05, see "many rows" below.
//
// Scores, maxima, sums and outputs are fp32.  Probabilities are rounded to the 16 bits of the values, as both tensor instructions
// want both operands of one type: that is at most half a step of each, like one more rounding of each value (fp16 below 2^-21 of the
// largest: 2^-32 of it, see kHeadroom).  The sum that the result is divided by is that of the unrounded ones.
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
  static constexpr int STATS = 2 * WARPS * kFewRows * 4 + 16;
  static constexpr int SMEM = RING + JOIN + STATS;
};

// ------------------------------------------------------------------ warp-wide pieces
// `ex2.approx`: relative error 2^-22, 2^-inf = 0.
__device__ __forceinline__ float pow2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 numbers that one instruction works on.
using f32x2 = uint64_t;
__device__ __forceinline__ f32x2 pair(uint32_t lo, uint32_t hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ f32x2 pair(float lo, float hi) { return pair(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ float low(f32x2 x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float high(f32x2 x) { return __uint_as_float((uint32_t)(x >> 32)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// The largest of three, or NaN if one of them is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
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

// Probabilities are made 2^kHeadroom times as large (the sums with them, so the result is the same): fp16 has no full precision below
// 2^-14, and one key that outweighs the others by more than that would coarsen theirs (20000 keys of 2^-19.3 beside one: 0.7 % off).
// With kLazy they reach 2^15 and no more, which fp16 holds.
template <typename T> constexpr float kHeadroom = DT<T>::id == SB200_F16 ? 7.f : 0.f;

// Lane i of a quad has row i's four pieces; afterwards v[j] is piece i of row j.
__device__ __forceinline__ void turn_quad(uint4 (&v)[4], int lane4) {
  auto swap = [&](uint4& x, uint4& y, int mask, bool upper) {  // the upper lane gives x and takes y's place
    uint4 s = upper ? x : y;
    s.x = __shfl_xor_sync(0xffffffffu, s.x, mask); s.y = __shfl_xor_sync(0xffffffffu, s.y, mask);
    s.z = __shfl_xor_sync(0xffffffffu, s.z, mask); s.w = __shfl_xor_sync(0xffffffffu, s.w, mask);
    if (upper) x = s;
    else y = s;
  };
  const bool up1 = lane4 & 1, up2 = lane4 & 2;
  swap(v[0], v[1], 1, up1);
  swap(v[2], v[3], 1, up1);
  swap(v[0], v[2], 2, up2);
  swap(v[1], v[3], 2, up2);
}

// What a product with P = 0 cannot do is to leave out a value that is not finite.  Called by a warp for a row of which some columns
// came out not finite; o: this lane's columns lane * HD / 32 ..., m: what was taken from the scores in the row's sum.  Only keys that
// the tile has and the row does not see can have spoilt it: if one of them is not finite in such a column, the column is
// made again, key by key (true is returned); if none is, the result stands.  So a value that is not finite costs the rows that see
// it a look at their tile's last keys, and only the rows of its own tile before it the long way.
template <typename T, int HD>
__device__ __noinline__ bool attn_repair_row(const AttnArgs& a, const AttnPiece& p, int r, float m, float* o) {
  constexpr int N = HD / 32;
  const int lane = threadIdx.x & 31;
  int token, head, pos;
  attn_row(a, p, r, &token, &head, &pos);
  const T* q = reinterpret_cast<const T*>(a.q) + token * a.ldq + head * HD + lane * N;
  const T* cache = reinterpret_cast<const T*>(a.cache) + p.head * HD + lane * N;
  const int64_t ldc = (int64_t)a.kv_heads * HD;
  const int begin = max(p.lo, (p.t.blk_lo + p.b0) * kAttnBlock), end = min(p.hi, (p.t.blk_lo + p.b1) * kAttnBlock);
  const int k0 = max(begin, a.window > 0 ? pos + 1 - a.window : 0), k1 = min(end, pos + 1);  // what the row sees of the piece
  bool spoilt[N] = {};
  auto look = [&](int from, int to) {
    for (int key = from; key < to; ++key) {
      const int at = attn_key_row(a, p.t.page_at, key);
      if (at < 0) continue;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (!(fabsf(o[j]) < INFINITY) && !(fabsf(DT<T>::to_f(cache[(at + a.page_size) * ldc + j])) < INFINITY)) spoilt[j] = true;
    }
  };
  look(begin, min(k0, end));
  look(max(k1, begin), end);
  bool any = false;
#pragma unroll
  for (int j = 0; j < N; ++j) any = any || spoilt[j];
  if (!__any_sync(0xffffffffu, any)) return false;
  float x[N], y[N];
#pragma unroll
  for (int j = 0; j < N; ++j) { x[j] = DT<T>::to_f(q[j]); y[j] = 0.f; }
  for (int key = k0; key < k1; ++key) {
    const int at = attn_key_row(a, p.t.page_at, key);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) s += at >= 0 ? x[j] * DT<T>::to_f(cache[at * ldc + j]) : x[j] * 0.f;
    s = warp_sum(s);
    const float pr = DT<T>::to_f(DT<T>::from_f(pow2(s * a.scale_log2 - m)));
#pragma unroll
    for (int j = 0; j < N; ++j) y[j] += pr * (at >= 0 ? DT<T>::to_f(cache[(at + a.page_size) * ldc + j]) : 0.f);
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (spoilt[j]) o[j] = y[j];
  return true;
}

// The steps of 16 keys that a warp loads (or computes) for the pieces of its CTA's share, one after the other.
template <int HD> struct FewSteps {
  AttnWalk walk;
  AttnPiece p;
  int key, end;   // next step of the current piece, and where it ends
  __device__ __forceinline__ FewSteps(const AttnArgs& a, const int4* share) : walk(a, share), key(0), end(0) { walk.only_few(a); }
  __device__ __forceinline__ bool next_piece(const AttnArgs& a, int warp) {
    if (!walk.next(a, &p)) return false;
    key = (max(p.lo, (p.t.blk_lo + p.b0) * kAttnBlock) & ~(kFewKeys - 1)) + warp * kFewKeys;
    end = min(p.hi, (p.t.blk_lo + p.b1) * kAttnBlock);
    return true;
  }
};

template <typename T, int HD>
__device__ void few_share(const AttnArgs& a, uint8_t* smem, const int4* share) {
  using F = Few<HD>;
  constexpr int CPR = HD / 8;              // 16-byte pieces of a key
  constexpr int KPI = 32 / CPR > 0 ? 32 / CPR : 1;  // keys that one copy instruction of the warp covers
  constexpr int IPK = CPR > 32 ? CPR / 32 : 1;
  static_assert(IPK == 1, "a key is at most 32 pieces");
  constexpr int KS = HD / 16, NT = HD / 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const uint32_t ring = ptx::smem_u32(smem) + warp * (F::STAGES * 2 * F::HALF);
  float* join = reinterpret_cast<float*>(smem + F::RING);               // [warp][row of a pass][HD], and the query rows before
  const uint32_t sq = ptx::smem_u32(join + warp * 8 * HD);
  float* stat_m = reinterpret_cast<float*>(smem + F::RING + F::JOIN);   // [warp][16]
  float* stat_l = stat_m + F::WARPS * kFewRows;
  int* rows_word = reinterpret_cast<int*>(stat_l + F::WARPS * kFewRows);  // rows of the piece, as the first warp sees them
  const T* cache = reinterpret_cast<const T*>(a.cache);
  const int64_t ldc = (int64_t)a.kv_heads * HD;
  constexpr int kStep = F::WARPS * kFewKeys;

  // loads: one step ahead of the copies the pages of the keys are asked for (lane i: key i of the step)
  FewSteps<HD> ld(a, share);
  bool more = true;
  AttnAhead next;
  int head_next = 0;
  auto look_up = [&]() {
    while (more && ld.key >= ld.end) more = ld.next_piece(a, warp);
    if (!more) return;
    const int key = ld.key + (lane & 15);
    next.ask(a, ld.p.t.page_at, key, key >= ld.p.lo && key < ld.p.hi);
    head_next = ld.p.head;
    ld.key += kStep;
  };
  int put = 0;
  auto load = [&]() {
    if (more) {
      const int rows = next.row(a), head = head_next;
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

  FewSteps<HD> st(a, share);
  int get = 0;
  while (st.next_piece(a, warp)) {
    const AttnPiece& p = st.p;
    // The query rows, 16 x HD, to this warp's part of the join buffer (swizzled like the keys): as the A operand they come from
    // there in every step, which costs less than the registers they would take.
    {
      T* q = reinterpret_cast<T*>(join + warp * 8 * HD);
      constexpr int RPI = 32 / CPR > 0 ? 32 / CPR : 1;
      const int sub = lane / CPR, chunk = lane % CPR;
      uint4 x[16 / RPI];
#pragma unroll
      for (int i = 0; i < 16 / RPI; ++i) {
        const int r = i * RPI + sub;
        int token, head, pos;
        attn_row(a, p, r, &token, &head, &pos);
        x[i] = make_uint4(0, 0, 0, 0);
        if (r < p.t.nrows) x[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + token * a.ldq + head * HD + chunk * 8);
      }
#pragma unroll
      for (int i = 0; i < 16 / RPI; ++i) {
        const int r = i * RPI + sub;
        *reinterpret_cast<uint4*>(q + r * HD + ((chunk ^ (r & 7)) << 3)) = x[i];
      }
      __syncwarp();
    }
    int pos_lo, pos_hi;  // of rows g and g + 8
    {
      int token, head;
      attn_row(a, p, min(g, max(p.t.nrows - 1, 0)), &token, &head, &pos_lo);
      attn_row(a, p, min(g + 8, max(p.t.nrows - 1, 0)), &token, &head, &pos_hi);
    }
    const int pos_first = p.t.pos0 + a.by_group.div(p.t.row0), pos_last = p.hi - 1;
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
        const int r = ((lane >> 4) << 3) + (lane & 7), c = (lane >> 3) & 1, rq = lane & 15, cq = lane >> 4;
#pragma unroll
        for (int k0 = 0; k0 < KS; k0 += 4) {
          constexpr int KB = 4;
          uint32_t kf[KB][4], qf[KB][4];
          load_matrices<KB, false>(kf, [&](int k) { return sk + r * F::ROW + ((((k0 + k) * 2 + c) ^ (r & 7)) << 4); });
          load_matrices<KB, false>(qf, [&](int k) { return sq + rq * F::ROW + ((((k0 + k) * 2 + cq) ^ (rq & 7)) << 4); });
          multiply<T, 2 * KB>([&](int i, float** cc, const uint32_t** aa, const uint32_t** bb) {
            *cc = s[i & 1]; *aa = qf[i >> 1]; *bb = &kf[i >> 1][2 * (i & 1)];
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
      const float b0 = (m0 == -INFINITY ? 0.f : m0) - kHeadroom<T>, b1 = (m1 == -INFINITY ? 0.f : m1) - kHeadroom<T>;
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
    if (threadIdx.x == 0) *rows_word = p.t.nrows;
    int all_rows = 1;  // (the same for all warps: they wait for each other in every pass)
    for (int pass = 0; pass * 8 < all_rows; ++pass) {
      if (pass * 8 + g < p.t.nrows) {
        float* dst = join + (warp * 8 + g) * HD + 2 * t4;
#pragma unroll
        for (int i = 0; i < NT; ++i)
          *reinterpret_cast<float2*>(dst + i * 8) = pass ? make_float2(o[i][2], o[i][3]) : make_float2(o[i][0], o[i][1]);
      }
      few_barrier(F::WARPS * 32);
      all_rows = *rows_word;
      const int rows = min(8, p.t.nrows - pass * 8);
      constexpr int N = HD / 32;
      for (int rr = warp; rr < rows; rr += F::WARPS) {  // a warp per row, N columns a lane
        const int r = pass * 8 + rr;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < F::WARPS; ++w) m = fmaxf(m, stat_m[w * kFewRows + r]);
        float base = m == -INFINITY ? 0.f : m;
        float l = 0.f, acc[N] = {};
#pragma unroll
        for (int w = 0; w < F::WARPS; ++w) {
          const float mw = stat_m[w * kFewRows + r], f = mw == -INFINITY ? 0.f : pow2(mw - base);
          l += f * stat_l[w * kFewRows + r];
#pragma unroll
          for (int j = 0; j < N; ++j) acc[j] += f * join[(w * 8 + rr) * HD + lane * N + j];
        }
        base -= kHeadroom<T>;
        bool fine = true;
#pragma unroll
        for (int j = 0; j < N; ++j) fine = fine && fabsf(acc[j]) < INFINITY;
        if (!__all_sync(0xffffffffu, fine) && l == l) {
          const AttnPiece copy = p;  // (p itself stays in registers)
          attn_repair_row<T, HD>(a, copy, r, base, acc);
        }
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
          if constexpr (N == 2)
            reinterpret_cast<float2*>(attn_part(a, HD, p.slot, p.stride, r, lane / 2))[lane & 1] = make_float2(acc[0] * inv, acc[1] * inv);
          else
#pragma unroll
            for (int j = 0; j < N; j += 4)
              *attn_part(a, HD, p.slot, p.stride, r, lane * (N / 4) + j / 4) =
                  make_float4(acc[j] * inv, acc[j + 1] * inv, acc[j + 2] * inv, acc[j + 3] * inv);
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
// TMEM holds S / P of both halves (2 x 128 columns) and O of both (2 x HD): with HD = 128 all of it.  Warps 0-3 make the
// probabilities of half A, warps 4-7 those of B, a row per thread; warp 8 issues the products, warp 9 loads keys and values,
// warps 10 and 11 the query rows of the next piece.  While the tensor pipe works for one half, the other half's warps turn S into P.
// P is handed over in two parts of 64 keys, so that P V of the first runs under the exponentials of the second; the next
// block's S follows P V at once.  (Steps of 64 keys with two score buffers per half take the tensor pipe 56 clocks per
// instruction of 64 columns, as long as one of 128: 4300 clocks a block.)  The maximum moves only when it has grown by 2^8 (kLazy), so
// O is hardly ever rescaled, and then by the warps that found out: S of a block is complete after O of the one before it.
// Keys and values come in boxes (128-byte swizzle) of as many rows, up to 128, as the page size has powers of two.  Pages
// outside the cache are fetched from behind its end, which fills zeros.  Values of keys that no row of the tile sees (behind
// the last, before the window) are cleared in shared memory, as 0 x NaN is not 0; rows that meet one all the same are recomputed
// (attn_repair_row).
// A block of 256 rows takes 1.7 us (2048 of its 3150 clocks the tensor pipe's), 1.5 with heads of 64, and 1.9 in mixed steps, whose
// other SMs use HBM up; a unit 5 us besides.  1999 tokens at 29001, 32 heads on 8 of 128: 820 us, 1.2 PFLOP/s, and 980 us where the
// power cap holds the clock at 1.6 GHz.  Bound by the chain S, softmax, P V of either half.
template <int HD> struct Many {
  static constexpr int HALVES = HD / 64;
  static constexpr int TILE = HALVES * 128 * 128;   // 128 rows
  static constexpr int QHALF = 128 * 128;           // query rows: [64 columns][128 rows]
  static constexpr int GROUP = HALVES * 1024;       // keys, values: [8 rows][64 columns][8 x 128 bytes]
  static constexpr int STAGES = HD == 128 ? 5 : 8;  // blocks of keys or values
  static constexpr int SMEM = (2 + STAGES) * TILE;
};

struct ManySync {
  uint64_t full[8], empty[8], q_full[2], q_empty[2], turn[2], p_full[2][2], drain;
  uint32_t tmem;
  int abort_word;
};

template <int HD>
__device__ __forceinline__ void many_load(const AttnArgs& a, const CUtensorMap* map, uint8_t* smem, ManySync& sy, AttnWalk walk) {
  using M = Many<HD>;
  const int lane = threadIdx.x & 31;
  volatile int* abort_flag = &sy.abort_word;
  const int box = min(a.page_size & -a.page_size, kAttnBlock), boxes = kAttnBlock / box, groups = box / 8;
  const int none = a.num_pages * 2 * (a.page_size / 8);  // the first group of 8 rows behind the cache
  int stage = 0, filled = 0;
  uint32_t phase = 0;
  bool ok = true;
  AttnPiece p;
  while (ok && walk.next(a, &p)) {
    // lane i: the page of box i, asked for a block ahead and looked at when its turn comes
    auto key_of = [&](int b) { return (p.t.blk_lo + b) * kAttnBlock + lane * box; };
    auto page_of = [&](int b) {
      const int key = key_of(b);
      const long long at = (long long)p.t.page_at + a.by_page.div(key);
      return b < p.b1 && lane < boxes && key < p.hi && at >= 0 && at < a.num_kv_indices ? a.kv_indices[at] : -1;
    };
    int next = page_of(p.b0);
    for (int b = p.b0; ok && b < p.b1; ++b) {
      const int page = next, key = key_of(b);
      next = page_of(b + 1);
      const bool want = lane < boxes && key < p.hi && key + box > p.lo;
      const uint32_t mask = __ballot_sync(0xffffffffu, want);
      const int slot = key - a.by_page.div(key) * a.page_size;
      const bool real = (unsigned)page < (unsigned)a.num_pages;
#pragma unroll 1
      for (int v = 0; ok && v < 2; ++v) {
        ok = ptx::mbar_wait_warp(&sy.empty[stage], phase ^ 1u, abort_flag);
        if (!ok) break;
        uint8_t* dst = smem + (2 + stage) * M::TILE;
        const int at = real ? (page * 2 + v) * (a.page_size / 8) + slot / 8 : none;
        if (ptx::elect_one()) ptx::mbar_expect_tx(&sy.full[stage], (uint32_t)(__popc(mask) * box * HD * 2));
        for (int i = 0; i < boxes; ++i) {
          const int g = __shfl_sync(0xffffffffu, at, i);
          if ((mask >> i) & 1u)
            if (ptx::elect_one()) ptx::tma_load_4d(dst + i * groups * M::GROUP, map, &sy.full[stage], 0, 0, p.head * M::HALVES, g);
        }
        ++filled;
        if (++stage == M::STAGES) { stage = 0; phase ^= 1u; }
      }
    }
  }
  {
    // wait (with a limit) for the copies that are still on their way before the CTA may end: those of a walk that was given up, or
    // of which another warp has seen less
    __shared__ int never;
    if (lane == 0) never = 0;
    __syncwarp();
    for (int i = max(0, filled - M::STAGES); i < filled; ++i) ptx::mbar_wait_warp(&sy.full[i % M::STAGES], (uint32_t)(i / M::STAGES) & 1u, &never);
  }
}

// The query rows of one half, a piece ahead of the warps that will use them.
template <typename T, int HD>
__device__ __forceinline__ void many_queries(const AttnArgs& a, uint8_t* smem, ManySync& sy, AttnWalk walk, int sub) {
  using M = Many<HD>;
  constexpr int CPR = HD / 8, RPI = 32 / CPR;  // 16-byte pieces of a row, rows per copy instruction of the warp
  const int lane = threadIdx.x & 31, chunk = lane % CPR, c = chunk & 7, first = lane / CPR;
  volatile int* abort_flag = &sy.abort_word;
  const uint32_t dst = ptx::smem_u32(smem) + sub * M::TILE + (chunk >> 3) * M::QHALF;
  const T* q = reinterpret_cast<const T*>(a.q) + chunk * 8;
  uint32_t pieces = 0;
  AttnPiece p;
  while (walk.next(a, &p)) {
    if (p.b0 >= p.b1 || (sub == 1 && p.t.nrows <= 128)) continue;
    if (!ptx::mbar_wait_warp(&sy.q_empty[sub], (pieces++ & 1u) ^ 1u, abort_flag)) break;
    // lane i knows where rows i, i + 32, ... begin (in units of 16 bytes)
    uint32_t at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = sub * 128 + i * 32 + lane;
      int token, head, pos;
      attn_row(a, p, row, &token, &head, &pos);
      at[i] = row < p.t.nrows ? (uint32_t)((token * a.ldq + head * HD) >> 3) : ~0u;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll 8
      for (int j = 0; j < 32; j += RPI) {
        const uint32_t from = __shfl_sync(0xffffffffu, at[i], j + first);
        const int rr = i * 32 + j + first;
        const bool real = from != ~0u;
        cp_async16(dst + rr * 128 + ((c ^ (rr & 7)) << 4), q + (real ? (int64_t)from * 8 : 0), real);
      }
    cp_async_commit();
    cp_async_wait<0>();
    ptx::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(&sy.q_full[sub]);
  }
}

// Every half has one barrier for "your turn": turn j of a piece is complete when S of block j is there and P V of block j - 1 is
// done; turn n, after the last block, stands for the end of O.  p_full[0 | 1]: the first | second part of P.  A barrier is
// never two phases ahead of its reader: turn j + 1 follows p_full of block j, which follows turn j, and the next piece's turn 0
// waits for an extra p_full[1], given when turn n has been seen.
template <typename T, int HD>
__device__ __forceinline__ void many_multiply(const AttnArgs& a, uint8_t* smem, ManySync& sy, AttnWalk walk) {
  using M = Many<HD>;
  const int lane = threadIdx.x & 31;
  volatile int* abort_flag = &sy.abort_word;
  constexpr int fmt = DT<T>::id == SB200_BF16 ? 1 : 0;
  const uint32_t id_s = ptx::make_idesc(fmt, 128), id_o = ptx::make_idesc(fmt, HD) | ptx::kIdescBRows;
  const uint32_t tmem = sy.tmem, sq = ptx::smem_u32(smem);
  // descriptors differ in the address field only, which counts 16 bytes
  const uint64_t d_query = ptx::make_smem_desc_sw128(sq), d_key = ptx::make_smem_desc_groups_sw128(sq, M::GROUP);
  const uint64_t d_value = ptx::make_smem_desc_rows_sw128(sq, 1024, M::GROUP);
  // The issuing lane's part.  S of half `sub` with the keys in `stage`:
  auto scores = [&](int sub, int stage) {
    const uint64_t dq = d_query + (uint64_t)(sub * (M::TILE >> 4)), dk = d_key + (uint64_t)((2 + stage) * (M::TILE >> 4));
#pragma unroll
    for (int k = 0; k < HD / 16; ++k)
      ptx::umma_f16(tmem + sub * 128, dq + (uint64_t)((k >> 2) * (M::QHALF >> 4) + (k & 3) * 2),
                    dk + (uint64_t)((k >> 2) * (1024 >> 4) + (k & 3) * 2), id_s, k > 0 ? 1u : 0u);
  };
  // O of half `sub` with the values in `stage` that go with a part of P.
  auto output = [&](int sub, int part, int stage, bool first) {
    const uint64_t dv = d_value + (uint64_t)((2 + stage) * (M::TILE >> 4) + part * (8 * M::GROUP >> 4));
#pragma unroll
    for (int k = 0; k < 4; ++k)
      ptx::umma_f16_ts(tmem + 256 + sub * HD, tmem + sub * 128 + part * 32 + k * 8, dv + (uint64_t)(k * (2 * M::GROUP >> 4)), id_o,
                       !first || part > 0 || k > 0 ? 1u : 0u);
  };
  int stage = 0;
  uint32_t phase = 0, p_phase[2][2] = {{0, 0}, {0, 0}}, q_phase[2] = {0, 0};
  bool ok = true;
  auto next_full = [&]() {  // the next stage, once it has been filled
    const int s = stage;
    ptx::mbar_wait_lanes(&sy.full[s], phase, abort_flag);
    if (++stage == M::STAGES) { stage = 0; phase ^= 1u; }
    return s;
  };
  auto wait_p = [&](int sub, int part) {
    ptx::mbar_wait_lanes(&sy.p_full[sub][part], p_phase[sub][part], abort_flag);
    p_phase[sub][part] ^= 1u;
    ptx::tc_fence_after();
  };
  AttnPiece p;
  while (ok && walk.next(a, &p)) {
    if (p.b0 >= p.b1) continue;
    const bool both = p.t.nrows > 128;
    const int ks0 = next_full();
#pragma unroll
    for (int s = 0; s < 2; ++s)
      if (s == 0 || both) {
        ptx::mbar_wait_lanes(&sy.q_full[s], q_phase[s], abort_flag);
        q_phase[s] ^= 1u;
        ptx::tc_fence_after();
        if (ptx::elect_one()) {
          scores(s, ks0);
          ptx::umma_commit(&sy.turn[s]);
          if (p.b0 + 1 == p.b1) ptx::umma_commit(&sy.q_empty[s]);
          if ((s == 1) == both) ptx::umma_commit(&sy.empty[ks0]);
        }
      }
    for (int b = p.b0; ok && b < p.b1; ++b) {
      const int vs = next_full(), key0 = (p.t.blk_lo + b) * kAttnBlock;
      const bool more = b + 1 < p.b1;
      if (key0 < p.lo || key0 + kAttnBlock > p.hi) {  // values that no row sees
        const int lo = p.lo - key0, hi = p.hi - key0;
        uint8_t* v = smem + (2 + vs) * M::TILE;
#pragma unroll 1
        for (int i = lane; i < 128 * 8; i += 32) {
          const int r = i >> 3;
          if (r < lo || r >= hi)
#pragma unroll
            for (int h = 0; h < M::HALVES; ++h)
              *reinterpret_cast<uint4*>(v + (r >> 3) * M::GROUP + h * 1024 + (r & 7) * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        ptx::fence_proxy_async_smem();
        __syncwarp();
      }
      int ks = 0;
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s == 0 || both) {
          wait_p(s, 0);
          if (ptx::elect_one()) output(s, 0, vs, b == p.b0);
          if (s == 0 && more) ks = next_full();
          wait_p(s, 1);
          if (ptx::elect_one()) {
            output(s, 1, vs, b == p.b0);
            if (more) scores(s, ks);
            ptx::umma_commit(&sy.turn[s]);
            if (b + 2 == p.b1) ptx::umma_commit(&sy.q_empty[s]);  // that was the last use of the queries
            if ((s == 1) == both) {
              ptx::umma_commit(&sy.empty[vs]);
              if (more) ptx::umma_commit(&sy.empty[ks]);
            }
          }
        }
      ok = __all_sync(0xffffffffu, *abort_flag == 0);  // a wait may have run out
    }
    if (ok)
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s == 0 || both) wait_p(s, 1);
  }
  {  // what has been issued may still read shared memory and write TMEM (under the other warps' last stores)
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
  // the maximum is taken before the scaling and masked scores are -inf, so the sign of the scale (or its being 0) goes first
  const float scale = a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2);
  uint32_t phase = 0;  // of this half's turns
  AttnPiece p;
  while (walk.next(a, &p)) {
    if (sub == 1 && p.t.nrows <= 128) continue;
    int token, head, pos;
    attn_row(a, p, min(r, max(p.t.nrows - 1, 0)), &token, &head, &pos);
    float m = -INFINITY, l = 0.f;
    // the warp's first and last position: keys that all of its rows see need no mask
    const int pos_warp_lo = __shfl_sync(0xffffffffu, pos, 0), pos_warp_hi = __shfl_sync(0xffffffffu, pos, 31);
    for (int b = p.b0; b < p.b1; ++b) {
      ptx::mbar_wait_lanes(&sy.turn[sub], phase, abort_flag);
      phase ^= 1u;
      ptx::tc_fence_after();
      uint32_t raw[128];
      ptx::tmem_ld_32x128(t_s, raw);
      if (a.scale_log2 <= 0.f) {
#pragma unroll
        for (int i = 0; i < 128; ++i) raw[i] = __float_as_uint(__uint_as_float(raw[i]) * (a.scale_log2 < 0.f ? -1.f : 0.f));
      }
      const int key = (p.t.blk_lo + b) * kAttnBlock;
      // (32 keys at a time, and none that all rows of the warp see.  Chunks of 500 and 100 decodes, heads of 64, window 1000: 69.6 -> 65.5 us)
      if (key + kAttnBlock - 1 > pos_warp_lo) {
        const int hi = pos - key;
#pragma unroll
        for (int c = 0; c < 128; c += 32)
          if (key + c + 31 > pos_warp_lo)
#pragma unroll
            for (int i = c; i < c + 32; ++i)
              if (i > hi) raw[i] = 0xff800000u;
      }
      if (a.window > 0 && key <= pos_warp_hi - a.window) {
        const int lo = pos - a.window - key;
#pragma unroll
        for (int c = 0; c < 128; c += 32)
          if (key + c <= pos_warp_hi - a.window)
#pragma unroll
            for (int i = c; i < c + 32; ++i)
              if (i <= lo) raw[i] = 0xff800000u;
      }
      // The probabilities of the first 64 keys are made with the maximum as it stands while the block's own is being found, and made
      // again in the rare case that it has grown too far.  (The maximum first, then the exponentials: 250 clocks of 2900 a block more.)
      uint32_t prob[32];
      f32x2 sum0, sum1;
      auto exponentials = [&](int part) {
        const float base = kHeadroom<T> - (m == -INFINITY ? 0.f : m * scale);
        const f32x2 sc = pair(scale, scale), bs = pair(base, base);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const f32x2 x = fma2(pair(raw[part * 64 + 2 * i], raw[part * 64 + 2 * i + 1]), sc, bs);
          const f32x2 y = pair(pow2(low(x)), pow2(high(x)));
          if (i == 0 && part == 0) sum0 = y;
          else if (i == 1 && part == 0) sum1 = y;
          else if (i & 1) sum1 = add2(sum1, y);
          else sum0 = add2(sum0, y);
          prob[i] = pack2<T>(low(y), high(y));
        }
      };
      auto publish = [&](int part) {
        ptx::tmem_st_32x32(t_s + part * 32, prob);
        ptx::tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&sy.p_full[sub][part]);
      };
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 64; ++i) top[i & 3] = max3(top[i & 3], __uint_as_float(raw[2 * i]), __uint_as_float(raw[2 * i + 1]));
      exponentials(0);
      const float now = max3(max3(top[0], top[1], top[2]), top[3], -INFINITY);
      const bool grow = now != -INFINITY && !((now - m) * scale <= kLazy);  // (also the first score, and one that is no number)
      if (__any_sync(0xffffffffu, grow)) {
        const float next = max3(m, now, -INFINITY), f = m == -INFINITY ? 0.f : pow2((m - next) * scale);
        m = next;
        l *= f;
        if (b > p.b0) {  // P V of the block before is done
#pragma unroll 1
          for (int i = 0; i < HD / 32; ++i) {
            uint32_t o[32];
            ptx::tmem_ld_32x32(t_o + i * 32, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            ptx::tmem_st_32x32(t_o + i * 32, o);
          }
        }
        exponentials(0);
      }
      publish(0);
      exponentials(1);
      publish(1);
      sum0 = add2(sum0, sum1);
      l += low(sum0) + high(sum0);
    }
    const bool any = p.b0 < p.b1;
    if (any) {
      ptx::mbar_wait_lanes(&sy.turn[sub], phase, abort_flag);
      phase ^= 1u;
      ptx::tc_fence_after();
      if (__any_sync(0xffffffffu, *abort_flag != 0)) return;
      if (lane == 0) ptx::mbar_arrive(&sy.p_full[sub][1]);  // the next piece's scores may begin
    }
    // ---- a row per thread
    const bool real = r < p.t.nrows;
    const bool some = l > 0.f || l != l;
    const float inv = p.slot < 0 ? attn_inverse(l, pos) : some ? 1.f / l : 0.f;
    const int64_t at = (int64_t)p.slot * a.slot_rows + r;
    const float base2 = (m == -INFINITY ? 0.f : m * scale) - kHeadroom<T>;
    bool fine = true;
    const long long mine = real ? token * a.ldo + head * HD : -1;  // where this thread's row goes
    long long quad_off[4];                                         // and those of its four lanes
#pragma unroll
    for (int j = 0; j < 4; ++j) quad_off[j] = __shfl_sync(0xffffffffu, mine, (lane & ~3) + j);
    const int lane4 = lane & 3;
#pragma unroll 1
    for (int i0 = 0; i0 < HD; i0 += 64) {  // (rolled: this code runs once a piece, and what it costs is fetching it)
      uint32_t o[64];
      if (any) ptx::tmem_ld_32x64(t_o + i0, o);
      else
#pragma unroll
        for (int j = 0; j < 64; ++j) o[j] = 0u;
      float none = 0.f;  // 0 x v is 0 unless v is not finite
#pragma unroll
      for (int j = 0; j < 64; ++j) {
        none = fmaf(__uint_as_float(o[j]), 0.f, none);
        o[j] = __float_as_uint(__uint_as_float(o[j]) * inv);
      }
      fine = fine && none == 0.f;
      // four lanes turn their rows' 4 x 16 bytes around, so that a store has 64 bytes of a row side by side
      if (p.slot < 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint4 v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t* x = o + 32 * h + 8 * j;
            auto two = [&](int e) { return pack2<T>(__uint_as_float(x[e]), __uint_as_float(x[e + 1])); };
            v[j] = make_uint4(two(0), two(2), two(4), two(6));
          }
          turn_quad(v, lane4);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (quad_off[j] >= 0) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + quad_off[j] + i0 + h * 32 + lane4 * 8) = v[j];
        }
      } else if (real) {
        uint4* dst = reinterpret_cast<uint4*>(attn_part(a, HD, p.slot, p.stride, r, i0 / 4));
#pragma unroll
        for (int j = 0; j < 16; ++j) dst[j * p.stride] = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
      }
    }
    if (real) {
      if (p.slot >= 0) a.part_l[at] = some ? base2 + log2f(l) : -INFINITY;
      else if (a.lse) a.lse[(int64_t)token * (a.kv_heads * a.group) + head] = (base2 + log2f(l)) * 0.69314718055994531f;
    }
    uint32_t bad = __ballot_sync(0xffffffffu, real && !fine && l == l);  // (a sum that is no number spoils the whole row, rightly)
    __syncwarp();
    while (bad) {
      const int who = __ffs(bad) - 1;
      bad &= bad - 1;
      constexpr int N = HD / 32;
      const AttnPiece copy = p;  // (p itself stays in registers)
      const int row = sub * 128 + quarter * 32 + who;
      int tk, hd, ps;
      attn_row(a, p, row, &tk, &hd, &ps);
      T* dst = reinterpret_cast<T*>(a.out) + tk * a.ldo + hd * HD;
      auto part = [&](int c) { return reinterpret_cast<float*>(attn_part(a, HD, p.slot, p.stride, row, c / 4)) + (c & 3); };
      float o[N];  // what the row's thread has just stored
#pragma unroll
      for (int j = 0; j < N; ++j) o[j] = p.slot < 0 ? DT<T>::to_f(dst[lane * N + j]) : *part(lane * N + j);
      bool ok[N];
#pragma unroll
      for (int j = 0; j < N; ++j) ok[j] = fabsf(o[j]) < INFINITY;
      const float f = __shfl_sync(0xffffffffu, inv, who);
      if (!attn_repair_row<T, HD>(a, copy, row, __shfl_sync(0xffffffffu, base2, who), o)) continue;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (ok[j]) continue;
        if (p.slot < 0) dst[lane * N + j] = DT<T>::from_f(o[j] * f);
        else *part(lane * N + j) = o[j] * f;
      }
    }
    ptx::tc_fence_before();  // O and S may be written again once the next q_full / p_full is seen
    __syncwarp();
  }
}

template <int HD> constexpr int tc_threads() { return HD == 256 ? Few<HD>::WARPS * 32 : 384; }
template <int HD> constexpr int tc_smem() {  // (1024: the kernel aligns its start)
  if constexpr (HD == 256) return Few<HD>::SMEM + 1024;
  else return (Few<HD>::SMEM > Many<HD>::SMEM ? Few<HD>::SMEM : Many<HD>::SMEM) + 1024;
}

// One CTA per SM: its share's tiles of many rows first, then those of few.
// 384 threads x 168 registers, dealt out again: 8 warps that compute x 216, and 72 for the four that issue products
// and loads.  (256 x 216 + 128 x 72 = 384 x 168.)
template <typename T, int HD>
__global__ void __launch_bounds__(tc_threads<HD>(), 1)
attn_tc_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap map) {
  extern __shared__ uint8_t smem_tc[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_tc) + 1023) & ~uintptr_t(1023));
  if constexpr (HD == 256) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    __shared__ int4 share[5];
    attn_share(a, share);
    few_share<T, HD>(a, smem, share);
  } else {
    // Barriers and TMEM before the wait, whether the share will need them or not: under the end of the kernel before.
    __shared__ __align__(8) ManySync sy;
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
    if (threadIdx.x == 0) {
      for (int i = 0; i < Many<HD>::STAGES; ++i) { ptx::mbar_init(&sy.full[i], 1); ptx::mbar_init(&sy.empty[i], 1); }
      for (int i = 0; i < 2; ++i) {
        ptx::mbar_init(&sy.q_full[i], 1); ptx::mbar_init(&sy.q_empty[i], 1); ptx::mbar_init(&sy.turn[i], 1);
        ptx::mbar_init(&sy.p_full[i][0], 4); ptx::mbar_init(&sy.p_full[i][1], 4);
      }
      ptx::mbar_init(&sy.drain, 1);
      sy.abort_word = 0;
      ptx::mbar_fence_init();
      if (a.page_size % 8 == 0) ptx::prefetch_tensormap(&map);  // (otherwise there is none)
    }
    if (warp == 8) { ptx::tmem_alloc(&sy.tmem, 512); ptx::tmem_relinquish(); }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();  // (the TMEM is ours, and the plan that the join reads at once is complete)
    __shared__ int4 share[5];
    attn_share(a, share);
    AttnWalk walk(a, share);
    walk.only_many(a);
    const bool many = walk.more();  // the same for the whole CTA
    __syncwarp();
    if (warp >= 8) {
      ptx::registers_shrink<72>();
      if (many) {
        if (warp == 9) many_load<HD>(a, &map, smem, sy, walk);
        else if (warp >= 10) many_queries<T, HD>(a, smem, sy, walk, warp - 10);
        else if (warp == 8) many_multiply<T, HD>(a, smem, sy, walk);
        __syncwarp();
        ptx::tc_fence_before();
        __syncthreads();
      }
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
      few_share<T, HD>(a, smem, share);
    }
  }
}

template <typename T, int HD>
static int launch_tc(const AttnArgs& a, bool many, int workers, cudaStream_t s) {
  constexpr int smem = tc_smem<HD>();
  CUtensorMap map = {};
  if (many) {
    // [64 columns][8 rows][kv heads x halves][groups of 8 rows]: a box is 64 columns x 8 rows x the halves of a head x its groups
    const uint64_t row = (uint64_t)a.kv_heads * HD * 2;
    const uint64_t dims[4] = {64, 8, (uint64_t)a.kv_heads * (HD / 64), (uint64_t)a.num_pages * 2 * (a.page_size / 8)};
    const uint64_t strides[3] = {row, 128, 8 * row};
    const uint32_t box[4] = {64, 8, HD / 64, (uint32_t)min(a.page_size & -a.page_size, kAttnBlock) / 8};
    const int rc = make_tmap_4d(&map, DT<T>::id, a.cache, dims, strides, box);
    if (rc) return rc;
  }
  static std::atomic<uint64_t> allowed{0};
  auto kern = attn_tc_kernel<T, HD>;  // (waits for its predecessor by hand)
  SB_CUDA(allow_smem(reinterpret_cast<const void*>(kern), smem, &allowed));
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

// Attention of fp16 / bf16 steps on the tensor cores.
//
// Few rows (a decoded token of a group of heads, a chunk of a handful of tokens: up to 16 rows a unit).  Every key and
// value is read once for at most 16 rows, 4 FLOP a byte and row: bound by HBM, far below what any tensor instruction asks
// for, so the products are warp-wide m16n8k16 with the rows as M, and everything is arranged for loads in flight.  The
// eight warps of a CTA take 16 keys each in turn and own a ring of three steps apiece in shared memory, filled by
// 16-byte asynchronous copies: no barrier between them while they stream, and 128 to 192 KB in flight per SM.  A warp keeps
// its own running maximum, sum and output; they are joined once a piece.  Its loads run ahead into the next piece.
#include "attention.cuh"

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
  __device__ __forceinline__ FewSteps(const AttnArgs& a, int worker) : walk(a, worker), key(0), end(0) {}
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
        for (int k0 = 0; k0 < KS; k0 += 8) {
          constexpr int KB = KS < 8 ? KS : 8;
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
        for (int n0 = 0; n0 < NT; n0 += 16) {
          constexpr int NB = NT < 16 ? NT : 16;
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
      constexpr int VPR = HD / 4, N = HD / 32;
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

template <typename T, int HD>
__global__ void __launch_bounds__(Few<HD>::WARPS * 32, 1)
attn_tc_kernel(const __grid_constant__ AttnArgs a) {
  grid_dependency_begin();
  extern __shared__ __align__(1024) uint8_t smem_tc[];
  const int workers = a.plan.header[1];
  for (int w = blockIdx.x; w < workers; w += gridDim.x) few_share<T, HD>(a, smem_tc, w);
}

template <typename T, int HD>
static int launch_tc(const AttnArgs& a, int workers, cudaStream_t s) {
  constexpr int smem = Few<HD>::SMEM;
  SB_CUDA(cudaFuncSetAttribute(attn_tc_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  SB_CUDA(launch_dependent(attn_tc_kernel<T, HD>, dim3((unsigned)workers), dim3(Few<HD>::WARPS * 32), smem, s, a));
  return SB200_OK;
}

int run_attn_tc(int dtype, int head_dim, const AttnArgs& a, const AttnShape& sh, int workers, cudaStream_t s) {
  (void)sh;
  if (dtype == SB200_BF16)
    return head_dim == 64    ? launch_tc<__nv_bfloat16, 64>(a, workers, s)
           : head_dim == 128 ? launch_tc<__nv_bfloat16, 128>(a, workers, s)
                             : launch_tc<__nv_bfloat16, 256>(a, workers, s);
  return head_dim == 64    ? launch_tc<__half, 64>(a, workers, s)
         : head_dim == 128 ? launch_tc<__half, 128>(a, workers, s)
                           : launch_tc<__half, 256>(a, workers, s);
}

}  // namespace sb200

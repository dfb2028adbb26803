// Attention on the FMA pipes: fp32 throughout (the parity configuration wants more than tf32 products).
//
// A CTA of 256 threads holds a tile of 32 query rows and walks the keys of its piece 32 at a time: keys and values through
// shared memory as fp32, four scores a thread (8 lanes share a row), running maximum and sum per row, and HD / 8 output
// columns a thread in registers.  Bound by shared memory and FMA alike: in both products a wavefront of 128 bytes feeds
// 128 multiply-adds.
#include "attention.cuh"

namespace sb200 {

constexpr int kSimtRows = 32, kSimtKeys = 32, kSimtThreads = 256;

template <int HD> constexpr size_t simt_smem() {
  return (size_t)(2 * 32 * (HD + 4) + 32 * HD + 32 * 33) * sizeof(float);
}

template <typename T, int HD>
__global__ void __launch_bounds__(kSimtThreads, 2)
attn_simt_kernel(const AttnArgs a) {
  grid_dependency_begin();
  extern __shared__ float smem_f[];
  constexpr int LD = HD + 4, N = Vec16<T>::N, VPR = HD / N;
  float* sq = smem_f;                 // [32][LD]
  float* sk = sq + kSimtRows * LD;    // [32][LD]
  float* sv = sk + kSimtKeys * LD;    // [32][HD]
  float* sp = sv + kSimtKeys * HD;    // [32][33]
  const int tid = threadIdx.x, row = tid >> 3, sub = tid & 7;
  const T* q = reinterpret_cast<const T*>(a.q);
  const T* cache = reinterpret_cast<const T*>(a.cache);
  const int64_t ldc = (int64_t)a.kv_heads * HD;

  for (int w = blockIdx.x; w < a.workers; w += gridDim.x) {
    AttnWalk walk(a, w);
    AttnPiece p;
    while (walk.next(a, &p)) {
      __syncthreads();  // the previous piece has been read
      for (int i = tid; i < kSimtRows * VPR; i += kSimtThreads) {
        const int r = i / VPR, v = i - r * VPR;
        int token, head, pos;
        attn_row(a, p, min(r, max(p.t.nrows - 1, 0)), &token, &head, &pos);
        Vec16<T> x;
        if (r < p.t.nrows) x = ld16(q + token * a.ldq + head * HD + v * N);
#pragma unroll
        for (int e = 0; e < N; ++e) sq[r * LD + v * N + e] = r < p.t.nrows ? DT<T>::to_f(x.v[e]) : 0.f;
      }
      int token, head, pos;
      attn_row(a, p, min(row, max(p.t.nrows - 1, 0)), &token, &head, &pos);
      const int seen_lo = a.window > 0 ? pos + 1 - a.window : 0;
      float m = -INFINITY, l = 0.f;
      float4 acc[HD / 32];
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      const int k0 = max(p.lo, (p.t.blk_lo + p.b0) * kAttnBlock) & ~(kSimtKeys - 1), k1 = min(p.hi, (p.t.blk_lo + p.b1) * kAttnBlock);
      for (int kb = k0; kb < k1; kb += kSimtKeys) {
        __syncthreads();
        for (int i = tid; i < 2 * kSimtKeys * VPR; i += kSimtThreads) {
          const bool val = i >= kSimtKeys * VPR;
          const int j = val ? i - kSimtKeys * VPR : i, r = j / VPR, v = j - r * VPR, key = kb + r;
          const int at = key >= p.lo && key < p.hi ? attn_key_row(a, p.t.page_at, key) : -1;
          Vec16<T> x;
          x.raw = make_uint4(0, 0, 0, 0);
          if (at >= 0) x = ld16(cache + (int64_t)(at + (val ? a.page_size : 0)) * ldc + p.head * HD + v * N);
          float* dst = val ? sv + r * HD + v * N : sk + r * LD + v * N;
#pragma unroll
          for (int e = 0; e < N; ++e) dst[e] = DT<T>::to_f(x.v[e]);
        }
        __syncthreads();
        float s[4] = {};
#pragma unroll 4
        for (int c = 0; c < HD; c += 4) {
          const float4 x = *reinterpret_cast<const float4*>(sq + row * LD + c);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 y = *reinterpret_cast<const float4*>(sk + (sub + 8 * i) * LD + c);
            s[i] += x.x * y.x + x.y * y.y + x.z * y.z + x.w * y.w;
          }
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = kb + sub + 8 * i;
          s[i] = key <= pos && key >= seen_lo ? s[i] * a.scale_log2 : -INFINITY;
          top = fmaxf(top, s[i]);
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float now = fmaxf(m, top), base = now == -INFINITY ? 0.f : now, keep = exp2f(m - base);
        m = now;
        l *= keep;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[i] = exp2f(s[i] - base);
          l += s[i];
          sp[row * 33 + sub + 8 * i] = s[i];
        }
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) { acc[i].x *= keep; acc[i].y *= keep; acc[i].z *= keep; acc[i].w *= keep; }
        __syncwarp();
#pragma unroll 4
        for (int k = 0; k < kSimtKeys; ++k) {
          const float pk = sp[row * 33 + k];
          if (pk == 0.f) continue;  // a key that the row does not see contributes nothing, whatever its value holds
#pragma unroll
          for (int i = 0; i < HD / 32; ++i) {
            const float4 v = *reinterpret_cast<const float4*>(sv + k * HD + i * 32 + sub * 4);
            acc[i].x += pk * v.x; acc[i].y += pk * v.y; acc[i].z += pk * v.z; acc[i].w += pk * v.w;
          }
        }
        __syncwarp();
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      if (row < p.t.nrows) {
        const float base = m == -INFINITY ? 0.f : m;
        if (p.slot < 0) {
          const float inv = attn_inverse(l, pos);
          T* dst = reinterpret_cast<T*>(a.out) + token * a.ldo + head * HD + sub * 4;
#pragma unroll
          for (int i = 0; i < HD / 32; ++i) {
            dst[i * 32] = DT<T>::from_f(acc[i].x * inv);
            dst[i * 32 + 1] = DT<T>::from_f(acc[i].y * inv);
            dst[i * 32 + 2] = DT<T>::from_f(acc[i].z * inv);
            dst[i * 32 + 3] = DT<T>::from_f(acc[i].w * inv);
          }
          if (a.lse && sub == 0) a.lse[(int64_t)token * (a.kv_heads * a.group) + head] = (base + log2f(l)) * 0.69314718055994531f;
        } else {
          const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
          const int64_t at = (int64_t)p.slot * a.slot_rows + row;
#pragma unroll
          for (int i = 0; i < HD / 32; ++i)
            *attn_part(a, HD, p.slot, p.stride, row, i * 8 + sub) = make_float4(acc[i].x * inv, acc[i].y * inv, acc[i].z * inv, acc[i].w * inv);
          if (sub == 0) a.part_l[at] = l > 0.f || l != l ? base + log2f(l) : -INFINITY;
        }
      }
    }
  }
}

template <typename T, int HD>
static int launch_simt(const AttnArgs& a, int workers, cudaStream_t s) {
  SB_CUDA(cudaFuncSetAttribute(attn_simt_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)simt_smem<HD>()));
  SB_CUDA(launch_dependent(attn_simt_kernel<T, HD>, dim3((unsigned)workers), dim3(kSimtThreads), simt_smem<HD>(), s, a));
  return SB200_OK;
}

int run_attn_simt(int head_dim, const AttnArgs& a, int workers, cudaStream_t s) {
  return head_dim == 64    ? launch_simt<float, 64>(a, workers, s)
         : head_dim == 128 ? launch_simt<float, 128>(a, workers, s)
                           : launch_simt<float, 256>(a, workers, s);
}

}  // namespace sb200

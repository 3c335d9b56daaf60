// The own rows of every sequence (and the shared ones where they are few) on warp-level tensor products: 16-bit types, heads of 32, 64
// and 128.
//
// Bound by HBM: a sequence's rows serve its own query heads only. The query heads of a KV head are the rows of a 16-row tile, both
// products are mma.sync.m16n8k16 with float32 sums, the maximum and the sum of a row run along. A CTA of four warps has one KV head of
// one sequence and a part of its keys, dealt to the warps 16 at a time; every warp is a pipeline of its own with 16-byte cp.async into
// padded stages, so that nothing but a warp barrier stands between a copy and its use. What lies behind the last row is not read:
// its place in a stage is filled with zeros and its score is -infinity.
// A weight is split into two 16-bit terms (two products into one sum): the products wait for memory anyway, and nothing of the
// weight is lost.
#include "attn_shared_common.cuh"

namespace nfai {

namespace {

using namespace shared_attn;

constexpr int kMW = 4, kMT = kMW * 32;
constexpr uint32_t kSlice = 16;  // keys per slice

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait_all_but() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(a));
}

template <typename T>
struct Half;
template <>
struct Half<__half> {
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ void split(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 r = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&r);
  }
};
template <>
struct Half<__nv_bfloat16> {
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ void split(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    const float2 f = __bfloat1622float2(h);
    const __nv_bfloat162 r = __floats2bfloat162_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&r);
  }
};

template <int D>
struct Shape {
  static constexpr int kStages = D == 128 ? 3 : 4;
  static constexpr int kLd = D + 8;  // elements of a staged row: 16 bytes more than it has, so that ldmatrix meets no bank twice
  static constexpr int kHalf = kSlice * kLd;  // elements of a slice of K or V
  static constexpr size_t kRing = (size_t)kMW * kStages * 2 * kHalf * 2;
};
template <int D, int ROWS>
constexpr size_t mma_smem() {
  constexpr size_t merge = (size_t)(kMW + 1) * ROWS * (D + 4) * 4 + (kMW + 1) * ROWS * 2 * 4;
  return Shape<D>::kRing > merge ? Shape<D>::kRing : merge;
}

// ROWS: 8 or 16 query heads
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kMT) attn_shared_mma_kernel(const SharedAttn p, const uint32_t hgroups) {
  using SH = Shape<D>;
  constexpr int NST = SH::kStages, LD = SH::kLd, HALF = SH::kHalf, R = ROWS / 8;
  extern __shared__ __align__(16) unsigned char sm_mma[];
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, qr = lane >> 2, qc = (lane & 3) * 2, G = p.qH / p.kvH;
  const uint32_t hg = blockIdx.x % hgroups, g = blockIdx.x / hgroups % p.kvH, b = blockIdx.x / hgroups / p.kvH;
  const uint32_t h0 = g * G + hg * ROWS, nh = min((uint32_t)ROWS, G - hg * ROWS), split = blockIdx.y;
  const Walk walk = walk_of(p, b, split);
  if (walk.idle || split >= walk.parts) return leave(p);
  const uint32_t slices = (walk.t1 - walk.t0 + kSlice - 1) / kSlice, mine = warp < slices ? (slices - warp + kMW - 1) / kMW : 0;
  const uint32_t kvDim = p.kvH * D;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(sm_mma) + warp * NST * 2 * HALF * 2;
  constexpr uint32_t CPR = D / 8;  // 16-byte pieces of a row
  const uint32_t c8 = (lane % CPR) * 8;
  auto issue = [&](uint32_t i) {
    const uint32_t n0 = walk.t0 + (i * kMW + warp) * kSlice, at = ring + (i % NST) * 2 * HALF * 2;
#pragma unroll
    for (uint32_t k = 0; k < kSlice * CPR / 32; ++k) {
      const uint32_t r = lane / CPR + k * (32 / CPR), t = n0 + r;
      const bool in = t < walk.t1;
      bool own;
      const uint64_t off = key_row(p, b, in ? t : walk.t0, own) * kvDim + g * D + c8;  // an address inside even where nothing is copied
      cp16(at + (r * LD + c8) * 2, reinterpret_cast<const T*>(own ? p.ko : p.kp) + off, in ? 16u : 0u);
      cp16(at + (HALF + r * LD + c8) * 2, reinterpret_cast<const T*>(own ? p.vo : p.vp) + off, in ? 16u : 0u);
    }
  };
#pragma unroll
  for (uint32_t i = 0; i < NST - 1; ++i) {
    if (i < mine) issue(i);
    cp_commit();  // (an empty group keeps the count uniform)
  }
  // the queries as they are: the left operand, rows beyond the heads zero
  uint32_t q[D / 16][4];
  {
    const T* const at = reinterpret_cast<const T*>(p.q) + ((uint64_t)b * p.qH + h0) * D + qc;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t row = qr + (u & 1) * 8;
        q[kk][u] = (u & 1) < R && row < nh ? __ldg(reinterpret_cast<const uint32_t*>(at + row * D + kk * 16 + (u >> 1) * 8)) : 0u;
      }
    }
  }
  float o[D / 8][4];
#pragma unroll
  for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
  }
  const uint32_t lm = lane >> 3, lr = lane & 7;
  const uint32_t k_lane = (((lm >> 1) * 8 + lr) * LD + (lm & 1) * 8) * 2, v_lane = (((lm & 1) * 8 + lr) * LD + (lm >> 1) * 8) * 2;

  for (uint32_t i = 0; i < mine; ++i) {
    __syncwarp();  // every lane is past its reads of the stage that is filled next
    if (i + NST - 1 < mine) issue(i + NST - 1);
    cp_commit();
    cp_wait_all_but<NST - 1>();
    __syncwarp();
    const uint32_t n0 = walk.t0 + (i * kMW + warp) * kSlice, ks = ring + (i % NST) * 2 * HALF * 2, vs = ks + HALF * 2;
    float s[2][4] = {};
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      uint32_t b0, b1, b2, b3;
      ldsm4(ks + kk * 32 + k_lane, b0, b1, b2, b3);
      Half<T>::mma(s[0], q[kk], b0, b1);
      Half<T>::mma(s[1], q[kk], b2, b3);
    }
    uint32_t hi[4] = {}, lo[4] = {};
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float x[4] = {s[0][2 * r] * p.scale2, s[0][2 * r + 1] * p.scale2, s[1][2 * r] * p.scale2, s[1][2 * r + 1] * p.scale2};
      if (n0 + kSlice > walk.t1) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n0 + (j >> 1) * 8 + qc + (j & 1) >= walk.t1) x[j] = -INFINITY;
      }
      float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)), m[r]);
      const float ref = top == -INFINITY ? 0.f : top, f = s_ex2(m[r] - ref);
      m[r] = top;
      float e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) e[j] = s_ex2(x[j] - ref);
      Half<T>::split(e[0], e[1], hi[r], lo[r]);
      Half<T>::split(e[2], e[3], hi[r + 2], lo[r + 2]);
      l[r] = l[r] * f + ((e[0] + e[1]) + (e[2] + e[3]));
      if (f != 1.f) {
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          o[j][2 * r] *= f;
          o[j][2 * r + 1] *= f;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < D / 8; j += 2) {
      uint32_t b0, b1, b2, b3;
      ldsm4t(vs + j * 16 + v_lane, b0, b1, b2, b3);
      Half<T>::mma(o[j], hi, b0, b1);
      Half<T>::mma(o[j + 1], hi, b2, b3);
      Half<T>::mma(o[j], lo, b0, b1);
      Half<T>::mma(o[j + 1], lo, b2, b3);
    }
  }
  cp_wait_all_but<0>();
  __syncthreads();  // every warp is past its last read of its stages: the warps' rows go where they were
  constexpr uint32_t PL = D + 4;
  float* const part = reinterpret_cast<float*>(sm_mma);            // [kMW][ROWS][PL]
  float* const rows = part + kMW * ROWS * PL;                      // [ROWS][PL]
  float* const ml = rows + ROWS * PL;                              // [kMW][ROWS][2]
  float* const M = ml + kMW * ROWS * 2;                            // [ROWS], [ROWS]
  float* const L = M + ROWS;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const uint32_t row = qr + r * 8;
#pragma unroll
    for (int j = 0; j < D / 8; ++j) *reinterpret_cast<float2*>(part + (warp * ROWS + row) * PL + j * 8 + qc) = make_float2(o[j][2 * r], o[j][2 * r + 1]);
    if ((lane & 3) == 0) {
      ml[(warp * ROWS + row) * 2] = m[r];
      ml[(warp * ROWS + row) * 2 + 1] = l[r];
    }
  }
  __syncthreads();
  for (uint32_t i = tid; i < nh * D; i += kMT) {
    const uint32_t j = i / D, e = i % D;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kMW; ++w) top = fmaxf(top, ml[(w * ROWS + j) * 2]);
    float acc = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kMW; ++w) {
      const float mw = ml[(w * ROWS + j) * 2], f = mw == -INFINITY ? 0.f : s_ex2(mw - top), lw = ml[(w * ROWS + j) * 2 + 1];
      if (f != 0.f || lw != lw) {
        acc = fmaf(f, part[(w * ROWS + j) * PL + e], acc);
        sum = fmaf(f, lw, sum);
      }
    }
    rows[j * PL + e] = acc;
    if (e == 0) {
      M[j] = top;
      L[j] = sum;
    }
  }
  __syncthreads();
  leave_rows<T, kMT>(p, b, h0, nh, walk, split, rows, PL, M, L);
}

template <typename T, int D, int ROWS>
cudaError_t launch_rows(cudaStream_t s, const SharedAttn& p) {
  constexpr size_t smem = mma_smem<D, ROWS>();
  cudaError_t e = cudaFuncSetAttribute(attn_shared_mma_kernel<T, D, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const uint32_t hgroups = (p.qH / p.kvH + ROWS - 1) / ROWS;
  return launch_pdl(attn_shared_mma_kernel<T, D, ROWS>, dim3(p.B * p.kvH * hgroups, p.own_splits), dim3(kMT), smem, s, p.pre_splits != 0, p, hgroups);
}
template <typename T, int D>
cudaError_t launch_d(cudaStream_t s, const SharedAttn& p, uint32_t rows) {
  return rows == 8 ? launch_rows<T, D, 8>(s, p) : launch_rows<T, D, 16>(s, p);
}
template <typename T>
cudaError_t launch_t(cudaStream_t s, const SharedAttn& p, uint32_t rows) {
  switch (p.d) {
    case 32: return launch_d<T, 32>(s, p, rows);
    case 64: return launch_d<T, 64>(s, p, rows);
    case 128: return launch_d<T, 128>(s, p, rows);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

cudaError_t launch_attn_shared_mma(cudaStream_t s, int dtype, const SharedAttn& p, uint32_t rows) {
  return dtype == 1 ? launch_t<__half>(s, p, rows) : dtype == 2 ? launch_t<__nv_bfloat16>(s, p, rows) : cudaErrorInvalidValue;
}

}  // namespace nfai

// Attention of one token of each of B sequences whose first rows are the same: softmax(q K^T scale) V over the `prefix` shared rows
// and over the sequence's own. Reference arithmetic: AttentionScoreCalculationShader.cs:170-205, AttentionSoftmaxShader.cs:145-177,
// AttentionWeightedValueSumShader.cs:181-215, once per sequence.
//
// This file holds the plan of a call and the kernel on the CUDA cores, for any type and head size: a CTA has the query heads of one KV
// head (up to 8) of one sequence and a part of its keys, 64 at a time as float32 in shared memory. Four threads share a key's scores
// (a quarter of the head each, all query heads), then a thread has four of the output's dimensions and every n-th key.
#include "attn_shared_common.cuh"

namespace nfai {

namespace {

using namespace shared_attn;

constexpr int kST = 256;
constexpr uint32_t kTK = 64;  // keys per tile
constexpr uint32_t kSharedWalk = 512;  // shared rows from which on they are walked once for all

__host__ __device__ constexpr uint32_t k_stride(uint32_t d) { return (d + 31) / 32 * 32 + 16; }  // two rows of a quarter-warp: other banks
size_t any_smem_floats(uint32_t d, uint32_t rows) {
  const size_t tiles = (size_t)kTK * (k_stride(d) + d), reduce = (size_t)kST * 4 * rows;
  return (size_t)rows * d + rows * kTK + 3 * rows + (tiles > reduce ? tiles : reduce);
}

template <typename T>
__device__ __forceinline__ void widen8(const T* at, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(at)), c = __ldg(reinterpret_cast<const float4*>(at) + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = c.x; f[5] = c.y; f[6] = c.z; f[7] = c.w;
  } else {
    WeightVec<T>::unpack(__ldg(reinterpret_cast<const uint4*>(at)), f);
  }
}

template <typename T, int NR>
__global__ void __launch_bounds__(kST) attn_shared_any_kernel(const SharedAttn p, const uint32_t hgroups) {
  extern __shared__ __align__(16) float sm_any[];
  const uint32_t d = p.d, kld = k_stride(d), d4 = d / 4, d8 = d / 8, G = p.qH / p.kvH;
  float* const q = sm_any;               // [NR][d]
  float* const w = q + NR * d;           // [kTK][NR] scores, then weights
  float* const m = w + NR * kTK;         // [NR]
  float* const l = m + NR;
  float* const f = l + NR;               // factors of the sums so far
  float* const K = f + NR + (4 - 3 * NR % 4) % 4;  // [kTK][kld]
  float* const V = K + kTK * kld;        // [kTK][d]
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t hg = blockIdx.x % hgroups, g = blockIdx.x / hgroups % p.kvH, b = blockIdx.x / hgroups / p.kvH;
  const uint32_t h0 = g * G + hg * NR, nh = min((uint32_t)NR, G - hg * NR);
  const Walk walk = walk_of(p, b, blockIdx.y);
  if (walk.idle || blockIdx.y >= walk.parts) return leave(p);
  {
    const T* const qg = reinterpret_cast<const T*>(p.q) + ((uint64_t)b * p.qH + h0) * d;
    for (uint32_t i = tid; i < NR * d; i += kST) q[i] = i < nh * d ? to_float(qg[i]) * p.scale2 : 0.f;
  }
  if (tid < NR) {
    m[tid] = -INFINITY;
    l[tid] = 0.f;
  }
  // score threads: a key each four; value threads: four dimensions, every KG-th key
  const uint32_t key = tid >> 2, part = tid & 3;
  const uint32_t KG = kST / d4, chunk = tid % d4, kg = tid / d4;
  const bool values = kg < KG;
  float o[NR][4];
#pragma unroll
  for (int r = 0; r < NR; ++r) o[r][0] = o[r][1] = o[r][2] = o[r][3] = 0.f;

  for (uint32_t n0 = walk.t0; n0 < walk.t1; n0 += kTK) {
    __syncthreads();  // the tile before has been used
    for (uint32_t i = tid; i < kTK * d8; i += kST) {
      const uint32_t r = i / d8, e = (i - r * d8) * 8, t = n0 + r;
      float a[8] = {}, c[8] = {};
      if (t < walk.t1) {
        bool own;
        const uint64_t at = (key_row(p, b, t, own) * p.kvH + g) * d + e;
        widen8(reinterpret_cast<const T*>(own ? p.ko : p.kp) + at, a);
        widen8(reinterpret_cast<const T*>(own ? p.vo : p.vp) + at, c);
      }
#pragma unroll
      for (int k = 0; k < 8; k += 4) {
        *reinterpret_cast<float4*>(K + r * kld + e + k) = make_float4(a[k], a[k + 1], a[k + 2], a[k + 3]);
        *reinterpret_cast<float4*>(V + r * d + e + k) = make_float4(c[k], c[k + 1], c[k + 2], c[k + 3]);
      }
    }
    __syncthreads();
    {
      float s[NR];
#pragma unroll
      for (int r = 0; r < NR; ++r) s[r] = 0.f;
      for (uint32_t c = part * 4; c < d; c += 16) {
        const float4 k4 = *reinterpret_cast<const float4*>(K + key * kld + c);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const float4 q4 = *reinterpret_cast<const float4*>(q + r * d + c);
          s[r] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[r]))));
        }
      }
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        s[r] += __shfl_xor_sync(0xffffffffu, s[r], 1);
        s[r] += __shfl_xor_sync(0xffffffffu, s[r], 2);
        if (part == 0) w[key * NR + r] = n0 + key < walk.t1 ? s[r] : -INFINITY;
      }
    }
    __syncthreads();
    if (warp < NR) {
      const float a = w[lane * NR + warp], c = w[(lane + 32) * NR + warp], before = m[warp];
      const float top = fmaxf(before, warp_max(fmaxf(a, c))), ref = top == -INFINITY ? 0.f : top;
      const float ea = exp2f(a - ref), ec = exp2f(c - ref), factor = exp2f(before - ref), sum = warp_sum(ea + ec);
      w[lane * NR + warp] = ea;
      w[(lane + 32) * NR + warp] = ec;
      if (lane == 0) {
        m[warp] = top;
        l[warp] = l[warp] * factor + sum;
        f[warp] = factor;
      }
    }
    __syncthreads();
    if (values) {
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float x = f[r];
        o[r][0] *= x; o[r][1] *= x; o[r][2] *= x; o[r][3] *= x;
      }
      for (uint32_t k = kg; k < kTK && n0 + k < walk.t1; k += KG) {
        const float4 v4 = *reinterpret_cast<const float4*>(V + k * d + chunk * 4);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const float x = w[k * NR + r];
          o[r][0] = fmaf(x, v4.x, o[r][0]);
          o[r][1] = fmaf(x, v4.y, o[r][1]);
          o[r][2] = fmaf(x, v4.z, o[r][2]);
          o[r][3] = fmaf(x, v4.w, o[r][3]);
        }
      }
    }
  }
  // the key groups' sums of a row, in their order, where the tiles were
  __syncthreads();
  if (values) {
#pragma unroll
    for (int r = 0; r < NR; ++r) *reinterpret_cast<float4*>(K + (r * KG + kg) * d + chunk * 4) = make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
  }
  __syncthreads();
  for (uint32_t i = tid; i < NR * d; i += kST) {
    const uint32_t r = i / d, e = i - r * d;
    float a = 0.f;
    for (uint32_t k = 0; k < KG; ++k) a += K[(r * KG + k) * d + e];
    q[i] = a;  // (the queries have been used)
  }
  __syncthreads();
  finish_rows<T, kST>(p, b, g, h0, nh, walk, blockIdx.y, blockIdx.x, q, d, m, l);
}

template <typename T, int NR>
cudaError_t launch_any(cudaStream_t s, const SharedAttn& p) {
  const size_t smem = (any_smem_floats(p.d, NR) + 4) * 4;
  cudaError_t e = cudaFuncSetAttribute(attn_shared_any_kernel<T, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const uint32_t hgroups = (p.qH / p.kvH + NR - 1) / NR;
  return launch_pdl(attn_shared_any_kernel<T, NR>, dim3(p.B * p.kvH * hgroups, p.own_splits), dim3(kST), smem, s, p.pre_splits != 0, p, hgroups);
}
template <typename T>
cudaError_t launch_own(cudaStream_t s, const SharedAttn& p, const SharedPlan& plan) {
  return plan.rows == 4 ? launch_any<T, 4>(s, p) : launch_any<T, 8>(s, p);
}

}  // namespace

SharedPlan plan_shared_attn(int dtype, uint32_t B, uint32_t qH, uint32_t kvH, uint32_t d, uint32_t prefix, uint32_t capacity) {
  SharedPlan a;
  const uint32_t G = qH / kvH;
  a.tensor = dtype != 0 && (d == 32 || d == 64 || d == 128);
  const bool shared = dtype != 0 && (d == 64 || d == 128) && B >= 2 && prefix >= kSharedWalk;
  if (shared) {
    // two CTAs on every SM at once, each with 128 rows (sequence, head of the group) and as many tiles of keys as the others
    const uint64_t groups = ((uint64_t)B * G + kPreRows - 1) / kPreRows * kvH;
    const uint32_t tiles = (prefix + kPreTile - 1) / kPreTile;
    uint64_t parts = 148 * 2 / groups;
    parts = parts < 1 ? 1 : parts > kMaxPreSplits ? kMaxPreSplits : parts;
    a.pre_tiles = (uint32_t)((tiles + parts - 1) / parts);
    a.pre_splits = (tiles + a.pre_tiles - 1) / a.pre_tiles;
  }
  const uint64_t keys = (uint64_t)capacity + (shared ? 0 : prefix);
  a.rows = a.tensor ? (G <= 8 ? 8 : 16) : (G <= 4 ? 4 : 8);
  const uint64_t groups = (uint64_t)B * kvH * ((G + a.rows - 1) / a.rows);
  // CTAs for every SM twice over (three times on the CUDA cores) where the keys go so far (parts of 64 at least)
  uint64_t parts = (148 * (a.tensor && d == 128 ? 2 : 3) + groups - 1) / groups;
  if (parts > (keys + 63) / 64) parts = (keys + 63) / 64;
  if (parts > kMaxOwnSplits) parts = kMaxOwnSplits;
  a.own_splits = parts < 1 ? 1 : (uint32_t)parts;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = (off + bytes + 255) / 256 * 256;
    return at;
  };
  const uint64_t rows = (uint64_t)B * qH;
  a.tickets = take(groups * 4);
  a.pre_ml = take(a.pre_splits * rows * 8);
  a.own_ml = take(a.own_splits > 1 ? a.own_splits * rows * 8 : 0);
  a.pre_o = take(a.pre_splits * rows * d * 4);
  a.own_o = take(a.own_splits > 1 ? a.own_splits * rows * d * 4 : 0);
  a.total = off;
  return a;
}

cudaError_t launch_shared_attn(cudaStream_t s, int dtype, const SharedAttn& p, const SharedPlan& plan) {
  cudaError_t e = cudaSuccess;
  if (plan.own_splits > 1) {
    const uint32_t G = p.qH / p.kvH;
    e = cudaMemsetAsync(p.tickets, 0, (size_t)p.B * p.kvH * ((G + plan.rows - 1) / plan.rows) * 4, s);
    if (e != cudaSuccess) return e;
  }
  if (plan.pre_splits) {
    e = launch_attn_shared_umma(s, dtype, p);
    if (e != cudaSuccess) return e;
  }
  if (plan.tensor) return launch_attn_shared_mma(s, dtype, p, plan.rows);
  switch (dtype) {
    case 0: return launch_own<float>(s, p, plan);
    case 1: return launch_own<__half>(s, p, plan);
    case 2: return launch_own<__nv_bfloat16>(s, p, plan);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace nfai

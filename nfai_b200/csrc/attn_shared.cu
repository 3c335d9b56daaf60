// Attention of one token of each of B sequences whose first rows are the same: softmax(q K^T scale) V over the `prefix` shared rows
// and over the sequence's own. Reference arithmetic: AttentionScoreCalculationShader.cs:170-205, AttentionSoftmaxShader.cs:145-177,
// AttentionWeightedValueSumShader.cs:181-215, once per sequence.
//
// This file holds the plan of a call, the join and the kernel on the CUDA cores, which serves float32 and heads above 128 (there, in 16 bits,
// the shared rows too, for every sequence once more: 64 sequences of 16 over 4 heads of 256 behind 16384 rows 3.7 ms, in float32, whose
// walk takes such heads, 0.67 ms): a CTA has the query heads of one KV head (up to 8) of one sequence and a part of its keys, 64 at a time
// as float32 in shared memory. Four threads share a key's scores (a quarter of the head each, all query heads), then a thread has four of
// the output's dimensions and every n-th key.
#include "attn_shared_common.cuh"

namespace nfai {

namespace {

using namespace shared_attn;

constexpr int kST = 256;
constexpr uint32_t kTK = 64;  // keys per tile

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
__global__ void __launch_bounds__(kST) attn_shared_any_kernel(const __grid_constant__ SharedAttn p, const uint32_t hgroups) {
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
  if (walk.idle || (p.joined && blockIdx.y >= walk.parts)) return leave(p);
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
  bool odd = false;
  for (uint32_t i = tid; i < NR * d; i += kST) {
    const uint32_t r = i / d, e = i - r * d;
    float a = 0.f;
    for (uint32_t k = 0; k < KG; ++k) a += K[(r * KG + k) * d + e];
    q[i] = a;  // (the queries have been used)
    odd |= a != a && is_sum(l[r]);
  }
  if (__syncthreads_or(odd)) {
    mend_part<T, kST>(p, b, h0, nh, walk.t0, walk.t1, q, d, l);
    __syncthreads();
  }
  leave_rows<T, kST, 4>(p, b, h0, nh, walk, blockIdx.y, q, d, m, l, K);  // (the groups' sums have been used)
}

template <typename T, int NR>
cudaError_t launch_any(cudaStream_t s, const SharedAttn& p) {
  const size_t smem = (any_smem_floats(p.d, NR) + 4) * 4;
  cudaError_t e = cudaFuncSetAttribute(attn_shared_any_kernel<T, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const uint32_t hgroups = (p.qH / p.kvH + NR - 1) / NR;
  return launch_pdl_cluster(attn_shared_any_kernel<T, NR>, dim3(p.B * p.kvH * hgroups, p.own_splits), dim3(kST), dim3(1, p.joined ? 1 : p.own_splits, 1), smem, s,
                            p.pre_splits != 0, p, hgroups);
}
// The join of partial results, a row of the output (sequence, query head) per WARPS warps. A lane has four dimensions (UNITS times) of a
// part; where LANES of them are a whole row, the warp has 32 / LANES parts at once. Eight parts are on their way at a time.
constexpr int kJT = 128;
template <typename T, int WARPS, int LANES, int UNITS>
__global__ void __launch_bounds__(kJT) attn_shared_join_kernel(const SharedAttn p) {
  constexpr int kRows = kJT / 32 / WARPS, kAtOnce = 32 / LANES;
  constexpr uint32_t kStep = WARPS * kAtOnce;
  __shared__ __align__(16) float part_o[WARPS > 1 ? kJT / 32 : 1][UNITS * 128];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % WARPS, row = blockIdx.x * kRows + warp / WARPS, d = p.d;
  pdl_wait();
  const bool there = row < p.B * p.qH;
  const uint32_t b = there ? row / p.qH : 0, h = row - b * p.qH, G = p.qH / p.kvH, g = h / G;
  const Walk walk = walk_of(p, b, 0);
  const bool busy = there && !walk.idle;
  const uint32_t own = busy ? walk.parts : 0, n = busy ? own + p.pre_splits : 0;
  const uint64_t BQ = (uint64_t)p.B * p.qH, R = (uint64_t)p.B * G, pre_step = p.kvH * R, pre0 = (uint64_t)g * R + (uint64_t)b * G + (h - g * G);
  // rows of parts, as offsets: a sequence's own, then the shared ones'
  auto own_row = [&](uint32_t i) { return (uint64_t)i * BQ + row; };
  auto pre_row = [&](uint32_t i) { return (uint64_t)(i - own) * pre_step + pre0; };
  const uint32_t slot = sub * kAtOnce + lane / LANES, e = lane % LANES * 4;  // parts slot, slot + kStep, ..
  const bool wide = UNITS > 1 || e < d;
  float M = -INFINITY, L = 0.f;
  float4 acc[UNITS] = {};
  for (uint32_t k0 = 0; k0 < n; k0 += 32) {  // 32 parts' maxima and sums, the same in every warp of the row
    const uint32_t cnt = min(32u, n - k0);
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < cnt) ml = __ldcg(reinterpret_cast<const float2*>(k0 + lane < own ? p.own_ml + own_row(k0 + lane) * 2 : p.pre_ml + pre_row(k0 + lane) * 2));
    const float top = fmaxf(M, warp_max(ml.x)), ref = top == -INFINITY ? 0.f : top, before = exp2f(M - ref), f = exp2f(ml.x - ref);
    M = top;
    // (a part without weights: nothing of it counts, but a sum that is not a number does)
    L = L * before + warp_sum(f != 0.f || ml.y != ml.y ? f * ml.y : 0.f);
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      acc[u].x *= before; acc[u].y *= before; acc[u].z *= before; acc[u].w *= before;
    }
#pragma unroll 1
    for (uint32_t k = slot; k < cnt + slot; k += 8 * kStep) {  // (the same count for all lanes: k - slot)
      float4 v[8][UNITS];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t i = k + j * kStep;
        const float* const o = (k0 + i < own ? p.own_o + own_row(k0 + i) * d : p.pre_o + pre_row(k0 + i) * d) + e;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          v[j][u] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (i < cnt && (UNITS > 1 ? u * 128 + e < d : wide)) v[j][u] = __ldcg(reinterpret_cast<const float4*>(o + u * 128));
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t i = k + j * kStep;
        float w = __shfl_sync(0xffffffffu, f, i & 31);
        w = i < cnt ? w : 0.f;
        if (w != 0.f) {
#pragma unroll
          for (int u = 0; u < UNITS; ++u) {
            acc[u].x = fmaf(w, v[j][u].x, acc[u].x); acc[u].y = fmaf(w, v[j][u].y, acc[u].y);
            acc[u].z = fmaf(w, v[j][u].z, acc[u].z); acc[u].w = fmaf(w, v[j][u].w, acc[u].w);
          }
        }
      }
    }
  }
#pragma unroll
  for (int o = LANES; o < 32; o <<= 1) {  // the parts that the warp had at once
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      acc[u].x += __shfl_xor_sync(0xffffffffu, acc[u].x, o);
      acc[u].y += __shfl_xor_sync(0xffffffffu, acc[u].y, o);
      acc[u].z += __shfl_xor_sync(0xffffffffu, acc[u].z, o);
      acc[u].w += __shfl_xor_sync(0xffffffffu, acc[u].w, o);
    }
  }
  if constexpr (WARPS > 1) {
    if (lane < LANES) {
#pragma unroll
      for (int u = 0; u < UNITS; ++u) *reinterpret_cast<float4*>(&part_o[warp][u * 128 + e]) = acc[u];
    }
    __syncthreads();
    if (sub != 0) return;
    for (int w = 1; w < WARPS; ++w) {  // (all of them to the same maximum)
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const float4 v = *reinterpret_cast<const float4*>(&part_o[warp + w][u * 128 + e]);
        acc[u].x += v.x; acc[u].y += v.y; acc[u].z += v.z; acc[u].w += v.w;
      }
    }
  }
  if (!busy || lane >= LANES) return;
  const float inv = p.prefix || walk.n ? 1.0f / L : 0.f;
  T* const out = reinterpret_cast<T*>(p.out) + (uint64_t)row * d;
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const uint32_t at = u * 128 + e;
    if (at < d) {
      alignas(16) T y[4];
      store_as(y, acc[u].x * inv);
      store_as(y + 1, acc[u].y * inv);
      store_as(y + 2, acc[u].z * inv);
      store_as(y + 3, acc[u].w * inv);
      if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out + at) = *reinterpret_cast<const float4*>(y);
      else *reinterpret_cast<uint2*>(out + at) = *reinterpret_cast<const uint2*>(y);
    }
  }
}

template <typename T, int LANES, int UNITS>
cudaError_t launch_join_of(cudaStream_t s, const SharedAttn& p) {
  const uint32_t rows = p.B * p.qH;
  // Four warps a row where there are many parts and CTAs for all of them at once, a warp a row | four: 3 sequences of 16 heads of 128 behind 100000
  // rows 29.1 | 22.9 us a call, 8 of 32 of 128 behind 2011 11.5 | 11.0, 5 of 32 of 64 behind 100003 40.7 | 40.5, in float32 9 of 8 of 32 behind 1000
  // 8.6 | 8.5; 64 of 32 of 128 behind 32768 (2048 rows, 18 parts) 67.8 | 69.7.
  if (p.pre_splits + p.own_splits > 16 && rows < 148 * 32)
    return launch_pdl(attn_shared_join_kernel<T, 4, LANES, UNITS>, dim3(rows), dim3(kJT), 0, s, true, p);
  return launch_pdl(attn_shared_join_kernel<T, 1, LANES, UNITS>, dim3((rows + 3) / 4), dim3(kJT), 0, s, true, p);
}
template <typename T>
cudaError_t launch_join(cudaStream_t s, const SharedAttn& p) {
  if (p.d == 32) return launch_join_of<T, 8, 1>(s, p);
  if (p.d == 64) return launch_join_of<T, 16, 1>(s, p);
  return p.d <= 128 ? launch_join_of<T, 32, 1>(s, p) : launch_join_of<T, 32, 2>(s, p);
}

template <typename T>
cudaError_t launch_own(cudaStream_t s, const SharedAttn& p, const SharedPlan& plan) {
  return plan.rows == 4 ? launch_any<T, 4>(s, p) : launch_any<T, 8>(s, p);
}

}  // namespace

namespace {
constexpr uint32_t kLeastOfAll = 32;  // keys of a part of the own rows at least
// Query heads of a CTA. On the tensor cores, 8 | 16: 64 sequences of 32 heads over 8 of 64 with 500 keys 15.5 | 15.9 us, of 8 over 1 with 900 9.2 | 9.4;
// of 16 over 1 of 128 with 2000 24.4 | 21.9 (16 are two CTAs on the same keys), 40 of 32 over 2 of 64 with 1300 16.7 | 14.0. On the CUDA cores, 4 | 8:
// 16 of 32 over 8 of 64 with 700 25.9 | 32.1, 20 of 16 over 4 of 256 with 800 97 | 124; of 16 over 2 88 | 49, 30 of 16 over 2 of 64 with 600 28.1 | 21.1.
constexpr uint32_t own_rows_of(bool tensor, uint32_t G) { return tensor ? (G <= 8 ? 8 : 16) : (G <= 4 ? 4 : 8); }
// CTAs that the own rows are cut into: two for an SM, on the CUDA cores four. 1 | 2 | 3 | 4: 8 sequences of 32 over 8 heads of 128 with 6000 keys 42.5 |
// 35.0 | 41.7 | 37.7 us, 4 of 64 with 9000 32.1 | 23.0 | 20.6 | 20.4, 20 of 64 with 1700 25.2 | 19.0 | 17.7 | 16.7, 3 of 16 over 1 of 128 with 20000
// 15.5 | 16.1 | 18.3 | 18.1. CUDA cores, 1 | 2 | 4 | 8: 4 of 32 over 8 of 64 with 5000 73 | 47 | 43 | 42, 9 of 8 over 2 of 32 behind 1000 10.7 | 9.2 |
// 8.6 | 8.5, in 16 bits 4 of 16 over 4 of 256 with 3300 67 | 53 | 60 | 59.
constexpr uint32_t own_ctas_of(bool tensor) { return 148 * (tensor ? 2 : 4); }
}  // namespace

SharedPlan plan_shared_attn(int dtype, uint32_t B, uint32_t qH, uint32_t kvH, uint32_t d, uint32_t prefix, uint32_t capacity) {
  SharedPlan a;
  const uint32_t G = qH / kvH;
  a.tensor = dtype != 0 && d <= 128;
  const uint64_t R = (uint64_t)B * G;  // rows of a KV head
  // The walk of the shared rows pays from a length on that makes up for its own two kernels. Measured, without | with it, 16-bit on either
  // side of the rule: 64 sequences of 8 KV heads of 64 behind 430 rows, 16 behind 900, 4 behind 2500 take the same, 32 of 2 of 32 behind
  // 2200, 250 behind 500. float32: 16 sequences of 2 KV heads of 32 behind 1024 rows 12.0 | 10.1 us, 512: 8.4 | 9.8; 2 of 8 of 64 behind 2048:
  // 15.4 | 12.2, 512: 8.5 | 10.0. One sequence gains from it in float32 only, whose other kernel keeps fewer loads on their way (8 KV heads of
  // 128 behind 16384 rows 75.8 | 65.5, 4096: 27.2 | 28.8); in 16 bits that one is at the memory's rate (130000 rows: 82 us of 81).
  const uint64_t work = (uint64_t)prefix * B * kvH * d;
  const bool shared = dtype != 0 ? B >= 2 && d <= 128 && (uint64_t)prefix >= 200 + 6000000 / ((uint64_t)B * kvH * d) : work >= (B == 1 ? 4000000 : 1200000);
  if (shared) {
    const bool umma = dtype != 0;
    a.pre_warps = umma ? 0 : R <= 16 ? 2 : R <= 32 || d > 64 ? 4 : 8;
    // On tcgen05 a CTA has an SM and two tiles of 128 rows (sequence, head of the group), or one tile twice. Up to 64 rows it waits for
    // memory, which 120 SMs keep busy while the own rows are walked on the others: 5 sequences of 32 over 8 heads of 64 behind 100003 rows
    // 40.4 us, on all SMs 42.8; 3 of 16 over 1 of 128 behind 200000 30.2 | 38.0; 16 of 16 of 64 behind 30000 28.9 | 30.5. More rows are bound
    // by what the SMs do (128 sequences of 32 over 8 of 64 behind 20000 on 112 SMs 49.8, all 44.3). On the CUDA cores 16 warps, of 8 rows
    // each, an SM (36 rows in 5 warps of one CTA rather than 8: 48 us for 39; of heads of 128, 4 warps or 8: 33 | 38). As many keys for one
    // CTA as for the others.
    const uint64_t row_tiles = umma ? (R + kPreRows - 1) / kPreRows : (R + a.pre_warps * 8 - 1) / (a.pre_warps * 8);
    const uint64_t groups = (umma ? (row_tiles + 1) / 2 : row_tiles) * kvH, room = umma ? (R <= 64 ? 120 : 148) : 148 * 16 / a.pre_warps;
    const uint32_t tile = umma ? kPreTile : attn_shared_rows_keys(d), tiles = (prefix + tile - 1) / tile;
    uint64_t parts = room / groups;
    parts = parts < 1 ? 1 : parts > kMaxPreSplits ? kMaxPreSplits : parts;
    a.pre_tiles = (uint32_t)((tiles + parts - 1) / parts);
    if (umma && row_tiles == 1 && a.pre_tiles < 2) a.pre_tiles = 2;  // (a tile for each of the CTA's streams)
    a.pre_splits = (tiles + a.pre_tiles - 1) / a.pre_tiles;
  }
  const uint64_t keys = (uint64_t)capacity + (shared ? 0 : prefix);
  a.rows = own_rows_of(a.tensor, G);
  const uint64_t groups = (uint64_t)B * kvH * ((G + a.rows - 1) / a.rows);
  // As many parts as there are CTAs for, where the keys go so far. A part has 128 keys at least where the walk of the
  // shared rows hides the time it takes (8 sequences behind 2011 rows: 11.4 us, 11.9 with 64, 12.3 with 32; 5 behind 100003: 46.3, 45.5,
  // 44.6), 32 where it is all there is (2 sequences of 340 keys and a join: 5.9 us, 6.2 with 64, 6.1 with 128). On the CUDA cores 64, a tile, 32 | 64 |
  // 128: 9 sequences of 8 over 2 heads of 32 behind 1000 rows 11.5 | 8.5 | 9.6, 2 of 8 over 2 of 64 with 340 keys 7.1 | 7.4 | 9.2, in 16 bits 3 of 16
  // over 4 of 256 with 1000 25.1 | 19.6 | 18.1.
  a.own_least = !a.tensor ? 64 : shared ? 128 : kLeastOfAll;
  uint64_t parts = (own_ctas_of(a.tensor) + groups - 1) / groups;
  if (parts > (keys + a.own_least - 1) / a.own_least) parts = (keys + a.own_least - 1) / a.own_least;
  if (parts > kMaxOwnSplits) parts = kMaxOwnSplits;
  // Up to 8 CTAs of a sequence's heads join their parts among each other, as a cluster, and where more are wanted for few keys it is 8: a
  // launch less is worth more to a host that makes the call than what the kernel then takes longer. 2 sequences of 32 over 8 heads of 64 with
  // 428 keys: 11.3 us a call from Python, with a join 13.4; in a graph 6.2 | 6.0 (one with 628: 6.9 | 6.5; with 10500, 16.5 | 10.5). The CUDA
  // cores take too long with fewer CTAs (9 of 8 over 2 of 32 with 1512: 11.0 | 8.5), and behind a walk of the shared rows a cluster
  // waits for room (8 sequences behind 2011 rows: 14.8 | 11.4).
  if (a.tensor && !shared && parts > kMostCtas && keys <= kMostCtas * 128) parts = kMostCtas;
  a.own_splits = parts < 1 ? 1 : (uint32_t)parts;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = (off + bytes + 255) / 256 * 256;
    return at;
  };
  const uint64_t rows = (uint64_t)B * qH;
  // The kernel for the own rows adds the parts of the shared ones to its sums where a CTA has all of a sequence's keys and heads enough to
  // make up for the wait, without a join | with one: 256 sequences of 32 over 8 heads of 64 behind 1500 rows 55.7 | 61.7 us, 128 behind 8000
  // 49.2 | 52.6, 100 of 128 behind 4000 42.6 | 47.7, 64 of 128 behind 16000 (16 parts) 57.7 | 57.7, behind 32768 (18) 72.0 | 68.4; with one
  // head a KV head, 300 of 16 of 64 behind 1500, 52.7 | 44.9. On the CUDA cores it takes registers that the walk needs: 10.8 us for 8.4.
  a.joined = a.own_splits > (shared ? 1 : kMostCtas) || (a.pre_splits && (!a.tensor || G < 4 || a.pre_splits > kFewParts));
  a.pre_ml = take(a.pre_splits * rows * 8);
  a.own_ml = take(a.joined ? a.own_splits * rows * 8 : 0);
  a.pre_o = take(a.pre_splits * rows * d * 4);
  a.own_o = take(a.joined ? a.own_splits * rows * d * 4 : 0);
  a.total = off > 256 ? off : 256;  // (one part per row needs none: a size is never 0)
  return a;
}

// A plan's scratch goes up and down with the sizes: more rows are cut into fewer parts. Of both kinds, rows times parts are bounded:
//   shared rows   parts <= CTAs / (CTAs that have all rows once), and a CTA has 256 rows at most (float32: 16 warps an SM with 8 each);
//   own rows      parts <= CTAs / (CTAs that have all rows once) + 1, and a CTA has own_rows_of rows;
// and parts are no more than tiles of keys. Each bound grows with the batch, the prefix and the capacity.
size_t shared_attn_scratch(int dtype, uint32_t B, uint32_t qH, uint32_t kvH, uint32_t d, uint32_t prefix, uint32_t capacity) {
  const bool tensor = dtype != 0 && d <= 128;
  const uint64_t G = qH / kvH, R = (uint64_t)B * G, rows = (uint64_t)B * qH;
  auto least = [](uint64_t a, uint64_t b) { return a < b ? a : b; };
  auto most = [](uint64_t a, uint64_t b) { return a > b ? a : b; };
  uint64_t pre = 0;
  if (tensor || dtype == 0) {
    const uint64_t tile = tensor ? kPreTile : attn_shared_rows_keys(d), ctas_rows = tensor ? 148 * least(R, 2 * kPreRows) : 148 * 16 * 8;
    pre = least(least((prefix + tile - 1) / tile, kMaxPreSplits) * rows, most(rows, ctas_rows));
  }
  const uint64_t keys = (uint64_t)capacity + prefix, own_rows = least(G, own_rows_of(tensor, (uint32_t)G));
  const uint64_t own = least(least(most(1, (keys + kLeastOfAll - 1) / kLeastOfAll), kMaxOwnSplits) * rows, own_ctas_of(tensor) * own_rows + rows);
  const uint64_t bytes = (pre + own) * (d + 2) * 4 + 4 * 255;  // sums, maxima and sums of weights, each on 256 bytes
  return (bytes + 255) / 256 * 256;
}

cudaError_t launch_shared_attn(cudaStream_t s, int dtype, const SharedAttn& p, const SharedPlan& plan) {
  cudaError_t e = cudaSuccess;
  // Each kernel starts while the one before drains; only the join waits. (The own rows first, so that they are done when the walk of the
  // shared rows has its SMs, which it wants whole: 45.6 us for 43.2 with 5 sequences behind 100003 rows, 77.4 for 74.7 with 64 behind 32768.)
  if (plan.pre_splits) {
    e = plan.pre_warps ? launch_attn_shared_rows(s, p, plan.pre_warps) : launch_attn_shared_umma(s, dtype, p);
    if (e != cudaSuccess) return e;
  }
  if (plan.tensor) e = launch_attn_shared_mma(s, dtype, p, plan.rows);
  else e = dtype == 0 ? launch_own<float>(s, p, plan) : dtype == 1 ? launch_own<__half>(s, p, plan) : launch_own<__nv_bfloat16>(s, p, plan);
  if (e != cudaSuccess || !p.joined) return e;
  return dtype == 0 ? launch_join<float>(s, p) : dtype == 1 ? launch_join<__half>(s, p) : launch_join<__nv_bfloat16>(s, p);
}

}  // namespace nfai

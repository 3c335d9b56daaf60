// The own rows of every sequence (and the shared ones where they are few) on warp-level tensor products: 16-bit types, heads up to 128
// (those that are not 32, 64 or 128 are filled up with zeros to the next of them by the copies).
//
// Bound by HBM: a sequence's rows serve its own query heads only. The query heads of a KV head are the rows of a 16-row tile, both
// products are mma.sync.m16n8k16 with float32 sums, the maximum and the sum of a row run along. A CTA of four warps has one KV head of
// one sequence and a part of its keys, dealt to the warps in slices of 16. Every warp is a pipeline of its own that one lane feeds by
// TMA (as 16-byte copies of all lanes the addresses took more issue slots than the products: 85 against 80 us with 64 sequences behind
// 32768 rows); at the end the warps are joined in shared memory. Rows behind the last that counts may come with a slice: their scores
// are -infinity and their values are overwritten with zeros. Warps that walk whole parts one after the other, asking for the next while
// they multiply this one's last, spare the joining but not the wait for the warp with one part more: 77 us for 68 with 256 sequences.
// A weight is split into two 16-bit terms (two products into one sum): the products wait for memory anyway. In float16 22 bits of it count,
// down to 2^-40 of the row's largest (kLift), in bfloat16 16.
// 256 sequences of 32 heads of 64 with 475 rows of their own on average (and 60 shared ones): 44.4 us, 5.6 TB/s; of 128, 64 sequences: 27.9 us,
// 4.5 TB/s (512 CTAs, three to an SM: the second wave is not full).
#include "attn_shared_common.cuh"

namespace nfai {

namespace {

using namespace shared_attn;
using namespace umma;

constexpr int kMW = 4, kMT = kMW * 32;
constexpr uint32_t kSlice = 16;  // keys per slice
// Weights are multiplied by 2^kLift before they are split (their sum has the factor too): float16, with 2^16 as its largest number, ends at
// 2^-25, so that its second term then reaches down to 2^-40 of a row's largest weight. bfloat16 has float32's range.
template <typename T>
constexpr float kLift = 0.0f;
template <>
constexpr float kLift<__half> = 15.0f;

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
  static constexpr int kStages = 2;  // more of them leave room for fewer CTAs: 79 us with 2, 82 with 3, 93 with 4 (64 sequences behind 32768 rows)
  static constexpr uint32_t kRowBytes = D == 32 ? 64 : 128;              // of a block: 32 or 64 elements, swizzled
  static constexpr uint32_t kBlock = kSlice * kRowBytes;
  static constexpr uint32_t kBlocks = D == 32 ? 1 : D / 64;
  static constexpr uint32_t kHalf = kBlocks * kBlock;                    // a slice of K or V
  static constexpr uint32_t kRing = kMW * kStages * 2 * kHalf;
  static constexpr uint32_t kTotal = kRing + kMW * kStages * 8 + 1024;   // (blocks begin on 1024 bytes)
  // piece c (16 bytes) of row r of a slice
  static __device__ __forceinline__ uint32_t at(uint32_t r, uint32_t c) {
    if constexpr (D == 32) return r * 64 + ((c ^ (r >> 1 & 3)) << 4);
    return (c >> 3) * kBlock + r * 128 + (((c & 7) ^ (r & 7)) << 4);
  }
};

template <int D, int ROWS>
constexpr size_t mma_smem() {  // the stages, or what the warps are joined in
  constexpr size_t join = ((size_t)(kMW + 1) * ROWS * (D + 4) + (kMW + 1) * ROWS * 2) * 4 + 1024;
  static_assert(leave_room(ROWS, kMT) <= kMW * ROWS * (D + 4), "room");
  return Shape<D>::kTotal > join ? Shape<D>::kTotal : join;
}

// ROWS: 8 or 16 query heads
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kMT) attn_shared_mma_kernel(const __grid_constant__ CUtensorMap pre_k, const __grid_constant__ CUtensorMap pre_v,
                                                              const __grid_constant__ CUtensorMap own_k, const __grid_constant__ CUtensorMap own_v,
                                                              const __grid_constant__ SharedAttn p, const uint32_t hgroups) {
  using SH = Shape<D>;
  constexpr int NST = SH::kStages, R = ROWS / 8;
  extern __shared__ unsigned char mma_raw[];
  unsigned char* const sm = reinterpret_cast<unsigned char*>(((uintptr_t)mma_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, qr = lane >> 2, qc = (lane & 3) * 2, G = p.qH / p.kvH;
  const uint32_t hg = blockIdx.x % hgroups, g = blockIdx.x / hgroups % p.kvH, b = blockIdx.x / hgroups / p.kvH, split = blockIdx.y;
  const uint32_t h0 = g * G + hg * ROWS, nh = min((uint32_t)ROWS, G - hg * ROWS);
  const Walk walk = walk_of(p, b, split);
  if (walk.idle || (p.joined && split >= walk.parts)) return leave(p);  // (a cluster's CTA without keys takes part in the join)
  // slices of the shared rows first, then of the sequence's own: none has keys of both
  const uint32_t shared = p.pre_splits ? 0u : p.prefix, cut = min(max(shared, walk.t0), walk.t1);
  const uint32_t before = (cut - walk.t0 + kSlice - 1) / kSlice, slices = before + (walk.t1 - cut + kSlice - 1) / kSlice;
  auto first_of = [&](uint32_t i) { return i < before ? walk.t0 + i * kSlice : cut + (i - before) * kSlice; };
  auto count_of = [&](uint32_t i) { return min(kSlice, (i < before ? cut : walk.t1) - first_of(i)); };
  unsigned char* const stages = sm + warp * NST * 2 * SH::kHalf;
  const uint32_t ring = s_u32(stages), full = s_u32(sm + SH::kRing) + warp * NST * 8;
  if (lane == 0) {
    for (int i = 0; i < NST; ++i) bar_init(full + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  uint32_t fill = 0;
  auto issue = [&](uint32_t i) {
    if (elect_one()) {
      const uint32_t at = ring + fill * 2 * SH::kHalf, bar = full + 8 * fill, t = first_of(i);
      const bool own = i >= before;
      const CUtensorMap *const k = own ? &own_k : &pre_k, *const v = own ? &own_v : &pre_v;
      const int row = (int)(own ? t - shared : t), seq = own ? (int)b : 0;
      bar_expect_tx(bar, 2 * SH::kHalf);
#pragma unroll
      for (uint32_t j = 0; j < SH::kBlocks; ++j) {
        tma_load_4d(at + j * SH::kBlock, k, (int)(j * 64), (int)g, row, seq, bar);
        tma_load_4d(at + SH::kHalf + j * SH::kBlock, v, (int)(j * 64), (int)g, row, seq, bar);
      }
    }
    fill = fill + 1 == NST ? 0 : fill + 1;
  };
#pragma unroll 1
  for (uint32_t i = 0; i < NST - 1; ++i)
    if (warp + i * kMW < slices) issue(warp + i * kMW);
  // lanes of ldmatrix: keys of two position tiles (K), keys of a tile for two pieces of the head (V)
  const uint32_t lm = lane >> 3, lr = lane & 7, k_row = (lm >> 1) * 8 + lr, v_row = (lm & 1) * 8 + lr;
  bool ok = true;
  uint32_t phase = 0;
  uint32_t use = 0;

  // the queries as they are: the left operand, rows beyond the heads zero
  uint32_t q[D / 16][4];
  {
    const T* const at = reinterpret_cast<const T*>(p.q) + ((uint64_t)b * p.qH + h0) * p.d + qc;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t row = qr + (u & 1) * 8, e = kk * 16 + (u >> 1) * 8;
        q[kk][u] = (u & 1) < R && row < nh && e < p.d ? __ldg(reinterpret_cast<const uint32_t*>(at + row * p.d + e)) : 0u;
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
#pragma unroll 1
  for (uint32_t i = warp; i < slices; i += kMW) {
    const uint32_t cnt = count_of(i);
    __syncwarp();  // every lane is past its reads of the stage that is filled next
    if (i + (NST - 1) * kMW < slices && ok) issue(i + (NST - 1) * kMW);
    ok = __all_sync(0xffffffffu, ok && wait_for(full + 8 * use, phase, p.wait_cycles));
    const uint32_t ks = ring + use * 2 * SH::kHalf, vs = ks + SH::kHalf;
    if (cnt < kSlice) {
      unsigned char* const v = stages + (use * 2 + 1) * SH::kHalf;
      for (uint32_t i = lane; i < (kSlice - cnt) * (D / 8); i += 32) *reinterpret_cast<uint4*>(v + SH::at(cnt + i / (D / 8), i % (D / 8))) = make_uint4(0, 0, 0, 0);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (the stage's next copy comes behind these)
      __syncwarp();
    }
    use = use + 1 == NST ? 0 : use + 1;
    if (use == 0) phase ^= 1;
    float s[2][4] = {};
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      uint32_t b0, b1, b2, b3;
      ldsm4(ks + SH::at(k_row, kk * 2 + (lm & 1)), b0, b1, b2, b3);
      Half<T>::mma(s[0], q[kk], b0, b1);
      Half<T>::mma(s[1], q[kk], b2, b3);
    }
    uint32_t hi[4] = {}, lo[4] = {};
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float x[4] = {s[0][2 * r] * p.scale2, s[0][2 * r + 1] * p.scale2, s[1][2 * r] * p.scale2, s[1][2 * r + 1] * p.scale2};
      if (cnt < kSlice) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if ((j >> 1) * 8 + qc + (j & 1) >= cnt) x[j] = -INFINITY;
      }
      float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      top = fmaxf(__fadd_ru(top, -kLift<T>), m[r]);  // (rounded up: no weight is above 2^kLift, however large the scores)
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
      ldsm4t(vs + SH::at(v_row, j + (lm >> 1)), b0, b1, b2, b3);
      Half<T>::mma(o[j], hi, b0, b1);
      Half<T>::mma(o[j + 1], hi, b2, b3);
      Half<T>::mma(o[j], lo, b0, b1);
      Half<T>::mma(o[j + 1], lo, b2, b3);
    }
  }
  if (!ok) {
    if (lane == 0 && p.err) atomicOr(p.err, 4u);
    let_land();
  }
  __syncthreads();  // every warp is past its last read of its stages: the warps' rows go where they were
  constexpr uint32_t PL = D + 4;
  float* const part = reinterpret_cast<float*>(sm);                // [kMW][ROWS][PL]
  float* const rows = part + kMW * ROWS * PL;                      // [ROWS][PL]
  float* const ml = rows + ROWS * PL;                              // [kMW][ROWS][2]
  float* const M = ml + kMW * ROWS * 2;                            // [ROWS], [ROWS]
  float* const L = M + ROWS;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    if (!ok) l[r] = __uint_as_float(0x7fffffffu);
    const uint32_t row = qr + r * 8;
#pragma unroll
    for (int j = 0; j < D / 8; ++j) *reinterpret_cast<float2*>(part + (warp * ROWS + row) * PL + j * 8 + qc) = make_float2(o[j][2 * r], o[j][2 * r + 1]);
    if ((lane & 3) == 0) *reinterpret_cast<float2*>(ml + (warp * ROWS + row) * 2) = make_float2(m[r], l[r]);
  }
  __syncthreads();
  float odd = 0.f;
  for (uint32_t i = tid; i < nh * (D / 4); i += kMT) {
    const uint32_t j = i / (D / 4), e = i % (D / 4) * 4;
    float2 w[kMW];
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < kMW; ++k) {
      w[k] = *reinterpret_cast<const float2*>(ml + (k * ROWS + j) * 2);
      top = fmaxf(top, w[k].x);
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < kMW; ++k) {
      const float f = w[k].x == -INFINITY ? 0.f : s_ex2(w[k].x - top);
      if (f != 0.f || w[k].y != w[k].y) {
        const float4 v = *reinterpret_cast<const float4*>(part + (k * ROWS + j) * PL + e);
        acc.x = fmaf(f, v.x, acc.x); acc.y = fmaf(f, v.y, acc.y); acc.z = fmaf(f, v.z, acc.z); acc.w = fmaf(f, v.w, acc.w);
        sum = fmaf(f, w[k].y, sum);
      }
    }
    *reinterpret_cast<float4*>(rows + j * PL + e) = acc;
    if (is_sum(sum)) note_nan(odd, acc);
    if (e == 0) {
      M[j] = top;
      L[j] = sum;
    }
  }
  if (__syncthreads_or(odd != odd)) {
    mend_part<T, kMT>(p, b, h0, nh, walk.t0, walk.t1, rows, PL, L);
    __syncthreads();
  }
  leave_rows<T, kMT, 8>(p, b, h0, nh, walk, split, rows, PL, M, L, part);  // (the warps' rows have been used)
}

template <typename T, int D, int ROWS>
cudaError_t launch_rows(cudaStream_t s, const SharedAttn& p) {
  constexpr size_t smem = mma_smem<D, ROWS>();
  cudaError_t e = cudaFuncSetAttribute(attn_shared_mma_kernel<T, D, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const uint32_t hgroups = (p.qH / p.kvH + ROWS - 1) / ROWS;
  CUtensorMap pre_k{}, pre_v{}, own_k{}, own_v{};
  constexpr uint32_t kElems = D == 32 ? 32 : 64;
  if (p.prefix && !p.pre_splits && (!encode_cache_map16(&pre_k, p.kp, 1, p.prefix, p.kvH, p.d, kElems, kSlice) || !encode_cache_map16(&pre_v, p.vp, 1, p.prefix, p.kvH, p.d, kElems, kSlice)))
    return cudaErrorInvalidValue;
  if (p.capacity && (!encode_cache_map16(&own_k, p.ko, p.B, p.capacity, p.kvH, p.d, kElems, kSlice) || !encode_cache_map16(&own_v, p.vo, p.B, p.capacity, p.kvH, p.d, kElems, kSlice)))
    return cudaErrorInvalidValue;
  return launch_pdl_cluster(attn_shared_mma_kernel<T, D, ROWS>, dim3(p.B * p.kvH * hgroups, p.own_splits), dim3(kMT), dim3(1, p.joined ? 1 : p.own_splits, 1),
                            smem, s, p.pre_splits != 0, pre_k, pre_v, own_k, own_v, p, hgroups);
}
template <typename T, int D>
cudaError_t launch_d(cudaStream_t s, const SharedAttn& p, uint32_t rows) {
  return rows == 8 ? launch_rows<T, D, 8>(s, p) : launch_rows<T, D, 16>(s, p);
}
template <typename T>
cudaError_t launch_t(cudaStream_t s, const SharedAttn& p, uint32_t rows) {
  if (p.d > 128) return cudaErrorInvalidValue;
  return p.d <= 32 ? launch_d<T, 32>(s, p, rows) : p.d <= 64 ? launch_d<T, 64>(s, p, rows) : launch_d<T, 128>(s, p, rows);
}

}  // namespace

cudaError_t launch_attn_shared_mma(cudaStream_t s, int dtype, const SharedAttn& p, uint32_t rows) {
  return dtype == 1 ? launch_t<__half>(s, p, rows) : dtype == 2 ? launch_t<__nv_bfloat16>(s, p, rows) : cudaErrorInvalidValue;
}

}  // namespace nfai

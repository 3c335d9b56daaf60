// The shared rows, once for every sequence, in true 32 bits: float32 queries and caches on the CUDA cores, any head size.
//
// The query heads of a KV head and the sequences are one list of rows; a warp has eight of them, a CTA up to eight warps on the same tiles
// of keys, which come by cp.async. Of a warp's lanes 16 share four rows: in the first product a lane has their scores with
// every 16th key of the tile, in the second four dimensions (per 64 of the head) of their sums, so that a row's maximum and sum stay
// among 16 lanes and nothing but the tiles is shared between warps. Four float4 of queries and four of keys make 64 multiply-adds, two to an
// instruction (pairs of dimensions); the loads of shared memory meet no bank twice. One tile at a time: what waits for it is covered by
// the SM's other CTAs, of which two buffers leave room for fewer (50 sequences of 6 heads of 128 behind 3800 rows: 44.7 us with two buffers,
// 32.9 with one; 36 of 16 of 64 behind 4000: 76.3 and 72.4). Partial results go to scratch as those of attn_shared_umma.cu.
//
// 15 to 18 TFLOP/s for the whole call with 36 rows and more of a KV head, a quarter of what the multiply-add units do (9 sequences of 32 heads of
// 64 behind 8000 rows: 43 us; 50 of 6 heads of 128 behind 3800: 33 us, where one sequence after another takes 123). Bound by waiting: a tile is
// fetched, then used, ten warps an SM issue in 42 % of the cycles, and what they wait for is the units' and shared memory's latency.
#include "attn_shared_common.cuh"

namespace nfai {

namespace {

using namespace shared_attn;
using namespace umma;

constexpr uint32_t kRowsOf = 8;  // a warp's

// CHUNKS: 64 dimensions each
template <int CHUNKS>
struct RowsShape {
  static constexpr uint32_t kKeys = CHUNKS == 1 ? 64 : 32;  // of a tile
  static constexpr uint32_t kMine = kKeys / 16;             // of them a lane's
  static constexpr uint32_t kPLd = kKeys + 4;
};
__host__ __device__ constexpr uint32_t rows_ld(uint32_t d) { return d + 4; }  // of queries and keys: lanes' rows on other banks
template <int CHUNKS>
size_t rows_smem(uint32_t d, uint32_t warps) {
  using SH = RowsShape<CHUNKS>;
  return ((size_t)warps * kRowsOf * rows_ld(d) + (size_t)SH::kKeys * (rows_ld(d) + d) + (size_t)warps * kRowsOf * SH::kPLd) * 4;
}

__device__ __forceinline__ void cp16(float* dst, const float* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s_u32(dst)), "l"(src), "r"(there ? 16u : 0u) : "memory");
}

template <int CHUNKS>
__global__ void __launch_bounds__(256) attn_shared_rows_kernel(const __grid_constant__ SharedAttn p, const uint32_t row_tiles) {
  using SH = RowsShape<CHUNKS>;
  constexpr uint32_t TK = SH::kKeys, NK = SH::kMine;
  extern __shared__ __align__(16) float rows_sm[];
  const uint32_t d = p.d, ld = rows_ld(d), d4 = d / 4, warps = blockDim.x / 32, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rg = lane >> 4, kg = lane & 15;
  float* const q = rows_sm;                                  // [warps * 8][ld], scaled
  float* const tiles = q + warps * kRowsOf * ld;             // of K [TK][ld] and V [TK][d]
  float* const w = tiles + TK * (ld + d) + warp * kRowsOf * SH::kPLd;  // this warp's weights [8][kPLd]
  const uint32_t G = p.qH / p.kvH, R = p.B * G, tile = blockIdx.x % row_tiles, g = blockIdx.x / row_tiles % p.kvH, split = blockIdx.x / row_tiles / p.kvH;
  const uint32_t row0 = tile * warps * kRowsOf, t0 = split * p.pre_tiles * TK, t1 = min(p.prefix, t0 + p.pre_tiles * TK), n = (t1 - t0 + TK - 1) / TK;
  pdl_launch_dependents();
  auto issue = [&](uint32_t it) {
    float* const k = tiles;
    float* const v = k + TK * ld;
    for (uint32_t i = tid; i < TK * d4; i += blockDim.x) {
      const uint32_t r = i / d4, e = (i - r * d4) * 4, t = t0 + it * TK + r;
      const bool in = t < t1;
      const uint64_t at = ((uint64_t)(in ? t : t0) * p.kvH + g) * d + e;  // (a row that is there even where nothing is copied)
      cp16(k + r * ld + e, reinterpret_cast<const float*>(p.kp) + at, in);
      cp16(v + r * d + e, reinterpret_cast<const float*>(p.vp) + at, in);
    }
  };
  for (uint32_t i = tid; i < warps * kRowsOf * d4; i += blockDim.x) {
    const uint32_t r = i / d4, e = (i - r * d4) * 4, row = row0 + r, b = row / G;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < R) v = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.q) + ((uint64_t)b * p.qH + g * G + (row - b * G)) * d + e));
    *reinterpret_cast<float4*>(q + r * ld + e) = make_float4(v.x * p.scale2, v.y * p.scale2, v.z * p.scale2, v.w * p.scale2);
  }
  const float* const my_q = q + (warp * kRowsOf + rg * 4) * ld;
  float m[4], l[4];
  uint64_t o[4][CHUNKS][2];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) o[r][c][0] = o[r][c][1] = 0;
  }
  const bool busy = row0 + warp * kRowsOf < R;

  for (uint32_t it = 0; it < n; ++it) {
    issue(it);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // everyone's part of this tile is there (and the queries are)
    const float* const k = tiles;
    const float* const v = k + TK * ld;
    if (busy) {
      uint64_t s2[4][NK];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (uint32_t j = 0; j < NK; ++j) s2[r][j] = 0;
#pragma unroll 2
      for (uint32_t e = 0; e < d; e += 4) {
        ulonglong2 qv[4], kv[NK];
#pragma unroll
        for (int r = 0; r < 4; ++r) qv[r] = *reinterpret_cast<const ulonglong2*>(my_q + r * ld + e);
#pragma unroll
        for (uint32_t j = 0; j < NK; ++j) kv[j] = *reinterpret_cast<const ulonglong2*>(k + (j * 16 + kg) * ld + e);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (uint32_t j = 0; j < NK; ++j) s2[r][j] = fma2(qv[r].y, kv[j].y, fma2(qv[r].x, kv[j].x, s2[r][j]));
      }
      const uint32_t n0 = t0 + it * TK;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float s[NK], top = m[r];
#pragma unroll
        for (uint32_t j = 0; j < NK; ++j) {
          float a, b;
          unpair(s2[r][j], a, b);
          s[j] = n0 + j * 16 + kg < t1 ? a + b : -INFINITY;
          top = fmaxf(top, s[j]);
        }
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float ref = top == -INFINITY ? 0.f : top, f = exp2f(m[r] - ref);
        m[r] = top;
        float sum = 0.f;
#pragma unroll
        for (uint32_t j = 0; j < NK; ++j) {
          const float x = exp2f(s[j] - ref);
          w[(rg * 4 + r) * SH::kPLd + j * 16 + kg] = x;
          sum += x;
        }
        l[r] = l[r] * f + sum;
        const uint64_t f2 = pair(f, f);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          o[r][c][0] = fma2(o[r][c][0], f2, 0);
          o[r][c][1] = fma2(o[r][c][1], f2, 0);
        }
      }
      __syncwarp();
#pragma unroll 2
      for (uint32_t j = 0; j < TK; j += 4) {
        float4 x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = *reinterpret_cast<const float4*>(w + (rg * 4 + r) * SH::kPLd + j);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          const uint32_t e = c * 64 + kg * 4;
          if (e >= d) continue;
          ulonglong2 vv[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) vv[t] = *reinterpret_cast<const ulonglong2*>(v + (j + t) * d + e);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint64_t x0 = pair(x[r].x, x[r].x), x1 = pair(x[r].y, x[r].y), x2 = pair(x[r].z, x[r].z), x3 = pair(x[r].w, x[r].w);
            o[r][c][0] = fma2(x3, vv[3].x, fma2(x2, vv[2].x, fma2(x1, vv[1].x, fma2(x0, vv[0].x, o[r][c][0]))));
            o[r][c][1] = fma2(x3, vv[3].y, fma2(x2, vv[2].y, fma2(x1, vv[1].y, fma2(x0, vv[0].y, o[r][c][1]))));
          }
        }
      }
      __syncwarp();  // (the weights are overwritten next)
    }
    __syncthreads();  // the tile has been used: the next may land there
  }
  float odd = 0.f;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
    const uint32_t row = row0 + warp * kRowsOf + rg * 4 + r;
    if (row >= R) continue;
    const uint64_t at = ((uint64_t)split * p.kvH + g) * R + row;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const uint32_t e = c * 64 + kg * 4;
      if (e >= d) continue;
      float4 y;
      unpair(o[r][c][0], y.x, y.y);
      unpair(o[r][c][1], y.z, y.w);
      *reinterpret_cast<float4*>(p.pre_o + at * d + e) = y;
      if (is_sum(l[r])) note_nan(odd, y);
    }
    if (kg == 0) *reinterpret_cast<float2*>(p.pre_ml + at * 2) = make_float2(m[r], l[r]);
  }
  const bool mend = __any_sync(0xffffffffu, odd != odd);
  __syncwarp();
  if (mend) mend_shared<float>(p, split, g, row0 + warp * kRowsOf, min(R, row0 + (warp + 1) * kRowsOf), t0, t1, 0, 1);
}

template <int CHUNKS>
cudaError_t launch_pre(cudaStream_t s, const SharedAttn& p, uint32_t warps) {
  const size_t smem = rows_smem<CHUNKS>(p.d, warps);
  cudaError_t e = cudaFuncSetAttribute(attn_shared_rows_kernel<CHUNKS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const uint64_t row_tiles = ((uint64_t)p.B * (p.qH / p.kvH) + warps * kRowsOf - 1) / (warps * kRowsOf), grid = row_tiles * p.kvH * p.pre_splits;
  if (grid > 0x7fffffffu) return cudaErrorInvalidValue;
  attn_shared_rows_kernel<CHUNKS><<<(unsigned)grid, warps * 32, smem, s>>>(p, (uint32_t)row_tiles);
  return cudaGetLastError();
}
}  // namespace

uint32_t attn_shared_rows_keys(uint32_t d) { return d <= 64 ? RowsShape<1>::kKeys : RowsShape<2>::kKeys; }

cudaError_t launch_attn_shared_rows(cudaStream_t s, const SharedAttn& p, uint32_t warps) {
  return p.d <= 64 ? launch_pre<1>(s, p, warps) : p.d <= 128 ? launch_pre<2>(s, p, warps) : launch_pre<4>(s, p, warps);
}

}  // namespace nfai

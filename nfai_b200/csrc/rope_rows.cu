// Rotary positions for a batch of tokens, each at a position of its own, queries to a buffer and keys and values to cache rows.
//
// y = turn(position * f_i) x for the pairs i of the first `dims` elements of every query and key head, times a magnitude; the other
// elements and the values are only converted. The angle is formed in 64 bits and brought into half a turn there (at position
// 1 000 000 a float32 angle is off by 0.06 radians), sine and cosine of the rest in float32.
//
// Bound by HBM: every element is read and written once. A CTA owns whole rows; a thread takes units of eight elements of a head
// (pairs layout) or eight elements and the eight they are paired with (halves), asks for its first unit before the CTA forms the
// rows' cosines and sines in shared memory, and so waits once for both. 9472 rows of 32 + 16 heads of 128, float32 to bfloat16: 54.4 us,
// 6.4 TB/s, what a copy reaches (65 us with two units asked for: fewer CTAs fit; 71 with 128 threads); one row 2.4 us.
//
// Reference arithmetic extended: RoPEShader (NFAI.Vulkan.Shaders/RoPEShader.cs:238-271), one row, pairs, float32 angles.
#include "answers.h"
#include "common.cuh"
#include "kernels.h"

namespace nfai {

namespace {

constexpr int kRT = 256;   // threads
constexpr int kAhead = 1;  // units per thread asked for before the cosines are formed
constexpr uint32_t kMaxTable = 4096;  // cosine and sine pairs in shared memory (32 KB)

// cos and sin of pos * f, pos * f reduced to (-pi, pi] in 64 bits
__device__ __forceinline__ float2 turn_of(int32_t pos, double f, float magnitude) {
  const double turns = (double)pos * (f * 0.15915494309189533577);
  float s, c;
  sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
  return make_float2(c * magnitude, s * magnitude);
}

// SECTORS: float32 buffers and rows begin on 32 bytes
template <typename T, bool SECTORS>
struct Vec8 {  // eight elements as they lie in memory
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(T) == 4 && SECTORS) {  // 32 bytes in one request: a whole sector per thread
      asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=r"(w[0].x), "=r"(w[0].y), "=r"(w[0].z), "=r"(w[0].w), "=r"(w[1].x), "=r"(w[1].y), "=r"(w[1].z), "=r"(w[1].w)
                   : "l"(p));
    } else {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = ld_stream16(reinterpret_cast<const uint4*>(p) + i);
    }
  }
  __device__ __forceinline__ void widen(float (&f)[8]) const {
    if constexpr (sizeof(T) == 4) {
      const uint32_t u[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(u[i]);
    } else {
      WeightVec<T>::unpack(w[0], f);
    }
  }
};
template <bool SECTORS>
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  if constexpr (!SECTORS) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    return;
  }
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(__float_as_uint(f[0])), "r"(__float_as_uint(f[1])),
               "r"(__float_as_uint(f[2])), "r"(__float_as_uint(f[3])), "r"(__float_as_uint(f[4])), "r"(__float_as_uint(f[5])),
               "r"(__float_as_uint(f[6])), "r"(__float_as_uint(f[7]))
               : "memory");
}
template <bool SECTORS, typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  alignas(16) T h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) store_as(h + i, f[i]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
}

// Where an element of row r goes; null: nowhere (a slot outside the cache).
template <typename OT>
__device__ __forceinline__ OT* place(const RopeRows& p, uint32_t r, uint32_t head, uint32_t e) {
  if (head < p.qH) return reinterpret_cast<OT*>(p.q) + ((uint64_t)r * p.qH + head) * p.d + e;
  const int64_t slot = p.slots ? (int64_t)p.slots[r] : (int64_t)r;
  if (slot < 0 || (uint64_t)slot >= p.cache_rows) return nullptr;
  head -= p.qH;
  const bool value = head >= p.kvH;
  return reinterpret_cast<OT*>(value ? p.v : p.k) + ((uint64_t)slot * p.kvH + (value ? head - p.kvH : head)) * p.d + e;
}

template <typename XT, typename OT, bool HALVES, bool SECTORS>
__global__ void __launch_bounds__(kRT) rope_rows_kernel(const RopeRows p, const uint32_t rows_per_cta) {
  extern __shared__ float2 table[];  // [rows_per_cta][dims / 2]
  const uint32_t r0 = blockIdx.x * rows_per_cta, n = min(rows_per_cta, p.rows - r0), half = p.dims / 2;
  // units of a head: turned ones first, then plain ones
  const uint32_t turned = HALVES ? half / 8 : p.dims / 8, plain = (p.d - p.dims) / 8, whole = p.d / 8;
  const uint32_t qk_units = (p.qH + p.kvH) * (turned + plain), units = qk_units + p.kvH * whole, total = n * units;
  const XT* const x = reinterpret_cast<const XT*>(p.x);
  struct Unit {
    uint32_t r, head, e, i;  // i: its first pair; pairs of no turn: ~0
  };
  auto unit = [&](uint32_t u) {
    Unit a;
    const uint32_t lr = u / units;
    u -= lr * units;
    a.r = r0 + lr;
    if (u < qk_units) {
      a.head = u / (turned + plain);
      u -= a.head * (turned + plain);
      const bool t = u < turned;
      a.e = t ? u * 8 : p.dims + (u - turned) * 8;
      a.i = t ? (HALVES ? u * 8 : u * 4) : ~0u;
    } else {
      u -= qk_units;
      a.head = p.qH + p.kvH + u / whole;
      a.e = u % whole * 8;
      a.i = ~0u;
    }
    return a;
  };
  Vec8<XT, SECTORS> va[kAhead], vb[HALVES ? kAhead : 1];
  auto fetch = [&](const Unit& a, Vec8<XT, SECTORS>& lo, Vec8<XT, SECTORS>& hi) {
    const XT* at = x + (uint64_t)a.r * p.x_stride + (uint64_t)a.head * p.d + a.e;
    lo.load(at);
    if (HALVES && a.i != ~0u) hi.load(at + half);
  };
  auto finish = [&](const Unit& a, const Vec8<XT, SECTORS>& lo, const Vec8<XT, SECTORS>& hi) {
    OT* const to = place<OT>(p, a.r, a.head, a.e);
    float f[8];
    lo.widen(f);
    if (a.i == ~0u) {
      if (to) store8<SECTORS>(to, f);
      return;
    }
    const float2* const cs = table + (a.r - r0) * half + a.i;
    if constexpr (HALVES) {
      float g[8], y[8], z[8];
      hi.widen(g);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 t = cs[i];
        y[i] = f[i] * t.x - g[i] * t.y;
        z[i] = f[i] * t.y + g[i] * t.x;
      }
      if (to) {
        store8<SECTORS>(to, y);
        store8<SECTORS>(to + half, z);
      }
    } else {
      float y[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 t = cs[i];
        y[2 * i] = f[2 * i] * t.x - f[2 * i + 1] * t.y;
        y[2 * i + 1] = f[2 * i] * t.y + f[2 * i + 1] * t.x;
      }
      if (to) store8<SECTORS>(to, y);
    }
  };
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const uint32_t u = threadIdx.x + k * kRT;
    if (u < total) fetch(unit(u), va[k], vb[HALVES ? k : 0]);
  }
  for (uint32_t j = threadIdx.x; j < n * half; j += kRT) {
    const uint32_t lr = j / half, i = j - lr * half;
    table[j] = turn_of(p.positions[r0 + lr], p.freqs[i], p.magnitude);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const uint32_t u = threadIdx.x + k * kRT;
    if (u < total) finish(unit(u), va[k], vb[HALVES ? k : 0]);
  }
  for (uint32_t u = threadIdx.x + kAhead * kRT; u < total; u += kRT) {
    const Unit a = unit(u);
    fetch(a, va[0], vb[0]);
    finish(a, va[0], vb[0]);
  }
}

// Any sizes, strides and alignment: a thread per element.
template <typename XT, typename OT, bool HALVES>
__global__ void __launch_bounds__(kRT) rope_rows_any_kernel(const RopeRows p) {
  const uint32_t heads = p.qH + 2 * p.kvH, half = p.dims / 2;
  const uint64_t per_row = (uint64_t)heads * p.d, total = per_row * p.rows;
  for (uint64_t j = (uint64_t)blockIdx.x * kRT + threadIdx.x; j < total; j += (uint64_t)gridDim.x * kRT) {
    const uint32_t r = (uint32_t)(j / per_row), w = (uint32_t)(j - r * per_row), head = w / p.d, e = w - head * p.d;
    OT* const to = place<OT>(p, r, head, e);
    if (!to) continue;
    const XT* const at = reinterpret_cast<const XT*>(p.x) + (uint64_t)r * p.x_stride + (uint64_t)head * p.d;
    float y = to_float(at[e]);
    if (head < p.qH + p.kvH && e < p.dims) {
      const uint32_t i = HALVES ? (e < half ? e : e - half) : e / 2;
      const bool first = HALVES ? e < half : (e & 1) == 0;
      const float other = to_float(at[HALVES ? (first ? e + half : e - half) : e ^ 1]);
      const float2 t = turn_of(p.positions[r], p.freqs[i], p.magnitude);
      y = first ? y * t.x - other * t.y : other * t.y + y * t.x;
    }
    store_as(to, y);
  }
}

template <typename XT, typename OT, bool HALVES>
cudaError_t launch_layout(cudaStream_t s, const RopeRows& p) {
  // Eight elements at a time where rows begin on 16 bytes, in float32 whole sectors where they begin on 32. 2011 rows of 32 + 16 heads of 64
  // on odd multiples of 16 bytes, in L2, halves: 16-bit 8.4 us, an element at a time 39.1; float32 12.6, an element at a time 38.6, on multiples
  // of 32 bytes 9.2.
  const uintptr_t in = (uintptr_t)p.x | p.x_stride * sizeof(XT), out = (uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v;
  const bool wide = ((in | out) & 15) == 0 && p.d % 8 == 0 && p.dims % (HALVES ? 16 : 8) == 0 && p.dims / 2 <= kMaxTable;
  const bool sectors = ((sizeof(XT) == 4 ? in : 0) | (sizeof(OT) == 4 ? out : 0)) % 32 == 0;
  if (!wide) {
    const uint64_t total = (uint64_t)p.rows * (p.qH + 2 * p.kvH) * p.d, blocks = (total + kRT - 1) / kRT;
    rope_rows_any_kernel<XT, OT, HALVES><<<(unsigned)(blocks < 148 * 32 ? blocks : 148 * 32), kRT, 0, s>>>(p);
    return cudaGetLastError();
  }
  const uint32_t qk = (HALVES ? p.dims / 16 : p.dims / 8) + (p.d - p.dims) / 8;
  const uint32_t units = (p.qH + p.kvH) * qk + p.kvH * (p.d / 8);
  uint32_t per = kRT / units;  // short rows share a CTA
  if (per > 1 && p.dims) per = per < kMaxTable / (p.dims / 2) ? per : kMaxTable / (p.dims / 2);
  if (per < 1) per = 1;
  const size_t smem = (size_t)per * (p.dims / 2) * sizeof(float2);
  if constexpr (sizeof(XT) == 4 || sizeof(OT) == 4) {
    if (!sectors) {
      rope_rows_kernel<XT, OT, HALVES, false><<<(p.rows + per - 1) / per, kRT, smem, s>>>(p, per);
      return cudaGetLastError();
    }
  }
  rope_rows_kernel<XT, OT, HALVES, true><<<(p.rows + per - 1) / per, kRT, smem, s>>>(p, per);
  return cudaGetLastError();
}
template <typename XT, typename OT>
cudaError_t launch_types(cudaStream_t s, const RopeRows& p) {
  return p.halves ? launch_layout<XT, OT, true>(s, p) : launch_layout<XT, OT, false>(s, p);
}
template <typename XT>
cudaError_t launch_x(cudaStream_t s, int out_dtype, const RopeRows& p) {
  switch (out_dtype) {
    case 0: return launch_types<XT, float>(s, p);
    case 1: return launch_types<XT, __half>(s, p);
    case 2: return launch_types<XT, __nv_bfloat16>(s, p);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace

cudaError_t launch_rope_rows(cudaStream_t s, int x_dtype, int out_dtype, const RopeRows& p) {
  switch (x_dtype) {
    case 0: return launch_x<float>(s, out_dtype, p);
    case 1: return launch_x<__half>(s, out_dtype, p);
    case 2: return launch_x<__nv_bfloat16>(s, out_dtype, p);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace nfai

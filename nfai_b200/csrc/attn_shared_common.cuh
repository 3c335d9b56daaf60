// What the kernels of attn_shared.cu share: which rows a sequence attends over, and how partial results become a row of the output.
//
// A partial result of one query head is (o[d], m, l): m the largest score (base 2) among its keys, l = sum 2^(s - m), o = sum 2^(s - m) v.
// No keys, or keys whose scores are all -infinity: m = -infinity, l = 0. Several are joined as
//   M = max m_i,  out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i
// in an order that follows from their indices alone: the same call gives the same bits.
#pragma once
#include "answers.h"
#include "common.cuh"
#include "kernels.h"
#include "umma.cuh"

namespace nfai {
namespace shared_attn {

constexpr uint32_t kMaxOwnSplits = 148;   // parts a sequence's keys are cut into
constexpr uint32_t kMaxPreSplits = 148;   // CTAs that the shared rows are divided among
constexpr uint32_t kFewParts = 16;        // parts of the shared rows that the kernel for the own rows adds by itself
constexpr uint32_t kMostCtas = 8;         // of a sequence's heads that join their parts in a cluster
constexpr uint32_t kPreRows = 128;        // (sequence, head of the group) of a CTA that walks the shared rows
constexpr uint32_t kPreTile = 128;        // ... and its keys per tile

__device__ __forceinline__ float s_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bounded waits as in umma.cuh, with the context's budget. It is counted in cycles (two a nanosecond), whose counter is read in a few of
// them (the nanosecond timer takes longer than some of these waits); 32 bits of it are enough for two seconds. How long one try may sleep is
// up to the hardware, so the barrier is asked without sleeping first: a budget of a few cycles is kept too.
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, uint32_t cycles) {
  if (bar_test(bar, parity)) return true;
  const uint32_t t0 = clock();
  do {
    if ((uint32_t)clock() - t0 > cycles) return false;
  } while (!umma::bar_try(bar, parity));
  return true;
}
// Where one gave up: a millisecond, for copies and products that are on their way to end before their memory is used for something else. (They
// take some microseconds.)
__device__ __forceinline__ void let_land() {
  const long long t0 = clock64();
  while (clock64() - t0 < 2000000ll) {
  }
}
__device__ __forceinline__ bool all_wait_for(uint32_t bar, uint32_t parity, uint32_t cycles) { return __all_sync(0xffffffffu, wait_for(bar, parity, cycles)); }

// The walk of one CTA: keys [t0, t1) of sequence b's n, the shared rows first unless they have kernels of their own.
struct Walk {
  uint32_t n, t0, t1, parts;  // parts: CTAs that this sequence's keys are divided among
  bool idle;
};
__device__ __forceinline__ Walk walk_of(const SharedAttn& p, uint32_t b, uint32_t split) {
  Walk w;
  const int32_t len = p.lens[b];
  w.idle = len < 0;
  const uint32_t own = w.idle ? 0u : min((uint32_t)len, p.capacity);
  w.n = own + (p.pre_splits ? 0u : p.prefix);
  const uint32_t chunk = max(p.own_least, ((w.n + p.own_splits - 1) / p.own_splits + 15) / 16 * 16);
  w.parts = max(1u, (w.n + chunk - 1) / chunk);
  w.t0 = min(w.n, split * chunk);
  w.t1 = min(w.n, w.t0 + chunk);
  return w;
}
// A CTA's way out. The join starts when this grid has ended and counts on the walk of the shared rows to have ended too: the last CTA
// sees to that.
__device__ __forceinline__ void leave(const SharedAttn& p) {
  if (p.joined) pdl_launch_dependents();
  if (p.pre_splits && blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1) pdl_wait();
}
// Offset of key t of sequence b: in the shared rows, or in the sequence's own (`own` set).
__device__ __forceinline__ uint64_t key_row(const SharedAttn& p, uint32_t b, uint32_t t, bool& own) {
  const uint32_t shared = p.pre_splits ? 0u : p.prefix;
  own = t >= shared;
  return own ? (uint64_t)b * p.capacity + (t - shared) : (uint64_t)t;
}

// ---- infinite values ----
// A sum of weighted values comes out as no number where an infinite value meets a weight, or a term of one, that is 0 in the type of the
// product: the second term of a weight that is exact, a key that belongs to another copy of the row, a weight that is too small for float16.
// Weights are above 0, so infinities of one sign are the sum, and those of both signs or a NaN are none. Which it is follows from the column of
// values alone; the kernels look at it again, for the keys of their part, where a row whose weights' sum is a number has such an element. (Only
// there: a free place of the batch may hold queries that are no numbers.)
// `acc` becomes NaN where one of the four is
__device__ __forceinline__ void note_nan(float& acc, float4 v) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(acc) : "f"(v.x));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(acc) : "f"(v.y));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(acc) : "f"(v.z));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(acc) : "f"(v.w));
}
__device__ __forceinline__ bool is_sum(float l) { return l > 0.f && l < INFINITY; }
// Of n values a `step` apart: 1: +infinity is among them, 2: -infinity, 4: NaN. For a whole warp.
template <typename T>
__device__ __forceinline__ uint32_t infinities(const T* v, uint64_t step, uint32_t n) {
  const uint32_t lane = threadIdx.x & 31;
  uint32_t f = 0;
#pragma unroll 1
  for (uint32_t t0 = 0; t0 < n && !__any_sync(0xffffffffu, f & 4); t0 += 128) {
    float x[4];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) x[k] = t0 + k * 32 + lane < n ? to_float(v[(t0 + k * 32 + lane) * step]) : 0.f;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) f |= x[k] == INFINITY ? 1u : x[k] == -INFINITY ? 2u : x[k] != x[k] ? 4u : 0u;
  }
  return __reduce_or_sync(0xffffffffu, f);
}
__device__ __forceinline__ float infinite_sum(uint32_t f) { return f == 1 ? INFINITY : f == 2 ? -INFINITY : __uint_as_float(0x7fffffffu); }

// The keys [t0, t1) of sequence b: rows[j][d] (stride ld) and l[j] of its nh query heads from h0 on, which are one KV head's, in shared memory.
// For a whole CTA. (A function of its own: the kernels keep the registers that they have without it.)
template <typename T, int THREADS>
__device__ __noinline__ void mend_part(const SharedAttn& p, uint32_t b, uint32_t h0, uint32_t nh, uint32_t t0, uint32_t t1, float* rows, uint32_t ld,
                                       const float* l) {
  const uint32_t d = p.d, lane = threadIdx.x & 31, shared = p.pre_splits ? 0u : p.prefix, cut = min(max(shared, t0), t1);
  const uint64_t step = (uint64_t)p.kvH * d, column = (uint64_t)(h0 / (p.qH / p.kvH)) * d;
  for (uint32_t e = threadIdx.x >> 5; e < d; e += THREADS / 32) {
    const bool odd = lane < nh && is_sum(l[lane]) && rows[lane * ld + e] != rows[lane * ld + e];
    if (!__any_sync(0xffffffffu, odd)) continue;
    const T* const vp = reinterpret_cast<const T*>(p.vp) + t0 * step + column + e;
    const T* const vo = reinterpret_cast<const T*>(p.vo) + ((uint64_t)b * p.capacity + (max(cut, shared) - shared)) * step + column + e;
    const uint32_t f = infinities(vp, step, cut - t0) | infinities(vo, step, t1 - cut);
    if (odd) rows[lane * ld + e] = infinite_sum(f);
  }
}
// The shared keys [t0, t1) of KV head g: rows [r0, r1) of part `split`, in scratch, written by this CTA (or, with one warp, by this warp).
template <typename T>
__device__ __noinline__ void mend_shared(const SharedAttn& p, uint32_t split, uint32_t g, uint32_t r0, uint32_t r1, uint32_t t0, uint32_t t1, uint32_t warp,
                                         uint32_t warps) {
  const uint32_t d = p.d, lane = threadIdx.x & 31;
  const uint64_t at = ((uint64_t)split * p.kvH + g) * p.B * (p.qH / p.kvH), step = (uint64_t)p.kvH * d;
  for (uint32_t e = warp; e < d; e += warps) {
    uint32_t f = ~0u;  // not looked at yet
    for (uint32_t r = r0; r < r1; r += 32) {
      float* const o = p.pre_o + (at + r + lane) * d + e;
      const bool odd = r + lane < r1 && is_sum(__ldcg(p.pre_ml + (at + r + lane) * 2 + 1)) && __ldcg(o) != __ldcg(o);
      if (!__any_sync(0xffffffffu, odd)) continue;
      if (f == ~0u) f = infinities(reinterpret_cast<const T*>(p.vp) + t0 * step + (uint64_t)g * d + e, step, t1 - t0);
      if (odd) *o = infinite_sum(f);
    }
  }
}

// A number, or four, of another CTA of the cluster
__device__ __forceinline__ float ld_far(const float* at, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(umma::s_u32(at)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

// Everything a CTA does behind its walk: rows[j][d] (stride ld), m[j], l[j] of its query heads h0 .. h0 + nh - 1 are in shared memory,
// all of it written and synchronised. They go to scratch for the join, or the CTAs of a sequence's heads, which are a cluster then, join
// them among each other, with what the shared rows gave where those have a kernel of their own: every CTA a share of the output.
// AHEAD: parts that are asked for at once. room: leave_room(..) floats of shared memory, free and aligned to 16 bytes.
__host__ __device__ constexpr uint32_t leave_room(uint32_t rows, uint32_t threads) { return (rows * (kFewParts + kMostCtas + 1) + 3) / 4 * 4 + threads * 4; }
template <typename T, int THREADS, int AHEAD>
__device__ __forceinline__ void leave_rows(const SharedAttn& p, uint32_t b, uint32_t h0, uint32_t nh, const Walk& w, uint32_t split,
                                           const float* rows, uint32_t ld, const float* m, const float* l, float* room) {
  const uint32_t tid = threadIdx.x, d = p.d, d4 = d / 4, row0 = b * p.qH + h0;
  if (p.joined) {
    const uint64_t at = (uint64_t)split * p.B * p.qH + row0;
    for (uint32_t i = tid; i < nh * d4; i += THREADS) {
      const uint32_t j = i / d4, e = (i - j * d4) * 4;
      *reinterpret_cast<float4*>(p.own_o + (at + j) * d + e) = *reinterpret_cast<const float4*>(rows + j * ld + e);
    }
    if (tid < nh) *reinterpret_cast<float2*>(p.own_ml + (at + tid) * 2) = make_float2(m[tid], l[tid]);
    leave(p);
    return;
  }
  T* const out = reinterpret_cast<T*>(p.out) + (uint64_t)row0 * d;
  auto store = [&](uint32_t j, uint32_t e, float4 v, float f) {
    alignas(16) T y[4];
    store_as(y, v.x * f);
    store_as(y + 1, v.y * f);
    store_as(y + 2, v.z * f);
    store_as(y + 3, v.w * f);
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out + j * d + e) = *reinterpret_cast<const float4*>(y);
    else *reinterpret_cast<uint2*>(out + j * d + e) = *reinterpret_cast<const uint2*>(y);
  };
  const uint32_t n = p.pre_splits, ctas = p.own_splits, all = n + ctas;  // parts: the shared rows', then the CTAs' own
  if (all == 1) {
    for (uint32_t i = tid; i < nh * d4; i += THREADS) {
      const uint32_t j = i / d4, e = (i - j * d4) * 4;
      store(j, e, *reinterpret_cast<const float4*>(rows + j * ld + e), w.n ? 1.0f / l[j] : 0.f);  // (no keys at all: zeros; none with a weight: 0 * infinity)
    }
    return;
  }
  if (ctas > 1) umma::cluster_sync();
  if (n) pdl_wait();  // (of a part of the shared rows the CTA's heads stand one after the other)
  const uint32_t G = p.qH / p.kvH, g = h0 / G, warp = tid >> 5, lane = tid & 31;
  const uint64_t R = (uint64_t)p.B * G, step = p.kvH * R, at0 = (uint64_t)g * R + (uint64_t)b * G + (h0 - g * G);
  float* const f = room;                // [nh][all]: the parts' factors
  float* const inv = room + nh * all;   // [nh]
  float4* const half = reinterpret_cast<float4*>(room + (nh * (all + 1) + 3) / 4 * 4);
  for (uint32_t j = warp; j < nh; j += THREADS / 32) {
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < n) ml = __ldcg(reinterpret_cast<const float2*>(p.pre_ml + (lane * step + at0 + j) * 2));
    else if (ctas == 1 && lane == n) ml = make_float2(m[j], l[j]);
    else if (lane < all) ml = make_float2(ld_far(m + j, lane - n), ld_far(l + j, lane - n));
    const float top = warp_max(ml.x), ref = top == -INFINITY ? 0.f : top, x = exp2f(ml.x - ref);
    if (lane < all) f[j * all + lane] = x;
    // (a part without weights: nothing of it counts, but a sum that is not a number does)
    const float total = warp_sum(x != 0.f || ml.y != ml.y ? x * ml.y : 0.f);
    if (lane == 0) inv[j] = w.n || n ? 1.0f / total : 0.f;
  }
  __syncthreads();
  // This CTA's share: a thread has four dimensions of a head; where threads are left, they share its parts.
  const uint32_t units = nh * d4, from = split * units / ctas, mine = (split + 1) * units / ctas - from;
  const uint32_t sets = mine && mine < THREADS ? THREADS / mine : 1u, set = sets > 1 ? tid / mine : 0u, first = sets > 1 ? tid - set * mine : tid;
  for (uint32_t i = first; i < mine && set < sets; i += sets > 1 ? mine : THREADS) {
    const uint32_t j = (from + i) / d4, e = (from + i - j * d4) * 4;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t k0 = set; k0 < all; k0 += AHEAD * sets) {
      float4 v[AHEAD];
#pragma unroll
      for (uint32_t k = 0; k < AHEAD; ++k) {
        const uint32_t part = k0 + k * sets;
        if (part < n) v[k] = __ldcg(reinterpret_cast<const float4*>(p.pre_o + (part * step + at0 + j) * d + e));
        else if (ctas == 1 && part == n) v[k] = *reinterpret_cast<const float4*>(rows + j * ld + e);
        else if (part < all) v[k] = umma::ld_cluster(umma::s_u32(rows + j * ld + e), part - n);
      }
#pragma unroll
      for (uint32_t k = 0; k < AHEAD; ++k) {
        const uint32_t part = k0 + k * sets;
        const float x = part < all ? f[j * all + part] : 0.f;
        if (x != 0.f) {
          acc.x = fmaf(x, v[k].x, acc.x); acc.y = fmaf(x, v[k].y, acc.y); acc.z = fmaf(x, v[k].z, acc.z); acc.w = fmaf(x, v[k].w, acc.w);
        }
      }
    }
    if (sets > 1) half[tid] = acc;
    else store(j, e, acc, inv[j]);
  }
  if (ctas > 1) umma::cluster_sync();  // (nobody leaves while others read its rows; and what follows is behind a barrier)
  else __syncthreads();
  if (sets > 1 && tid < mine) {
    float4 acc = half[tid];
    for (uint32_t k = 1; k < sets; ++k) {
      const float4 v = half[k * mine + tid];
      acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
    }
    const uint32_t j = (from + tid) / d4;
    store(j, (from + tid - j * d4) * 4, acc, inv[j]);
  }
}

}  // namespace shared_attn
}  // namespace nfai

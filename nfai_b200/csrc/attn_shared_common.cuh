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
constexpr uint32_t kPreRows = 128;        // (sequence, head of the group) of a CTA that walks the shared rows
constexpr uint32_t kPreTile = 128;        // ... and its keys per tile

__device__ __forceinline__ float s_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bounded waits as in umma.cuh; the limit is counted in cycles, whose counter is read in a few of them (the nanosecond timer takes
// longer than some of these waits).
constexpr long long kWaitCycles = 2000000000ll;
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity) {
  if (umma::bar_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (!umma::bar_try(bar, parity))
    if (clock64() - t0 > kWaitCycles) return false;
  return true;
}
__device__ __forceinline__ bool all_wait_for(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, wait_for(bar, parity)); }

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

// Everything a CTA does behind its walk: rows[j][d] (stride ld), m[j], l[j] of its query heads h0 .. h0 + nh - 1 are in shared memory,
// all of it written and synchronised. The only part of a sequence is its result, others go to scratch for the join.
template <typename T, int THREADS>
__device__ __forceinline__ void leave_rows(const SharedAttn& p, uint32_t b, uint32_t h0, uint32_t nh, const Walk& w, uint32_t split,
                                           const float* rows, uint32_t ld, const float* m, const float* l) {
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
  for (uint32_t i = tid; i < nh * d4; i += THREADS) {
    const uint32_t j = i / d4, e = (i - j * d4) * 4;
    const float f = w.n ? 1.0f / l[j] : 0.f;  // (no keys at all: zeros; none with a weight: 0 * infinity)
    const float4 v = *reinterpret_cast<const float4*>(rows + j * ld + e);
    store_as(out + j * d + e, v.x * f);
    store_as(out + j * d + e + 1, v.y * f);
    store_as(out + j * d + e + 2, v.z * f);
    store_as(out + j * d + e + 3, v.w * f);
  }
}

}  // namespace shared_attn
}  // namespace nfai

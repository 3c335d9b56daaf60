// What the kernels of attn_shared.cu share: which rows a sequence attends over, and how partial results become a row of the output.
//
// A partial result of one query head is (o[d], m, l): m the largest score (base 2) among its keys, l = sum 2^(s - m), o = sum 2^(s - m) v.
// No keys, or keys whose scores are all -infinity: m = -infinity, l = 0. Several are joined as
//   M = max m_i,  out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i
// in the order of their index, whichever CTA does it: the result does not depend on who came last.
#pragma once
#include "answers.h"
#include "common.cuh"
#include "kernels.h"

namespace nfai {
namespace shared_attn {

constexpr uint32_t kMaxOwnSplits = 148;   // parts a sequence's keys are cut into
constexpr uint32_t kMaxPreSplits = 148;   // parts of the shared rows
constexpr uint32_t kPreRows = 128;        // (sequence, head of the group) of a CTA that walks the shared rows
constexpr uint32_t kPreTile = 128;        // ... and its keys per tile
constexpr uint32_t kSources = kMaxOwnSplits + kMaxPreSplits;
constexpr uint32_t kMaxRows = 16;         // query heads per CTA

__device__ __forceinline__ float s_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

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
  const uint32_t chunk = max(64u, ((w.n + p.own_splits - 1) / p.own_splits + 63) / 64 * 64);
  w.parts = max(1u, (w.n + chunk - 1) / chunk);
  w.t0 = min(w.n, split * chunk);
  w.t1 = min(w.n, w.t0 + chunk);
  return w;
}
// A CTA's way out before it has seen the shared rows' parts: the next kernel in the stream counts on this grid to end behind theirs.
__device__ __forceinline__ void leave(const SharedAttn& p) {
  if (p.pre_splits) pdl_wait();
}
// Offset of key t of sequence b: in the shared rows, or in the sequence's own (`own` set).
__device__ __forceinline__ uint64_t key_row(const SharedAttn& p, uint32_t b, uint32_t t, bool& own) {
  const uint32_t shared = p.pre_splits ? 0u : p.prefix;
  own = t >= shared;
  return own ? (uint64_t)b * p.capacity + (t - shared) : (uint64_t)t;
}

// Everything a CTA does behind its walk: rows[j][d] (stride ld), m[j], l[j] of its query heads h0 .. h0 + nh - 1 are in shared memory,
// all of it written and synchronised.
template <typename T, int THREADS>
__device__ __forceinline__ void finish_rows(const SharedAttn& p, uint32_t b, uint32_t g, uint32_t h0, uint32_t nh, const Walk& w,
                                            uint32_t split, uint32_t ticket, const float* rows, uint32_t ld, const float* m,
                                            const float* l) {
  __shared__ float weight[kMaxRows][kSources];
  __shared__ float inverse[kMaxRows];
  __shared__ uint32_t last;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, d = p.d, G = p.qH / p.kvH, BQ = p.B * p.qH;
  const uint32_t row0 = b * p.qH + h0;
  if (w.parts > 1) {
    for (uint32_t i = tid; i < nh * d; i += THREADS) {
      const uint32_t j = i / d, e = i - j * d;
      p.own_o[((uint64_t)split * BQ + row0 + j) * d + e] = rows[j * ld + e];
    }
    if (tid < nh) *reinterpret_cast<float2*>(p.own_ml + ((uint64_t)split * BQ + row0 + tid) * 2) = make_float2(m[tid], l[tid]);
    __threadfence();
    __syncthreads();
    if (tid == 0) last = atomicAdd(p.tickets + ticket, 1u) == w.parts - 1 ? 1u : 0u;
    __syncthreads();
    if (!last) return leave(p);
    __threadfence();
  }
  if (p.pre_splits) pdl_wait();  // the parts of the shared rows are there
  const uint32_t own = w.parts, n = own + p.pre_splits;
  auto pre_row = [&](uint32_t i, uint32_t j) { return ((uint64_t)i * p.kvH + g) * ((uint64_t)p.B * G) + (uint64_t)b * G + (h0 - g * G) + j; };
  for (uint32_t j = warp; j < nh; j += THREADS / 32) {
    auto ml = [&](uint32_t i) {
      if (i >= own) return __ldcg(reinterpret_cast<const float2*>(p.pre_ml + pre_row(i - own, j) * 2));
      if (own > 1) return __ldcg(reinterpret_cast<const float2*>(p.own_ml + ((uint64_t)i * BQ + row0 + j) * 2));
      return make_float2(m[j], l[j]);
    };
    float M = -INFINITY;
    for (uint32_t i = lane; i < n; i += 32) {
      const float2 a = ml(i);
      weight[j][i] = a.x;
      M = fmaxf(M, a.x);
    }
    M = warp_max(M);
    float L = 0.f;
    for (uint32_t i = lane; i < n; i += 32) {
      const float f = weight[j][i] == -INFINITY ? 0.f : exp2f(weight[j][i] - M);
      weight[j][i] = f;
      const float li = ml(i).y;
      if (f != 0.f || li != li) L = fmaf(f, li, L);
    }
    L = warp_sum(L);
    if (lane == 0) inverse[j] = 1.0f / L;
  }
  __syncthreads();
  const bool nothing = p.prefix == 0 && w.n == 0;
  T* const out = reinterpret_cast<T*>(p.out) + (uint64_t)row0 * d;
  for (uint32_t i = tid; i < nh * d; i += THREADS) {
    const uint32_t j = i / d, e = i - j * d;
    float acc = 0.f;
    if (own > 1) {
#pragma unroll 4
      for (uint32_t k = 0; k < own; ++k) {
        const float f = weight[j][k], v = __ldcg(p.own_o + ((uint64_t)k * BQ + row0 + j) * d + e);
        acc = f != 0.f ? fmaf(f, v, acc) : acc;
      }
    } else if (weight[j][0] != 0.f) {
      acc = weight[j][0] * rows[j * ld + e];
    }
#pragma unroll 4
    for (uint32_t k = 0; k < p.pre_splits; ++k) {
      const float f = weight[j][own + k], v = __ldcg(p.pre_o + pre_row(k, j) * d + e);
      acc = f != 0.f ? fmaf(f, v, acc) : acc;
    }
    store_as(out + i, nothing ? 0.f : acc * inverse[j]);
  }
}

}  // namespace shared_attn
}  // namespace nfai

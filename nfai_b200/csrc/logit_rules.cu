// What a host wants of the next token, applied to the logits of every row before it is drawn:
//
//   c = how often the token stands in the row's history
//   c > 0:  y = x > 0 ? x / repetition : x * repetition, else y = x
//   y -= frequency * c + presence * [c > 0]
//   y += the row's bias for the token (the last listing of it)
//   y = -infinity where the row's grammar does not allow the token
//
// Bound by HBM: logits in, logits out, a bit a token for the mask. A CTA owns a slice of one row's vocabulary: its threads ask for
// their logits, then the CTA goes through the row's history and counts what falls into its slice in shared memory (whole numbers:
// the order of the additions makes no difference) while they are on their way.
//
// In front of SamplingUtils.TopP (NFAI.Models.Llama3/SamplingUtils.cs:5-33); the reference has no such rules.
#include "answers.h"
#include "common.cuh"
#include "kernels.h"

namespace nfai {

namespace {

constexpr int kLT = 256;  // threads

// VEC: rows can be taken in quads (both bases 16-byte aligned). QUADS: quads per thread.
template <int QUADS, bool VEC>
__global__ void __launch_bounds__(kLT) logit_rules_kernel(const LogitRules p, const uint32_t slices) {
  constexpr uint32_t S = kLT * QUADS * 4;
  constexpr uint32_t kTable = S + 4;  // the slice, and up to three tokens in front of the first quad of the row
  extern __shared__ __align__(16) uint32_t smem[];
  uint32_t* const count = smem;            // [kTable]
  uint32_t* const listing = smem + kTable; // [kTable] 1 + the last listing of a bias; only where there are biases
  const uint32_t row = blockIdx.x / slices, slice = blockIdx.x % slices, tid = threadIdx.x;
  const uint64_t base = (uint64_t)row * p.V;
  const uint32_t peel = VEC ? min((uint32_t)(-(int64_t)base & 3), p.V) : 0;  // rows of odd lengths start anywhere
  const uint32_t t0 = peel + slice * S;            // the slice's first token
  const uint32_t t1 = min(p.V, t0 + S);
  const float* const x = p.logits + base;
  float* const y = p.out + base;

  // What decides what else is read comes first, the logits right behind it: nothing of the row is waited for twice.
  int32_t hist_len = p.history && p.history_len ? __ldg(p.history_len + row) : 0x7fffffff;
  int32_t bias_lo = p.n_bias ? __ldg(p.bias_start + row) : 0, bias_hi = p.n_bias ? __ldg(p.bias_start + row + 1) : 0;
  const int64_t mrow = p.n_masks ? (p.mask_rows ? (int64_t)__ldg(p.mask_rows + row) : (int64_t)row) : -1;
  const float rep = p.repetition ? __ldg(p.repetition + row) : 1.f, freq = p.frequency ? __ldg(p.frequency + row) : 0.f,
              pres = p.presence ? __ldg(p.presence + row) : 0.f;
  float v[QUADS][4];
#pragma unroll
  for (int k = 0; k < QUADS; ++k) {
    const uint32_t t = t0 + (k * kLT + tid) * 4;
    if (VEC && t + 4 <= t1) {
      const uint4 w = ld_stream16(x + t);
      v[k][0] = __uint_as_float(w.x); v[k][1] = __uint_as_float(w.y); v[k][2] = __uint_as_float(w.z); v[k][3] = __uint_as_float(w.w);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[k][i] = t + i < t1 ? x[t + i] : 0.f;
    }
  }
  float early = 0.f;  // tokens in front of the first quad: the first slice's
  const bool has_early = slice == 0 && tid < peel;
  if (has_early) early = x[tid];
  const bool masked = mrow >= 0 && mrow < (int64_t)p.n_masks;
  uint32_t allowed[QUADS], allowed_early = 0xffffffffu;
  if (masked) {
    const uint32_t* const mask = p.masks + (uint64_t)mrow * ((p.V + 31) / 32);
#pragma unroll
    for (int k = 0; k < QUADS; ++k) {
      const uint32_t t = t0 + (k * kLT + tid) * 4;
      allowed[k] = t < t1 ? __funnelshift_r(__ldg(mask + (t >> 5)), __ldg(mask + (min(t + 3, p.V - 1) >> 5)), t & 31) : 0u;
    }
    if (has_early) allowed_early = __ldg(mask) >> tid;
  } else {
#pragma unroll
    for (int k = 0; k < QUADS; ++k) allowed[k] = 0xffffffffu;
  }
  const uint32_t n_hist = p.history ? (uint32_t)min((int64_t)max(hist_len, 0), (int64_t)p.history_stride) : 0u;
  const uint32_t b0 = min((uint32_t)max(bias_lo, 0), p.n_bias), b1 = min((uint32_t)max(bias_hi, 0), p.n_bias);
  const bool counted = n_hist > 0, biased = b1 > b0;
  // a token's place in the tables; anything else (another slice's, no token at all): kTable
  auto cell = [&](uint32_t t) { return t >= t0 ? (t < t1 ? t - t0 : kTable) : (slice == 0 && t < peel ? S + t : kTable); };
  if (counted || biased) {
    for (uint32_t i = tid; i < kTable / 4; i += kLT) {
      if (counted) reinterpret_cast<uint4*>(count)[i] = make_uint4(0, 0, 0, 0);
      if (biased) reinterpret_cast<uint4*>(listing)[i] = make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
    const uint32_t* const h = p.history + (uint64_t)row * p.history_stride;
    for (uint32_t i = tid; i < n_hist; i += kLT * 8) {  // eight at a time on their way
      uint32_t t[8];
#pragma unroll
      for (uint32_t k = 0; k < 8; ++k) t[k] = i + k * kLT < n_hist ? __ldg(h + i + k * kLT) : 0xffffffffu;
#pragma unroll
      for (uint32_t k = 0; k < 8; ++k) {
        const uint32_t c = cell(t[k]);
        if (c != kTable) atomicAdd(count + c, 1u);
      }
    }
    for (uint32_t i = b0 + tid; i < b1; i += kLT) {
      const uint32_t c = cell(__ldg(p.bias_ids + i));
      if (c != kTable) atomicMax(listing + c, i + 1);
    }
    __syncthreads();
  }
  auto ruled = [&](float a, uint32_t c, uint32_t listed) {
    if (c) {
      a = a > 0.f ? __fdiv_rn(a, rep) : a * rep;
      a = __fsub_rn(__fsub_rn(a, __fmul_rn(freq, (float)c)), pres);
    }
    return listed ? __fadd_rn(a, __ldg(p.bias + listed - 1)) : a;
  };
#pragma unroll
  for (int k = 0; k < QUADS; ++k) {
    const uint32_t at = (k * kLT + tid) * 4, t = t0 + at;
    if (t >= t1) continue;
    uint4 c = make_uint4(0, 0, 0, 0), l = c;
    if (counted) c = *reinterpret_cast<const uint4*>(count + at);
    if (biased) l = *reinterpret_cast<const uint4*>(listing + at);
    if (c.x | c.y | c.z | c.w | l.x | l.y | l.z | l.w) {
      v[k][0] = ruled(v[k][0], c.x, l.x);
      v[k][1] = ruled(v[k][1], c.y, l.y);
      v[k][2] = ruled(v[k][2], c.z, l.z);
      v[k][3] = ruled(v[k][3], c.w, l.w);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (!(allowed[k] >> i & 1)) v[k][i] = -INFINITY;
    if (VEC && t + 4 <= t1) {
      *reinterpret_cast<float4*>(y + t) = make_float4(v[k][0], v[k][1], v[k][2], v[k][3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t + i < t1) y[t + i] = v[k][i];
    }
  }
  if (has_early) {
    early = ruled(early, counted ? count[S + tid] : 0u, biased ? listing[S + tid] : 0u);
    if (!(allowed_early & 1)) early = -INFINITY;
    y[tid] = early;
  }
}

template <int QUADS>
cudaError_t launch_quads(cudaStream_t s, const LogitRules& p) {
  constexpr uint32_t S = kLT * QUADS * 4;
  const bool vec = (((uintptr_t)p.logits | (uintptr_t)p.out) & 15) == 0;
  const uint32_t slices = (p.V + S - 1) / S;  // (the tokens in front of a row's first quad do not add one: fewer are left)
  const uint64_t grid = (uint64_t)p.rows * slices;
  if (grid > 0x7fffffffu) return cudaErrorInvalidValue;
  const size_t smem = (size_t)(p.n_bias ? 2 : 1) * (S + 4) * 4;
  if (vec) logit_rules_kernel<QUADS, true><<<(unsigned)grid, kLT, smem, s>>>(p, slices);
  else logit_rules_kernel<QUADS, false><<<(unsigned)grid, kLT, smem, s>>>(p, slices);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_logit_rules(cudaStream_t s, const LogitRules& p) {
  // few rows: slices small enough to occupy every SM
  return (uint64_t)p.rows * p.V >= 148ull * 4 * 4096 ? launch_quads<4>(s, p) : launch_quads<1>(s, p);
}

}  // namespace nfai

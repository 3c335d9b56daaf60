// What a host wants of the next token, applied to the logits of every row before it is drawn:
//
//   c = how often the token stands in the row's history
//   c > 0:  y = x > 0 ? x / repetition : x * repetition, else y = x
//   y -= frequency * c + presence * [c > 0]
//   y += the row's bias for the token (the last listing of it)
//   y = -infinity where the row's grammar does not allow the token
//
// Bound by HBM: logits in, logits out, a bit a token for the mask. A CTA owns a slice of one row's vocabulary. One thread has the slice
// copied into shared memory and, at the end, out of it; meanwhile all count what of the row's history falls into the slice (whole
// numbers: the order of the additions makes no difference). A thread remembers which of its tokens were the first in their place: for
// those it applies the penalties. The last listing of a bias is found among the lanes of a warp, or in the table, which is empty again.
// The mask comes last: a lane has the bits of 32 tokens, which the warp then takes one lane's after the other, so that neighbouring lanes
// write neighbouring tokens.
// 48 rows of 128256: 9.5 us with nothing asked for (5.2 TB/s), 14.5 with 4000 tokens of history, 12.4 with a mask for every row (17.0 where a
// thread had four neighbouring tokens: stores to the same banks), 17.0 with history, biases, and masks for half of the rows. Bound by waiting:
// a CTA walks a chain of steps (lengths, history, counts, penalties, biases, mask, store) while its copy has long arrived and its store has
// not begun; issue slots are used in 48 % of the cycles, DRAM to less than half of its rate. Tried: 16 tokens of the history asked for at
// once (17.5 for 17.1), penalties where the logits are stored (22.3: nearly every warp has a touched token and takes the path for all), one
// wave of slices twice as long with the logits in registers (18.5), clusters of eight slices that share the history and add to one
// another's counts (21.7: 14.2 with nothing asked for), a look at every token's count a second time (19.1), a plain copy and behind it a
// CTA a row that has the touched tokens in a hash table (26.2).
//
// In front of SamplingUtils.TopP (NFAI.Models.Llama3/SamplingUtils.cs:5-33); the reference has no such rules.
#include "answers.h"
#include "attn_shared_common.cuh"
#include "common.cuh"
#include "kernels.h"

namespace nfai {

namespace {

constexpr int kLT = 256;
constexpr uint32_t kLongest = 6144;  // tokens of a slice: 8 bytes of shared memory each, four CTAs to an SM
constexpr uint32_t kShortest = 1024;
constexpr uint32_t kSeen = 8;   // tokens of the history that a thread asks for at once
constexpr uint32_t kKept = 32;  // ... and for which it remembers whether they were the first in their place

// VEC: rows can be taken 16 bytes at a time (both bases aligned to them). S: tokens of a slice, a multiple of 4.
template <bool VEC>
__global__ void __launch_bounds__(kLT) logit_rules_kernel(const LogitRules p, const uint32_t slices, const uint32_t S) {
  extern __shared__ __align__(16) unsigned char rules_smem[];
  // the slice, and behind it up to three tokens in front of the first 16 bytes of the row
  float* const value = reinterpret_cast<float*>(rules_smem);               // [S + 4]
  uint32_t* const count = reinterpret_cast<uint32_t*>(value + S + 4);      // [S + 4]
  __shared__ __align__(8) uint64_t landed;
  const uint32_t row = blockIdx.x / slices, slice = blockIdx.x - row * slices, tid = threadIdx.x;
  const uint64_t base = (uint64_t)row * p.V;
  const uint32_t peel = VEC ? min((uint32_t)(-(int64_t)base & 3), p.V) : 0;  // rows of odd lengths start anywhere
  const uint32_t t0 = peel + slice * S;              // the slice's first token
  const uint32_t t1 = max(t0, min(p.V, t0 + S));
  const bool front = VEC && slice == 0;              // ... and it has the tokens in front
  const uint32_t whole = VEC ? (t1 - t0) & ~3u : 0;  // what goes 16 bytes at a time
  const float* const x = p.logits + base;
  float* const y = p.out + base;
  const uint32_t bar = umma::s_u32(&landed);
  if (tid == 0) {
    umma::bar_init(bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (whole) {
      umma::bar_expect_tx(bar, whole * 4);
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(umma::s_u32(value)), "l"(x + t0),
                   "r"(whole * 4), "r"(bar)
                   : "memory");
    }
  }
  // What decides what else is read comes first. A row's history has history_stride places whatever its length, behind which the next row's
  // begin: the first are asked for too. Behind the last row's tokens there need be no memory.
  const uint32_t* const h = p.history + (uint64_t)row * p.history_stride;
  const int32_t hist_len = p.history && p.history_len ? __ldg(p.history_len + row) : 0x7fffffff;
  const int32_t bias_lo = p.n_bias ? __ldg(p.bias_start + row) : 0, bias_hi = p.n_bias ? __ldg(p.bias_start + row + 1) : 0;
  const int64_t mrow = p.n_masks ? (p.mask_rows ? (int64_t)__ldg(p.mask_rows + row) : (int64_t)row) : -1;
  uint32_t seen[kSeen];
  auto ask = [&](uint32_t places) {
#pragma unroll
    for (uint32_t k = 0; k < kSeen; ++k) seen[k] = tid + k * kLT < places ? __ldg(h + tid + k * kLT) : 0xffffffffu;
  };
  if (!p.history || row + 1 < p.rows) ask(p.history ? p.history_stride : 0u);
  else ask((uint32_t)min((int64_t)max(hist_len, 0), (int64_t)p.history_stride));
  const float rep = p.repetition ? __ldg(p.repetition + row) : 1.f, freq = p.frequency ? __ldg(p.frequency + row) : 0.f,
              pres = p.presence ? __ldg(p.presence + row) : 0.f;
  // what does not go 16 bytes at a time: the end of the slice, and tokens in front
  for (uint32_t i = whole + tid; i < t1 - t0; i += kLT) value[i] = x[t0 + i];
  if (front && tid < peel) value[S + tid] = x[tid];
  for (uint32_t i = tid; i < S / 4 + 1; i += kLT) reinterpret_cast<uint4*>(count)[i] = make_uint4(0, 0, 0, 0);
  const bool masked = mrow >= 0 && mrow < (int64_t)p.n_masks;
  const uint32_t* const mask = p.masks + (masked ? (uint64_t)mrow * ((p.V + 31) / 32) : 0);
  auto open = [&](uint32_t t) { return !masked || (__ldg(mask + (t >> 5)) >> (t & 31) & 1); };
  const uint32_t n_hist = p.history ? (uint32_t)min((int64_t)max(hist_len, 0), (int64_t)p.history_stride) : 0u;
  const uint32_t b0 = min((uint32_t)max(bias_lo, 0), p.n_bias), b1 = min((uint32_t)max(bias_hi, 0), p.n_bias), lane = tid & 31;
  const bool few = b1 <= b0 + 32;  // biases of a row that one warp has at once
  uint32_t listed = 0xffffffffu;
  float bias = 0.f;
  if (few && tid < 32 && b0 + lane < b1) {
    listed = __ldg(p.bias_ids + b0 + lane);
    bias = __ldg(p.bias + b0 + lane);
  }
  __syncthreads();  // the table is empty
  // A warp masks a stretch of the slice, a lane has the bits of 32 tokens of it (one: allowed, or not in the slice).
  const uint32_t len = t1 - t0, chunks = (S + kLT - 1) / kLT, warp = tid >> 5;
  static_assert(kLongest / kLT <= 32, "chunks of a warp");
  uint32_t word = ~0u;
  if (masked && lane < chunks && (warp * chunks + lane) * 32 < len) {
    const uint32_t c = (warp * chunks + lane) * 32, t = t0 + c, w = t >> 5;
    word = __ldg(mask + w);
    if (t & 31) word = __funnelshift_r(word, __ldg(mask + min(w + 1, (p.V - 1) >> 5)), t & 31);
    if (len - c < 32) word |= ~0u << (len - c);
  }

  // a token's place in the tables; another slice's, or no token at all: `len` or more. (Tokens in front have theirs behind the slice; they
  // are looked for apart, where there are any: the history is what costs instructions, twice for every slice.)
  auto in_front = [&](auto&& each) {
    for (uint32_t i = tid; i < n_hist; i += kLT) {
      const uint32_t t = __ldg(h + i);
      if (t < peel) each(S + t, t);
    }
  };
  uint32_t first = 0;  // bit k: token k of this thread was the first to be counted in its place, and is the one that the penalties are applied for
  auto add = [&](const uint32_t (&t)[8], uint32_t k0) {
    uint32_t before[8];
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) before[k] = t[k] < len ? atomicAdd(count + t[k], 1u) : 1u;
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) first |= (before[k] == 0 ? 1u : 0u) << (k0 + k);
  };
#pragma unroll
  for (uint32_t k = 0; k < 8; ++k) seen[k] = tid + k * kLT < n_hist ? seen[k] - t0 : 0xffffffffu;
  add(seen, 0);
  for (uint32_t k0 = 8; k0 < kKept && k0 * kLT < n_hist; k0 += 8) {
    uint32_t t[8];
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) t[k] = tid + (k0 + k) * kLT < n_hist ? __ldg(h + tid + (k0 + k) * kLT) - t0 : 0xffffffffu;
    add(t, k0);
  }
  for (uint32_t i = tid + kKept * kLT; i < n_hist; i += kLT) {
    const uint32_t t = __ldg(h + i) - t0;
    if (t < len) atomicAdd(count + t, 1u);
  }
  if (front && peel) in_front([&](uint32_t c, uint32_t) { atomicAdd(count + c, 1u); });
  const bool ok = __syncthreads_and(!whole || shared_attn::wait_for(bar, 0, p.wait_cycles));  // the slice is there, and everything is counted
  if (n_hist) {
    auto rule = [&](uint32_t c, uint32_t t) {  // whoever finds a count takes it and leaves none
      const uint32_t n = atomicExch(count + c, 0u);
      if (!n) return;
      float a = value[c];
      a = a > 0.f ? __fdiv_rn(a, rep) : a * rep;
      value[c] = __fsub_rn(__fsub_rn(a, __fmul_rn(freq, (float)n)), pres);
    };
    for (; first; first &= first - 1) {
      const uint32_t t = __ldg(h + tid + (__ffs(first) - 1) * kLT);
      rule(t - t0, t);
    }
    for (uint32_t i = tid + kKept * kLT; i < n_hist; i += kLT) {  // (places that only these have; the others' counts are gone, or come to the same)
      const uint32_t t = __ldg(h + i);
      if (t - t0 < len && *reinterpret_cast<volatile uint32_t*>(count + (t - t0))) rule(t - t0, t);
    }
    if (front && peel) in_front(rule);
  }
  const uint32_t none = S + 4;
  auto cell = [&](uint32_t t) { return t - t0 < len ? t - t0 : (front && t < peel ? S + t : none); };
  if (b1 > b0) {
    __syncthreads();  // penalties come first, and the table is empty again
    if (few) {
      if (tid < 32) {
        const uint32_t same = __match_any_sync(0xffffffffu, listed), c = cell(listed);
        if (lane == 31 - __clz(same) && c != none) value[c] = __fadd_rn(value[c], bias);
      }
    } else {
      for (uint32_t i = b0 + tid; i < b1; i += kLT) {
        const uint32_t c = cell(__ldg(p.bias_ids + i));
        if (c != none) atomicMax(count + c, i + 1);
      }
      __syncthreads();
      for (uint32_t i = b0 + tid; i < b1; i += kLT) {
        const uint32_t t = __ldg(p.bias_ids + i), c = cell(t);
        if (c != none && count[c] == i + 1) value[c] = __fadd_rn(value[c], __ldg(p.bias + i));
      }
    }
  }
  if (masked) __syncthreads();  // the mask comes last
  if (masked) {
#pragma unroll 4
    for (uint32_t i = 0; i < chunks; ++i) {
      const uint32_t gone = ~__shfl_sync(0xffffffffu, word, i);
      if (gone >> lane & 1) value[(warp * chunks + i) * 32 + lane] = -INFINITY;
    }
  }
  if (front && tid < peel && !open(tid)) value[S + tid] = -INFINITY;
  if (!ok) {
    if (p.err && tid == 0) atomicOr(p.err, 4u);
    shared_attn::let_land();
    __syncthreads();
    for (uint32_t i = tid; i < whole; i += kLT) value[i] = __int_as_float(0x7fffffff);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
  if (tid == 0 && whole) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(y + t0), "r"(umma::s_u32(value)), "r"(whole * 4) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
  for (uint32_t i = whole + tid; i < t1 - t0; i += kLT) y[t0 + i] = value[i];
  if (front && tid < peel) y[tid] = value[S + tid];
  if (tid == 0 && whole) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}

}  // namespace

cudaError_t launch_logit_rules(cudaStream_t s, const LogitRules& p) {
  const bool vec = (((uintptr_t)p.logits | (uintptr_t)p.out) & 15) == 0;
  // Slices of one length, as many as the CTAs that run at once have room for (a few rounds of them where a row needs more), none so short
  // that starting it takes longer.
  const uint64_t room = 148 * 4, fewest = (p.V + kLongest - 1) / kLongest, rounds = (fewest * p.rows + room - 1) / room;
  uint64_t slices = room * rounds / p.rows, most = (p.V + kShortest - 1) / kShortest;
  slices = slices < fewest ? fewest : slices > most ? most : slices;
  const uint32_t S = (uint32_t)(((p.V + slices - 1) / slices + 3) / 4 * 4);
  slices = (p.V + S - 1) / S;  // (the tokens in front of a row's first quad do not add one: as many fewer are left)
  if (slices * p.rows > 0x7fffffffu) return cudaErrorInvalidValue;
  const size_t smem = (size_t)(S + 4) * 8;
  auto kernel = vec ? logit_rules_kernel<true> : logit_rules_kernel<false>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kLongest + 4) * 8);
  if (e != cudaSuccess) return e;
  kernel<<<(unsigned)(slices * p.rows), kLT, smem, s>>>(p, (uint32_t)slices, S);
  return cudaGetLastError();
}

}  // namespace nfai

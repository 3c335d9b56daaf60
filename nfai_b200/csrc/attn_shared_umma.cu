// The shared rows, once for every sequence: 16-bit types, heads up to 128, on the 5th-generation tensor cores. Heads that are not 64 or 128
// are filled up with zeros to the next of them by the copies.
//
// The query heads of a KV head and the sequences are one list of rows (row = sequence * G + head of the group). A CTA has two streams of
// 128 rows each, one accumulator lane a row, and walks a part of the keys in tiles of 128. With more than 128 rows the streams are
// neighbouring row tiles on the same keys, which are then fetched once for 256 rows; with fewer they are the same rows on every second
// tile of keys. While one stream forms its weights the tensor pipe works for the other:
//   warp 16  K and V tiles by TMA into a ring of 128-byte swizzled slots, in the order in which they are multiplied
//   warp 17  one lane issues S(0), S(1), then for every unit (stream, tile) u: O += P(u) V, S(u + 2) = Q K^T, with P in tensor memory where
//            S(u) was (for heads up to 64 there is room for a third unit: S(u + 3)) and V as it lies (its rows run along N). (A warp for
//            each stream was no faster, 76 us for 72 with 64 sequences behind 32768 rows: the streams fell into step and wanted the same
//            units at the same time.)
//   warp 18  sees the ring's slots fill, in order, and arrives with the softmax warps on the barrier that warp 17 waits for: waiting for the
//            tiles itself cost that warp 600 of 3700 cycles in which nothing was multiplied
//   warps 0-7 and 8-15  softmax of a stream, two threads to a row (64 keys each): weights back into tensor memory as the 16-bit
//            operand of the second product, their float32 sums kept
// Up to 64 (32) rows are in the lanes twice (four times), each copy with the weights of its own half (quarter) of a tile's keys and zeros
// for the others: a row's exponentials are then spread over the schedulers, whose warps each see 32 lanes only.
// At the end sums of weighted values, maxima and sums of weights go to scratch line by line, by way of shared memory, where streams and
// copies of the same rows are joined; attn_shared_join_kernel joins the parts with those of the own rows.
// Bound by what a stream's tile takes one after the other: a tile of 128 keys takes the softmax warps 1850 cycles (scores from tensor memory,
// maximum and first half of the weights 900, second half 790, the way back 150; the unit for exponentials works 768 of them, 1024 without the
// fourth of the weights that is computed as a polynomial), the two products 1290 more, of which the other stream's softmax covers a part; no
// unit is busy for more than half of the time. 128 sequences of 32 heads of 64 behind 20000 rows: 48.4 us, with a third unit 45.6, with the
// polynomial 43.5 (for an eighth of the weights 43.7, a third 44.3), 44.5 since scores and values of any size are looked after. 64 of 32 of 128
// behind 32768: 67.6, and 69.0; the kernel itself takes 40 us, 0.85 PFLOP/s, where 1.68 have been measured; 4 us at its end are the
// sums' way to memory. With few rows it is bound by memory: 5 sequences of 32 heads of 64 behind 100003 rows 40 us, 5.2 TB/s.
// Weights are rounded to the caches' type, as the product takes both operands of one type and a second term would double its time: a result is
// 1.05 to 1.4 times as far from the one in 64 bits as with weights of 32, where the rounding of the result is nearly all.
// Scores are products of the 16-bit queries as they are; the scale goes into the exponent's multiply-add. A row's sums are rescaled only
// when its maximum has grown by more than 2^8 since the last time.
#include <float.h>

#include <type_traits>

#include "attn_shared_common.cuh"

namespace nfai {

namespace {

using namespace umma;
using shared_attn::all_wait_for;
using shared_attn::kPreRows;
using shared_attn::kPreTile;
using shared_attn::s_ex2;
using shared_attn::wait_for;

constexpr int kSoftmax = 512, kThreads = kSoftmax + 96;
constexpr float kGrowth = 8.0f;
constexpr float kFar = 1048576.0f;  // 2^20: from here on a ref is off by 2^-3 and more
// Weights are multiplied by 2^kLift before they are rounded (the weights' sum has the factor too, and the maximum that goes to scratch is
// lower by it). float16 ends at 2^-25: without the factor a key that is 2^-25 lighter than its row's heaviest counts for nothing, and 100 000 of
// them behind a heavy one are 0.003 of the row. 2^(kGrowth + kLift) is within float16, whose largest number is 2^16. (2^4 and 2^11 rescale more
// often: 64 sequences of 32 heads of 128 behind 32768 rows 71.2 us for 67.3.) bfloat16 has float32's range.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.0f : 0.0f;

template <int D>
struct PreSmem {
  static constexpr uint32_t kTile = kPreTile * D * 2;
  static constexpr uint32_t kSlots = D == 64 ? 12 : 5;
  static constexpr uint32_t kQ = kPreRows * D * 2;  // of one stream
  static constexpr uint32_t kPlaces = D == 64 ? 3 : 2;  // units that have their scores or weights in tensor memory
  static constexpr uint32_t kRing = 2 * kQ;
  static constexpr uint32_t kBarOff = kRing + kSlots * kTile;
  static constexpr uint32_t kSwapOff = kBarOff + 512;  // [stream][half][row]: maxima of the halves of a row, later their sums, maxima and sums
  static constexpr uint32_t kTotal = kSwapOff + 4 * kPreRows * 4;
};
static_assert(PreSmem<64>::kTotal <= 232448 && PreSmem<128>::kTotal <= 232448, "shared memory of a CTA");
static_assert(2 * kPreRows * 64 * 4 <= PreSmem<64>::kBarOff && 2 * kPreRows * 128 * 4 <= PreSmem<128>::kBarOff, "both streams' sums go where Q and the ring were");

// 2^x of two numbers (x up to 127, NaN stays NaN, below -126.5 gives 0) without the unit for it: x = n + f with a whole n and f in
// [-1/2, 1/2], 2^f as a polynomial of degree 5 (fitted to the least relative error by weighted least squares on Chebyshev points; in
// float32 off by 2.2e-7 at most), and 2^n put together from its exponent.
__device__ __forceinline__ void poly_ex2(float& a, float& b) {
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(a));  // -127
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(b));
  auto both = [](float v) { return pair(v, v); };
  constexpr float kWhole = 12583039.f;  // 1.5 * 2^23 + 127: adding it leaves n + 127 in the last bits
  const uint64_t x = pair(a, b), t = add2(x, both(kWhole)), f = fma2(add2(t, both(-kWhole)), both(-1.f), x);
  uint64_t y = fma2(f, both(0.0013276472454890609f), both(0.009675540961325169f));
  y = fma2(y, f, both(0.05550713092088699f));
  y = fma2(y, f, both(0.24022120237350464f));
  y = fma2(y, f, both(0.6931469440460205f));
  y = fma2(y, f, both(1.0000001192092896f));
  unpair(t, a, b);
  unpair(fma2(y, pair(__uint_as_float(__float_as_uint(a) << 23), __uint_as_float(__float_as_uint(b) << 23)), 0), a, b);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[8]) {
  __syncwarp();
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
               "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
using umma::tmem_st;

// COPIES: how often the rows are in the lanes (2 and 4: one row tile)
template <typename T, int D, int COPIES>
__global__ void __launch_bounds__(kThreads, 1) attn_shared_umma_kernel(const __grid_constant__ CUtensorMap mapQ,
                                                                       const __grid_constant__ CUtensorMap mapK,
                                                                       const __grid_constant__ CUtensorMap mapV, const __grid_constant__ SharedAttn p,
                                                                       const uint32_t row_tiles) {
  using SM = PreSmem<D>;
  // columns of tensor memory: NB places for the scores and weights of a unit, the streams' sums behind them
  constexpr uint32_t NB = SM::kPlaces, kSP = 128, kO = NB * kSP;
  static_assert(kO + 2 * D <= 512, "tensor memory");
  constexpr uint32_t kTypes = (1u << 4) | (std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u);
  constexpr uint32_t kKeys = kPreTile / COPIES, kMine = kKeys / 2, kLanesOf = kPreRows / COPIES;  // of a copy: keys, a thread's keys, lanes
  extern __shared__ __align__(1024) unsigned char pre_raw[];
  unsigned char* const sm = pre_raw;
  uint64_t* const bars = reinterpret_cast<uint64_t*>(sm + SM::kBarOff);
  const uint32_t full0 = s_u32(bars), empty0 = s_u32(bars + SM::kSlots), q_ready = s_u32(bars + 2 * SM::kSlots);
  // A wait knows a phase by its parity only. So whoever waits for one of these sees every phase of it: the softmax warps their stream's
  // units (every second one), warps 17 and 18 all of them.
  constexpr uint32_t NS = NB % 2 ? 2 * NB : NB;
  auto s_ready = [&](uint32_t u) { return q_ready + 8 + 8 * (u % NS); };
  auto s_turn = [&](uint32_t u) { return u / NS & 1; };
  auto p_ready = [&](uint32_t u) { return q_ready + 8 + 8 * NS + 8 * (u % NB); };
  auto p_turn = [&](uint32_t u) { return u / NB & 1; };
  auto pv_last = [&](uint32_t st) { return q_ready + 8 + 8 * (NS + NB) + 8 * st; };  // the stream's last product with values is done
  // Every one of them, for a wait that is seldom needed: who waits for that of the stream's tile `it` knows that the one before is done
  // and that the one after has not been issued.
  auto pv_done = [&](uint32_t st) { return pv_last(2) + 8 * st; };
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * SM::kSlots + NS + NB + 5);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  // CTAs of the same keys are neighbours
  const bool twice = COPIES > 1 || row_tiles == 1;  // one row tile: the streams have it both
  const uint32_t d = p.d, pairs = (row_tiles + 1) / 2, G = p.qH / p.kvH, R = p.B * G, tile = blockIdx.x % pairs * 2, g = blockIdx.x / pairs % p.kvH,
                 split = blockIdx.x / pairs / p.kvH;
  const uint32_t all = (p.prefix + kPreTile - 1) / kPreTile, first = split * p.pre_tiles, n = min(p.pre_tiles, all - first);  // tiles of keys
  // Q comes by TMA where the rows of a copy are whole sequences' heads, by the softmax warps otherwise; one stream's, where both have the
  // same. (By the softmax warps it holds up the first tiles by 1.6 us, or waits behind them for 6.)
  const bool whole_q = kLanesOf % G == 0;
  const uint32_t st = warp >> 3, row0 = (tile + (twice ? 0u : st)) * kPreRows;
  if (tid == 0) {
    for (uint32_t i = 0; i < SM::kSlots; ++i) {
      bar_init(full0 + 8 * i, 1);
      bar_init(empty0 + 8 * i, 1);
    }
    bar_init(q_ready, whole_q ? 2 : 17);
    for (uint32_t i = 0; i < NS; ++i) bar_init(s_ready(i), 1);
    for (uint32_t i = 0; i < NB; ++i) bar_init(p_ready(i), 9);
    for (uint32_t i = 0; i < 2; ++i) {
      bar_init(pv_last(i), 1);
      bar_init(pv_done(i), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 17) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();  // the own rows do not wait for the shared ones, only the join does
  const uint32_t units = twice ? n : 2 * n;  // unit u: stream u % 2, tile of keys u or u / 2
  bool ok = true;
  float odd = 0.f;  // NaN: one is among the sums of this thread's row

  if (warp == 16) {
    if (whole_q && elect_one()) {
      const uint32_t streams = twice ? 1 : 2;
      bar_expect_tx(q_ready, streams * SM::kQ);
      for (uint32_t i = 0; i < streams; ++i)
#pragma unroll
        for (uint32_t k = 0; k < COPIES; ++k)
#pragma unroll
          for (uint32_t b = 0; b < D / 64; ++b)
            tma_load_4d(s_u32(sm) + i * SM::kQ + b * (kPreRows * 128) + k * (kLanesOf * 128), &mapQ, (int)(b * 64), 0, (int)g, (int)((tile + i) * kPreRows / G), q_ready);
    }
    __syncwarp();
    uint32_t j = 0;
    auto load = [&](const CUtensorMap* map, uint32_t it) {
      const uint32_t s = j % SM::kSlots;
      if (j >= SM::kSlots && !all_wait_for(empty0 + 8 * s, (j / SM::kSlots - 1) & 1, p.wait_cycles)) return ok = false;
      if (elect_one()) {
        bar_expect_tx(full0 + 8 * s, SM::kTile);
#pragma unroll
        for (uint32_t b = 0; b < D / 64; ++b)
          tma_load_4d(s_u32(sm) + SM::kRing + s * SM::kTile + b * (kPreTile * 128), map, (int)(b * 64), (int)g, (int)((first + it) * kPreTile), 0, full0 + 8 * s);
      }
      ++j;
      return true;
    };
    if (twice) {  // K0 K1, V0 K2, V1 K3, .. (K0 K1 K2, V0 K3, ..)
      for (uint32_t u = 0; u < NB && u < n && ok; ++u) load(&mapK, u);
      for (uint32_t u = 0; u < n && ok; ++u)
        if (!load(&mapV, u) || (u + NB < n && !load(&mapK, u + NB))) break;
    } else {  // K0 V0, K1 V1, ..
      for (uint32_t it = 0; it < n && ok; ++it)
        if (!load(&mapK, it) || !load(&mapV, it)) break;
    }
    // the last slots' products, as drain_ring does, within the budget
    for (uint32_t i = j > SM::kSlots ? j - SM::kSlots : 0; i < j && ok; ++i) ok = all_wait_for(empty0 + 8 * (i % SM::kSlots), i / SM::kSlots & 1, p.wait_cycles);
  } else if (warp == 17) {
    // 16-bit operands, float32 sums; A along K in both products; B along K (K tile) or along N (V tile)
    constexpr uint32_t idesc_s = kTypes | ((kPreTile >> 3) << 17) | ((kPreRows >> 4) << 24);
    constexpr uint32_t idesc_o = kTypes | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((kPreRows >> 4) << 24);
    const uint32_t base = s_u32(sm);
    // the place in the ring's order of the keys of unit u, and of its values
    auto keys_of = [&](uint32_t u) { return twice ? (u < NB ? u : 2 * u - NB + 1) : (u >> 1) * 2; };
    auto values_of = [&](uint32_t u) { return twice ? min(u + NB, units) + u : (u >> 1) * 2 + 1; };
    auto scores = [&](uint32_t u) {
      const uint32_t st = u & 1, s = keys_of(u) % SM::kSlots;
      if (elect_one()) {
        const uint32_t k_s = base + SM::kRing + s * SM::kTile, q_s = base + (twice ? 0u : st * SM::kQ);
#pragma unroll
        for (uint32_t kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * (kPreRows * 128) + (kk & 3) * 32;
          umma_f16(tmem + u % NB * kSP, smem_desc_sw128(q_s + off), smem_desc_sw128(k_s + off), idesc_s, kk != 0);
        }
        if (twice || st) umma_commit(empty0 + 8 * s);
        umma_commit(s_ready(u));
      }
    };
    ok = all_wait_for(q_ready, 0, p.wait_cycles);  // Q, and the first keys' tiles
    fence_after();
    for (uint32_t u = 0; u < NB && u < units && ok; ++u) scores(u);
    for (uint32_t u = 0; u < units && ok; ++u) {
      const uint32_t st = u & 1, it = u >> 1, j = values_of(u);  // it: the stream's own count
      if (!(ok = all_wait_for(p_ready(u), p_turn(u), p.wait_cycles))) break;  // the weights, the values' tile and the next scores' keys
      fence_after();
      if (elect_one()) {
        const uint32_t s = j % SM::kSlots, v_s = base + SM::kRing + s * SM::kTile;
#pragma unroll
        for (uint32_t kk = 0; kk < kPreTile / 16; ++kk)
          umma_f16_ta(tmem + kO + st * D, tmem + u % NB * kSP + kk * 8, smem_desc_mn_sw128(v_s + kk * 2048, kPreTile * 128), idesc_o, (it | kk) != 0);
        if (twice || st) umma_commit(empty0 + 8 * s);
        if (NB > 2) umma_commit(pv_done(st));
        if (u + 2 >= units) umma_commit(pv_last(st));
      }
      // (the weights lie where the next scores go: products of one thread run in their order)
      if (u + NB < units) scores(u + NB);
    }
  } else if (warp == 18) {
    // All slots, each phase, in the ring's order: a wait knows a phase by its parity only.
    const uint32_t tiles = 2 * n;
    uint32_t seen = 0;
    auto see = [&](uint32_t upto) {  // the first `upto` tiles have arrived
      for (; seen < upto && ok; ++seen) ok = all_wait_for(full0 + 8 * (seen % SM::kSlots), (seen / SM::kSlots) & 1, p.wait_cycles);
    };
    see(min(tiles, twice ? NB : (NB - 1) / 2 * 2 + 1));
    if (ok && lane == 0) bar_arrive(q_ready);
    for (uint32_t u = 0; u < units && ok; ++u) {
      see(min(tiles, twice ? 2 * u + NB + 2 : (u + NB) / 2 * 2 + 1));
      if (u >= NB && ok) ok = all_wait_for(p_ready(u), p_turn(u - NB), p.wait_cycles);  // (the phase before has ended: this arrival is for the next)
      if (ok && lane == 0) bar_arrive(p_ready(u));
    }
  } else {
    if (!whole_q) {  // the rows as they are, each piece of 16 bytes to its place under the swizzle
      constexpr uint32_t kLanes = D / 8, kRows = 32 / kLanes;  // lanes to a row
      const uint32_t qc = (lane % kLanes) * 8;
      if (!twice || st == 0) {
#pragma unroll
        for (uint32_t i = 0; i < 16; i += kRows) {
          const uint32_t r = (warp & 7) * 16 + i + lane / kLanes, row = row0 + r % kLanesOf, b = row / G;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (row < R && qc < d) v = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + ((uint64_t)b * p.qH + g * G + (row - b * G)) * d + qc));
          *reinterpret_cast<uint4*>(sm + st * SM::kQ + (qc >> 6) * (kPreRows * 128) + r * 128 + ((((qc & 63) >> 3) ^ (r & 7)) << 4)) = v;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      __syncwarp();
      if (lane == 0) bar_arrive(q_ready);
    }
    const uint32_t quarter = warp & 3, half = warp >> 2 & 1, place = quarter * 32 + lane, copy = quarter / (4 / COPIES);
    const uint32_t col0 = copy * kKeys + half * kMine, row = row0 + place % kLanesOf;
    const uint32_t lanes = tmem + (quarter * 32u << 16), cO = kO + st * D;
    const uint32_t tiles = twice ? (n + 1 - st) / 2 : n;  // of this stream
    const bool there = __any_sync(0xffffffffu, row < R);  // else this warp's exponentials are left out
    const float c = p.scale2, growth = __fdiv_rd(kGrowth, c), floor = c > 1.f ? __fdiv_rz(-FLT_MAX, c) : -FLT_MAX;
    const uint64_t c2 = pair(c, c);
    float* const swap = reinterpret_cast<float*>(sm + SM::kSwapOff) + st * 2 * kPreRows;  // [half][place]
    auto meet = [&]() { asm volatile("barrier.cta.sync %0, 64;" ::"r"(st * 4 + quarter + 1) : "memory"); };
    auto all_meet = [&]() { asm volatile("barrier.cta.sync 9, %0;" ::"n"(kSoftmax) : "memory"); };
    auto either = [&](bool mine) {  // a condition on a row of either warp
      uint32_t r;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbarrier.cta.red.or.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
          : "=r"(r)
          : "r"(st * 4 + quarter + 1), "r"((uint32_t)mine)
          : "memory");
      return r != 0;
    };
    // m: the maximum that counts, of the scores as they are; ref: what their exponents are taken from, an addend of the multiply-add. Both this
    // and the limit on growth are rounded such that no weight is above 2^(kGrowth + kLift). far: the row's ref is so large that its last bit
    // counts; the maximum is then taken from the scores before they are multiplied. (Row by row: a row of no numbers has a ref of this kind,
    // and its neighbours keep their bits.)
    // floor: the lowest score that times c is a number, so that every such score counts.
    float m = floor, ref = 0.f, l = 0.f;
    bool far = false;
    for (uint32_t it = 0; it < tiles; ++it) {
      // These scores are there, and the products that were issued before them are done: with NB = 2 that of this stream's last tile is
      // one of them, with NB = 3 that of the tile before. (A warp that gave up still meets the other one.)
      const uint32_t u = 2 * it + st, cS = u % NB * kSP;
      ok = __all_sync(0xffffffffu, ok && wait_for(s_ready(u), s_turn(u), p.wait_cycles));
      if (!there) {
        __syncwarp();
        if (lane == 0) bar_arrive(p_ready(u));
        continue;
      }
      const uint32_t n0 = (first + (twice ? it * 2 + st : it)) * kPreTile + col0;
      // The weights are formed from the maximum as it stands; a row that turns out to have grown too far (the first tile always
      // has) makes its two warps raise their maxima and do the tile again.
      uint64_t sum[2];
      bool raise = it == 0;
      constexpr uint32_t kPart = kMine < 32 ? kMine / 2 : 16;  // registers of packed weights that are stored at once
      for (;;) {
        uint32_t s[kMine];
        fence_after();
        tmem_ld(lanes + cS + col0, s);
        if (n0 + kMine > p.prefix) {  // keys behind the last: nothing (their rows were filled with zeros)
#pragma unroll
          for (uint32_t j = 0; j < kMine; ++j)
            if (n0 + j >= p.prefix) s[j] = 0xff800000u;
        }
        float t[4] = {__uint_as_float(s[0]), __uint_as_float(s[1]), __uint_as_float(s[2]), __uint_as_float(s[3])};
#pragma unroll
        for (uint32_t j = 4; j < kMine; j += 8)
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i)
            t[i] = j + 4 + i < kMine ? fmaxf(fmaxf(t[i], __uint_as_float(s[j + i])), __uint_as_float(s[j + 4 + i])) : fmaxf(t[i], __uint_as_float(s[j + i]));
        float top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
        if (raise) {
          swap[half * kPreRows + place] = top;
          meet();
          top = fmaxf(fmaxf(top, swap[(half ^ 1) * kPreRows + place]), m);
          const float before = ref;
          const bool was_far = far;
          ref = __fadd_ru(__fmul_ru(top, c), -kLift<T>);
          far = fabsf(ref) > kFar;
          if (far) ref = 0.f;  // (and no lift: what a part hands on could not be lower by it)
          if (it) {
            const float lifted = far == was_far ? 0.f : far ? -kLift<T> : kLift<T>;
            const float f = s_ex2(far || was_far ? (m - top) * c + lifted : before - ref);
            l *= f;
            if (NB > 2) ok = __all_sync(0xffffffffu, ok && wait_for(pv_done(st), (it - 1) & 1, p.wait_cycles));
            fence_after();
#pragma unroll 1
            for (uint32_t k = half * (D / 2); k < (half + 1) * (D / 2); k += 16) {
              uint32_t o[16];
              tmem_ld(lanes + cO + k, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st(lanes + cO + k, o);
            }
          }
          m = top;
        }
        sum[0] = sum[1] = 0;
        if (__any_sync(0xffffffffu, far)) {
          const float less = far ? m : 0.f;
#pragma unroll
          for (uint32_t j = 0; j < kMine; ++j) s[j] = __float_as_uint(__uint_as_float(s[j]) - less);
        }
        const uint64_t minus_ref = pair(-ref, -ref);
        auto weights = [&](uint32_t k, uint32_t (&w)[kPart]) {
#pragma unroll
          for (uint32_t j = 0; j < kPart; ++j) {
            float a, b;
            unpair(fma2(pair(__uint_as_float(s[(k * kPart + j) * 2]), __uint_as_float(s[(k * kPart + j) * 2 + 1])), c2, minus_ref), a, b);
            if (j % 4 == 3) {
              poly_ex2(a, b);
            } else {
              a = s_ex2(a);
              b = s_ex2(b);
            }
            sum[j & 1] = add2(sum[j & 1], pair(a, b));
            w[j] = pack2(a, b, T());
          }
        };
        uint32_t w[kPart];
        weights(0, w);
        fence_before();  // (the other warp's scores may lie where this one's weights go: both have read theirs now)
        if (either(top > __fadd_rd(m, growth)) && !raise) {
          raise = true;
          continue;
        }
        fence_after();
        tmem_st(lanes + cS + col0 / 2, w);
        if constexpr (COPIES == 1) {
          uint32_t more[kPart];
          weights(1, more);
          tmem_st(lanes + cS + col0 / 2 + kPart, more);
        } else {  // other copies' keys have no weight here
          uint32_t zero[kPart] = {};
#pragma unroll
          for (uint32_t k = 1; k < COPIES; ++k) tmem_st(lanes + cS + (((copy + k) % COPIES) * kKeys + half * kMine) / 2, zero);
        }
        break;
      }
      float s0, s1;
      unpair(add2(sum[0], sum[1]), s0, s1);
      l += s0 + s1;
      tmem_st_wait();
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(p_ready(u));
    }
    if (tiles) ok = __all_sync(0xffffffffu, ok && wait_for(pv_last(st), 0, p.wait_cycles));
    if (there) {
      swap[half * kPreRows + place] = l;
      meet();
      l += swap[(half ^ 1) * kPreRows + place];
    }
    // Every score -infinity: as if there were no keys.
    // (What a part hands on is rounded as the kernel for the own rows rounds: equal scores stay equal there, however large.)
    float2 ml = make_float2(far ? m * c : ref, l);
    if (m <= floor && l < 0.5f) ml = make_float2(-INFINITY, 0.f);
    // The sums go where Q and the ring were: the first stream's to Q's place (all scores have been multiplied when its last product is
    // done), the second's behind it (everything has); where the streams' number of tiles differs, when both are done. Pieces of 16 bytes,
    // eight by eight in an order that follows from the row: no bank is met twice.
    if (twice) all_meet();
    constexpr uint32_t kPieces = D / 4;
    unsigned char* const sums = sm + st * (kPreRows * D * 4);
    auto piece = [&](uint32_t at, uint32_t e) { return (at * kPieces + (e ^ (at & 7))) * 16; };
    if (there && tiles && ok) {
      fence_after();
#pragma unroll
      for (uint32_t k = 0; k < kPieces / 2; k += 8) {
        uint32_t o[32];
        tmem_ld(lanes + cO + half * (D / 2) + k * 4, o);
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
          const float4 v = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
          *reinterpret_cast<float4*>(sums + piece(place, half * (kPieces / 2) + k + e)) = v;
          shared_attn::note_nan(odd, v);
        }
      }
    }
    if (!shared_attn::is_sum(ml.y)) odd = 0.f;
    if (twice) {
      if (half == 0) {
        swap[place] = ml.x;
        swap[kPreRows + place] = ml.y;
      }
      all_meet();
      const float* const mls = reinterpret_cast<const float*>(sm + SM::kSwapOff);
      for (uint32_t i = tid; i < R * kPieces; i += kSoftmax) {  // a row's streams and copies
        const uint32_t r = i / kPieces, e = i % kPieces;
        float top = -INFINITY, f[2 * COPIES], total = 0.f;
        auto from = [&](uint32_t k) { return (k / COPIES) * 2 * kPreRows + (k % COPIES) * kLanesOf + r; };
#pragma unroll
        for (uint32_t k = 0; k < 2 * COPIES; ++k) top = fmaxf(top, f[k] = mls[from(k)]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (uint32_t k = 0; k < 2 * COPIES; ++k) {
          f[k] = f[k] == -INFINITY ? 0.f : s_ex2(f[k] - top);
          const float lk = mls[from(k) + kPreRows];
          if (f[k] != 0.f || lk != lk) {
            const float4 v = *reinterpret_cast<const float4*>(sm + (k / COPIES) * (kPreRows * D * 4) + piece((k % COPIES) * kLanesOf + r, e));
            acc.x = fmaf(f[k], v.x, acc.x); acc.y = fmaf(f[k], v.y, acc.y); acc.z = fmaf(f[k], v.z, acc.z); acc.w = fmaf(f[k], v.w, acc.w);
            total = fmaf(f[k], lk, total);
          }
        }
        const uint64_t at = ((uint64_t)split * p.kvH + g) * R + r;
        if (e * 4 < d) *reinterpret_cast<float4*>(p.pre_o + at * d + e * 4) = acc;
        if (e == 0) *reinterpret_cast<float2*>(p.pre_ml + at * 2) = make_float2(top, total);
      }
    } else if (there) {
      __syncwarp();
      const uint64_t at0 = ((uint64_t)split * p.kvH + g) * R;
      if (half == 0 && row < R) *reinterpret_cast<float2*>(p.pre_ml + (at0 + row) * 2) = ml;
#pragma unroll 4
      for (uint32_t i = lane; i < 32 * (kPieces / 2); i += 32) {
        const uint32_t r = i / (kPieces / 2), e = half * (kPieces / 2) + i % (kPieces / 2);
        const float4 v = *reinterpret_cast<const float4*>(sums + piece(quarter * 32 + r, e));
        if (row - lane + r < R && e * 4 < d) *reinterpret_cast<float4*>(p.pre_o + (at0 + row - lane + r) * d + e * 4) = v;
      }
    }
  }
  fence_before();
  const uint32_t r0 = tile * kPreRows, r1 = min(R, r0 + 2 * kPreRows);
  const bool mend = __syncthreads_or(odd != odd || !ok);
  // A warp that gave up has arrived where it had not worked, for its own rows and those of others: no row of the CTA is a number then.
  if (mend && __syncthreads_or(!ok)) {
    if (tid == 0 && p.err) atomicOr(p.err, 4u);
    for (uint32_t r = r0 + tid; r < r1; r += kThreads)
      *reinterpret_cast<float2*>(p.pre_ml + (((uint64_t)split * p.kvH + g) * R + r) * 2) = make_float2(0.f, __uint_as_float(0x7fffffffu));
    shared_attn::let_land();  // nobody issues copies or products any more, but some may be in flight
    __syncthreads();
  } else if (mend) {
    shared_attn::mend_shared<T>(p, split, g, r0, r1, first * kPreTile, min(p.prefix, (first + n) * kPreTile), warp, kThreads / 32);
  }
  if (warp == 17) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

template <typename T, int D, int COPIES>
cudaError_t launch_copies(cudaStream_t s, const SharedAttn& p) {
  CUtensorMap mapQ{}, mapK, mapV;
  if (!encode_cache_map16(&mapK, p.kp, 1, p.prefix, p.kvH, p.d, 64, kPreTile) || !encode_cache_map16(&mapV, p.vp, 1, p.prefix, p.kvH, p.d, 64, kPreTile))
    return cudaErrorInvalidValue;
  const uint32_t G = p.qH / p.kvH;
  if (kPreRows / COPIES % G == 0 && !encode_query_map16(&mapQ, p.q, p.B, p.kvH, G, p.d, kPreRows / COPIES / G)) return cudaErrorInvalidValue;
  cudaError_t e = cudaFuncSetAttribute(attn_shared_umma_kernel<T, D, COPIES>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PreSmem<D>::kTotal);
  if (e != cudaSuccess) return e;
  const uint64_t row_tiles = ((uint64_t)p.B * (p.qH / p.kvH) + kPreRows - 1) / kPreRows;
  const uint64_t grid = (row_tiles + 1) / 2 * p.kvH * p.pre_splits;
  if (grid > 0x7fffffffu) return cudaErrorInvalidValue;
  attn_shared_umma_kernel<T, D, COPIES><<<(unsigned)grid, kThreads, PreSmem<D>::kTotal, s>>>(mapQ, mapK, mapV, p, (uint32_t)row_tiles);
  return cudaGetLastError();
}

template <typename T, int D>
cudaError_t launch_pre(cudaStream_t s, const SharedAttn& p) {
  const uint32_t rows = p.B * (p.qH / p.kvH);
  return rows <= 32 ? launch_copies<T, D, 4>(s, p) : rows <= 64 ? launch_copies<T, D, 2>(s, p) : launch_copies<T, D, 1>(s, p);
}

}  // namespace

cudaError_t launch_attn_shared_umma(cudaStream_t s, int dtype, const SharedAttn& p) {
  if (p.d > 128) return cudaErrorInvalidValue;
  if (dtype == 1) return p.d <= 64 ? launch_pre<__half, 64>(s, p) : launch_pre<__half, 128>(s, p);
  if (dtype == 2) return p.d <= 64 ? launch_pre<__nv_bfloat16, 64>(s, p) : launch_pre<__nv_bfloat16, 128>(s, p);
  return cudaErrorInvalidValue;
}

}  // namespace nfai

// The shared rows, once for every sequence: 16-bit types, heads of 64 and 128, on the 5th-generation tensor cores.
//
// The query heads of a KV head and the sequences are one list of rows (row = sequence * G + head of the group). A CTA owns 128 of
// them, one accumulator lane each, and walks a part of the keys in tiles of 128:
//   warp 8   K and V tiles by TMA into a ring of 128-byte swizzled slots, in the order in which they are multiplied
//   warp 9   one lane issues S = Q K^T and O += P V (P in tensor memory, V as it lies: its rows run along N)
//   warps 0-7  softmax, two threads to a row (64 keys each): weights back into tensor memory as the 16-bit operand of the second
//            product, their float32 sums kept; at the end (sums of weighted values, maximum, sum of weights) go to scratch, and the kernel of
//            the own rows joins them.
// Every key is fetched once per 128 rows (the CTAs of further rows find it in L2). With fewer rows than 128 the warps of rows that are
// not there leave the exponentials out. Scores are products of the 16-bit queries as they are; the scale goes into the exponent's
// multiply-add. A row's sums are rescaled only when its maximum has grown by more than 2^8 since the last time.
#include <type_traits>

#include "attn_phases.h"
#include "attn_shared_common.cuh"
#include "umma.cuh"

namespace nfai {

namespace {

using namespace umma;
using shared_attn::kPreRows;
using shared_attn::kPreTile;

constexpr int kThreads = 320;
constexpr float kGrowth = 8.0f;
using Values = ValuePhases<1>;

template <int D>
struct PreSmem {
  static constexpr uint32_t kTile = kPreTile * D * 2;
  static constexpr uint32_t kSlots = D == 64 ? 5 : 2;  // two CTAs on an SM
  static constexpr uint32_t kQ = kPreRows * D * 2;
  static constexpr uint32_t kBarOff = kQ + kSlots * kTile;
  static constexpr uint32_t kSwapOff = kBarOff + 256;
  static constexpr uint32_t kTotal = kSwapOff + 2 * kPreRows * 4 + 1024;
};

__device__ __forceinline__ float p_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2) attn_shared_umma_kernel(const __grid_constant__ CUtensorMap mapK,
                                                                       const __grid_constant__ CUtensorMap mapV, const SharedAttn p,
                                                                       const uint32_t row_tiles) {
  using SM = PreSmem<D>;
  constexpr uint32_t kS = 0, kP = D == 64 ? 128 : 0, kO = D == 64 ? 192 : 128;  // columns of tensor memory
  constexpr bool kAhead = D == 64;  // scores of the next tile beside the weights of this one
  constexpr uint32_t kTypes = (1u << 4) | (std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u);
  extern __shared__ unsigned char pre_raw[];
  unsigned char* const sm = reinterpret_cast<unsigned char*>(((uintptr_t)pre_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* const bars = reinterpret_cast<uint64_t*>(sm + SM::kBarOff);
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * SM::kSlots + 5);
  const uint32_t full0 = s_u32(bars), empty0 = s_u32(bars + SM::kSlots), q_ready = s_u32(bars + 2 * SM::kSlots), s_ready = q_ready + 8,
                 s_free = q_ready + 16, p_ready = q_ready + 24, pv_done = q_ready + 32;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (tid == 0) {
    for (uint32_t i = 0; i < SM::kSlots; ++i) {
      bar_init(full0 + 8 * i, 1);
      bar_init(empty0 + 8 * i, 1);
    }
    bar_init(q_ready, 8);
    bar_init(s_ready, 1);
    bar_init(s_free, 8);
    bar_init(p_ready, 8);
    bar_init(pv_done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_u32(tmem_slot)), "r"(256u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();  // the own rows do not wait for the shared ones, only the join does

  // CTAs of the same keys are neighbours
  const uint32_t G = p.qH / p.kvH, R = p.B * G, tile = blockIdx.x % row_tiles, g = blockIdx.x / row_tiles % p.kvH,
                 split = blockIdx.x / row_tiles / p.kvH;
  const uint32_t row0 = tile * kPreRows, all = (p.prefix + kPreTile - 1) / kPreTile, first = split * p.pre_tiles,
                 n = min(p.pre_tiles, all - first);  // tiles of keys
  bool ok = true;

  if (warp == 8) {
    uint32_t j = 0;
    auto load = [&](const CUtensorMap* map, uint32_t it) {
      const uint32_t s = j % SM::kSlots;
      if (j >= SM::kSlots && !warp_wait(empty0 + 8 * s, (j / SM::kSlots - 1) & 1)) return ok = false;
      if (elect_one()) {
        bar_expect_tx(full0 + 8 * s, SM::kTile);
#pragma unroll
        for (uint32_t b = 0; b < D / 64; ++b)
          tma_load_2d(s_u32(sm) + SM::kQ + s * SM::kTile + b * (kPreTile * 128), map, (int)(g * D + b * 64), (int)((first + it) * kPreTile), full0 + 8 * s);
      }
      ++j;
      return true;
    };
    if constexpr (kAhead) {
      load(&mapK, 0);
      for (uint32_t it = 0; it < n && ok; ++it) {
        if (it + 1 < n && !load(&mapK, it + 1)) break;
        if (!load(&mapV, it)) break;
      }
    } else {
      for (uint32_t it = 0; it < n && ok; ++it)
        if (!load(&mapK, it) || !load(&mapV, it)) break;
    }
    if (ok) ok = drain_ring<SM::kSlots>(empty0, j);
  } else if (warp == 9) {
    // 16-bit operands, float32 sums; A along K in both products; B along K (K tile) or along N (V tile)
    constexpr uint32_t idesc_s = kTypes | ((kPreTile >> 3) << 17) | ((kPreRows >> 4) << 24);
    constexpr uint32_t idesc_o = kTypes | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((kPreRows >> 4) << 24);
    const uint32_t q_s = s_u32(sm);
    uint32_t j = 0;
    auto slot = [&](uint32_t& s) {  // wait for the next tile
      s = j % SM::kSlots;
      ok = warp_wait(full0 + 8 * s, (j / SM::kSlots) & 1);
      fence_after();
      ++j;
      return ok;
    };
    auto scores = [&]() {
      uint32_t s;
      if (!slot(s)) return false;
      if (elect_one()) {
        const uint32_t k_s = q_s + SM::kQ + s * SM::kTile;
#pragma unroll
        for (uint32_t kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * (kPreRows * 128) + (kk & 3) * 32;
          umma_f16(tmem + kS, smem_desc_sw128(q_s + off), smem_desc_sw128(k_s + off), idesc_s, kk != 0);
        }
        umma_commit(empty0 + 8 * s);
        umma_commit(s_ready);
      }
      return true;
    };
    ok = warp_wait(q_ready, 0);
    fence_after();
    if (ok) scores();
    for (uint32_t it = 0; it < n && ok; ++it) {
      if (kAhead && it + 1 < n) {
        if (!(ok = warp_wait(s_free, it & 1))) break;
        fence_after();
        if (!scores()) break;
      }
      if (!(ok = warp_wait(p_ready, it & 1))) break;
      fence_after();
      uint32_t s;
      if (!slot(s)) break;
      if (elect_one()) {
        const uint32_t v_s = q_s + SM::kQ + s * SM::kTile;
#pragma unroll
        for (uint32_t kk = 0; kk < kPreTile / 16; ++kk)
          umma_f16_ta(tmem + kO, tmem + kP + kk * 8, smem_desc_mn_sw128(v_s + kk * 2048, kPreTile * 128), idesc_o, (it | kk) != 0);
        umma_commit(empty0 + 8 * s);
        umma_commit(pv_done);
      }
      // (the weights lie where the next scores go: products of one thread run in their order)
      if (!kAhead && it + 1 < n && !scores()) break;
    }
  } else {
    {  // the rows of Q as they are
      constexpr uint32_t kLanes = D / 8, kRows = 32 / kLanes;
      const uint32_t c = (lane % kLanes) * 8;
      const T* const q = reinterpret_cast<const T*>(p.q);
#pragma unroll
      for (uint32_t i = 0; i < 16; i += kRows) {
        const uint32_t r = warp * 16 + i + lane / kLanes, row = row0 + r, b = row / G;
        const uint4 v = row < R ? __ldg(reinterpret_cast<const uint4*>(q + ((uint64_t)b * p.qH + g * G + (row - b * G)) * D + c)) : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(sm + (c >> 6) * (kPreRows * 128) + r * 128 + ((((c & 63) >> 3) ^ (r & 7)) << 4)) = v;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive(q_ready);
    }
    const uint32_t quarter = warp & 3, half = warp >> 2, col0 = half * (kPreTile / 2), r_own = quarter * 32 + lane, row = row0 + r_own;
    const uint32_t lanes = tmem + (quarter * 32u << 16);
    const bool there = row0 + quarter * 32 < R;  // some row of this warp is: else its exponentials are left out
    const float c = p.scale2, growth = kGrowth / c, floor = c > 1.f ? -1e38f / c : -1e38f;
    const uint64_t c2 = pair(c, c);
    float* const swap = reinterpret_cast<float*>(sm + SM::kSwapOff);  // [2][kPreRows]
    auto meet = [&]() { asm volatile("barrier.cta.sync %0, 64;" ::"r"(quarter + 1) : "memory"); };
    auto either = [&](bool mine) {  // a condition on a row of either warp
      uint32_t r;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbarrier.cta.red.or.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
          : "=r"(r)
          : "r"(quarter + 1), "r"((uint32_t)mine)
          : "memory");
      return r != 0;
    };
    auto value = [&](uint32_t j) {  // the product of tile j with its values is done
      ok = __all_sync(0xffffffffu, ok && bar_wait(pv_done, Values::parity(j)));
    };
    float m = 0.f, l = 0.f;  // m: of the scores as they are
    for (uint32_t it = 0; it < n; ++it) {
      ok = __all_sync(0xffffffffu, ok && bar_wait(s_ready, it & 1));  // (a warp that gave up still meets the other one)
      if (!kAhead) Values::at_tile(it, value);
      if (!there) {
        if (kAhead) {
          __syncwarp();
          if (lane == 0) bar_arrive(s_free);
          Values::at_tile(it, value);
        }
        __syncwarp();
        if (lane == 0) bar_arrive(p_ready);
        continue;
      }
      const uint32_t n0 = (first + it) * kPreTile + col0;
      // The weights are formed from the maximum as it stands; a row that turns out to have grown too far (the first tile always
      // has) makes its two warps raise their maxima and do the tile again.
      uint64_t sum[2];
      bool raise = it == 0;
      for (;;) {
        uint32_t s[kPreTile / 2];
        fence_after();
        tmem_ld(lanes + kS + col0, s);
        if (n0 + kPreTile / 2 > p.prefix) {  // keys behind the last: nothing (their rows were filled with zeros)
#pragma unroll
          for (uint32_t j = 0; j < kPreTile / 2; ++j)
            if (n0 + j >= p.prefix) s[j] = 0xff800000u;
        }
        float t[4] = {__uint_as_float(s[0]), __uint_as_float(s[1]), __uint_as_float(s[2]), __uint_as_float(s[3])};
#pragma unroll
        for (uint32_t j = 4; j < kPreTile / 2; j += 8)
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i)
            t[i] = j + 4 + i < kPreTile / 2 ? fmaxf(fmaxf(t[i], __uint_as_float(s[j + i])), __uint_as_float(s[j + 4 + i])) : fmaxf(t[i], __uint_as_float(s[j + i]));
        float top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
        if (raise) {
          swap[half * kPreRows + r_own] = top;
          meet();
          top = fmaxf(fmaxf(top, swap[(half ^ 1) * kPreRows + r_own]), it ? m : floor);
          if (it) {
            Values::at_rescaling(it, value);
            fence_after();
            const float f = p_ex2((m - top) * c);
            l *= f;
#pragma unroll 1
            for (uint32_t k = half * (D / 2); k < (half + 1) * (D / 2); k += 16) {
              uint32_t o[16];
              tmem_ld(lanes + kO + k, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st(lanes + kO + k, o);
            }
          }
          m = top;
        }
        sum[0] = sum[1] = 0;
        const uint64_t minus_m = pair(-m * c, -m * c);
        uint32_t w[2][16];
        auto weights = [&](uint32_t k) {
#pragma unroll
          for (uint32_t j = 0; j < 16; ++j) {
            const uint64_t x = fma2(pair(__uint_as_float(s[k * 32 + 2 * j]), __uint_as_float(s[k * 32 + 2 * j + 1])), c2, minus_m);
            float a, b;
            unpair(x, a, b);
            a = p_ex2(a);
            b = p_ex2(b);
            sum[j & 1] = add2(sum[j & 1], pair(a, b));
            w[k][j] = pack2(a, b, T());
          }
        };
        weights(0);
        if (!kAhead) fence_before();  // (the other warp's scores may lie where this one's weights go: both have read theirs now)
        if (either(top > m + growth) && !raise) {
          raise = true;
          continue;
        }
        if (!kAhead) fence_after();
        if (kAhead) {
          fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(s_free);
          Values::at_tile(it, value);  // the weights of the tile before have been used
          fence_after();
        }
        tmem_st(lanes + kP + col0 / 2, w[0]);
        weights(1);
        tmem_st(lanes + kP + col0 / 2 + 16, w[1]);
        break;
      }
      float s0, s1;
      unpair(add2(sum[0], sum[1]), s0, s1);
      l += s0 + s1;
      tmem_st_wait();
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(p_ready);
    }
    Values::at_end(n, value);
    if (there) {
      swap[half * kPreRows + r_own] = l;
      meet();
      l += swap[(half ^ 1) * kPreRows + r_own];
      const uint64_t at = ((uint64_t)split * p.kvH + g) * R + row;
      if (row < R && half == 0) {
        // Every score -infinity (a row's sum has the 1 of its maximum otherwise): as if there were no keys. A wait that gave up: NaN.
        float2 ml = make_float2(m * c, l);
        if (l < 0.5f) ml = make_float2(-INFINITY, 0.f);
        if (!ok) ml = make_float2(0.f, __uint_as_float(0x7fffffffu));
        *reinterpret_cast<float2*>(p.pre_ml + at * 2) = ml;
      }
      if (ok) {
        fence_after();
        float* const out = p.pre_o + at * D;
#pragma unroll 1
        for (uint32_t k = half * (D / 2); k < (half + 1) * (D / 2); k += 32) {
          uint32_t o[32];
          tmem_ld(lanes + kO + k, o);
          if (row >= R) continue;
#pragma unroll
          for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(out + k + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
      }
    }
  }
  if (!ok) {
    if (lane == 0 && p.err) atomicOr(p.err, 4u);
    // copies and products of this CTA may still be in flight: a bounded time for them to end before their memory is released
    for (volatile uint32_t spin = 0; spin < (1u << 20); ++spin) {
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256u) : "memory");
}

template <typename T, int D>
cudaError_t launch_pre(cudaStream_t s, const SharedAttn& p) {
  CUtensorMap mapK, mapV;
  const uint64_t width = (uint64_t)p.kvH * D;
  if (!encode_tile_map16(&mapK, p.kp, p.prefix, width, kPreTile) || !encode_tile_map16(&mapV, p.vp, p.prefix, width, kPreTile)) return cudaErrorInvalidValue;
  cudaError_t e = cudaFuncSetAttribute(attn_shared_umma_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PreSmem<D>::kTotal);
  if (e != cudaSuccess) return e;
  const uint64_t row_tiles = ((uint64_t)p.B * (p.qH / p.kvH) + kPreRows - 1) / kPreRows, grid = row_tiles * p.kvH * p.pre_splits;
  if (grid > 0x7fffffffu) return cudaErrorInvalidValue;
  attn_shared_umma_kernel<T, D><<<(unsigned)grid, kThreads, PreSmem<D>::kTotal, s>>>(mapK, mapV, p, (uint32_t)row_tiles);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attn_shared_umma(cudaStream_t s, int dtype, const SharedAttn& p) {
  if (dtype == 1) return p.d == 64 ? launch_pre<__half, 64>(s, p) : p.d == 128 ? launch_pre<__half, 128>(s, p) : cudaErrorInvalidValue;
  if (dtype == 2) return p.d == 64 ? launch_pre<__nv_bfloat16, 64>(s, p) : p.d == 128 ? launch_pre<__nv_bfloat16, 128>(s, p) : cudaErrorInvalidValue;
  return cudaErrorInvalidValue;
}

}  // namespace nfai

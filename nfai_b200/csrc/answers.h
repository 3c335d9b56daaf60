// Launch interface of the operators of a step of several answers to one prompt (rope_rows.cu, attn_shared*.cu, logit_rules.cu);
// their entry points are in answers_api.cu.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace nfai {

// ---- rotary rows ---------------------------------------------------------------------------------------------------------
struct RopeRows {
  const void* x = nullptr;            // [rows][x_stride], of which (qH + 2 kvH) * d elements: queries, keys, values
  uint64_t x_stride = 0;
  uint32_t rows = 0, qH = 0, kvH = 0, d = 0;
  uint32_t dims = 0;                  // the first `dims` elements of a query or key head are turned
  int halves = 0;                     // 0: pairs (2i, 2i + 1), 1: (i, i + dims / 2)
  const double* freqs = nullptr;      // [dims / 2] radians per position
  float magnitude = 1.f;
  const int32_t* positions = nullptr; // [rows]
  const int32_t* slots = nullptr;     // [rows] cache rows; null: row r
  uint64_t cache_rows = 0;
  void* q = nullptr;                  // [rows][qH * d]
  void* k = nullptr;                  // [cache_rows][kvH * d]
  void* v = nullptr;
};
cudaError_t launch_rope_rows(cudaStream_t s, int x_dtype, int out_dtype, const RopeRows& p);

// ---- rules on logits -------------------------------------------------------------------------------------------------------
struct LogitRules {
  const float* logits = nullptr;      // [rows][V]
  float* out = nullptr;               // [rows][V], may be logits
  uint32_t rows = 0, V = 0;
  const uint32_t* history = nullptr;  // [rows][history_stride]
  uint32_t history_stride = 0;
  const int32_t* history_len = nullptr;  // null: all of them
  const float* repetition = nullptr;  // [rows] each; null: 1, 0, 0
  const float* frequency = nullptr;
  const float* presence = nullptr;
  const int32_t* bias_start = nullptr;  // [rows + 1]
  const uint32_t* bias_ids = nullptr;
  const float* bias = nullptr;
  uint32_t n_bias = 0;
  const uint32_t* masks = nullptr;    // [n_masks][(V + 31) / 32]
  uint32_t n_masks = 0;
  const int32_t* mask_rows = nullptr; // [rows]; null: row r has mask r
  uint32_t* err = nullptr;            // device word of the context; may be null
  uint32_t wait_cycles = 2000000000u; // budget of a wait
};
cudaError_t launch_logit_rules(cudaStream_t s, const LogitRules& p);

// ---- attention over shared rows ----------------------------------------------------------------------------------------------
struct SharedAttn {
  const void* q = nullptr;            // [B][qH * d]
  const void* kp = nullptr;           // [prefix][kvH * d]
  const void* vp = nullptr;
  const void* ko = nullptr;           // [B][capacity][kvH * d]
  const void* vo = nullptr;
  const int32_t* lens = nullptr;      // [B] own rows of each; negative: the place is free
  uint32_t prefix = 0, capacity = 0, B = 0, qH = 0, kvH = 0, d = 0;
  float scale2 = 0.f;                 // scale * log2(e)
  void* out = nullptr;                // [B][qH * d]
  // scratch, in floats: sums [..][d] and (maximum, sum of weights) of partial results
  float* pre_o = nullptr;             // [pre_splits][kvH][B * G][d]
  float* pre_ml = nullptr;            // [pre_splits][kvH][B * G][2]
  float* own_o = nullptr;             // [own_splits][B * qH][d]
  float* own_ml = nullptr;            // [own_splits][B * qH][2]
  uint32_t pre_splits = 0, pre_tiles = 0;  // parts of the shared rows, tiles of keys per CTA; 0: they are walked like a sequence's own
  uint32_t own_splits = 1, own_least = 64; // parts of a sequence's keys at most, and keys of a part at least
  bool joined = false;                // partial results go to scratch and a last kernel joins them (else the CTAs of a row do, if it has more than one)
  uint32_t* err = nullptr;            // device word of the context; may be null
  uint32_t wait_cycles = 2000000000u; // budget of a wait
};
// What the sizes alone decide: which kernels run, into how many parts, and what scratch they need.
struct SharedPlan {
  uint32_t pre_warps = 0;             // shared rows on the CUDA cores: warps of a CTA (0: on tcgen05)
  bool tensor = false;                // own rows on the warp-level tensor kernel (else CUDA cores)
  uint32_t rows = 8;                  // query heads per CTA there
  uint32_t pre_splits = 0, pre_tiles = 0, own_splits = 1, own_least = 64;
  bool joined = false;
  size_t pre_o = 0, pre_ml = 0, own_o = 0, own_ml = 0, total = 0;  // byte offsets
};
SharedPlan plan_shared_attn(int dtype, uint32_t B, uint32_t qH, uint32_t kvH, uint32_t d, uint32_t prefix, uint32_t capacity);
// Scratch that serves these sizes and every smaller batch, prefix and capacity: grows with each of them, as a plan's own does not.
size_t shared_attn_scratch(int dtype, uint32_t B, uint32_t qH, uint32_t kvH, uint32_t d, uint32_t prefix, uint32_t capacity);
// the shared rows, partial results into pre_o and pre_ml; and everything else on the warp-level products
cudaError_t launch_attn_shared_umma(cudaStream_t s, int dtype, const SharedAttn& p);
cudaError_t launch_attn_shared_rows(cudaStream_t s, const SharedAttn& p, uint32_t warps);  // float32, eight queries a warp
uint32_t attn_shared_rows_keys(uint32_t d);                                                // keys of its tiles
cudaError_t launch_attn_shared_mma(cudaStream_t s, int dtype, const SharedAttn& p, uint32_t rows);
cudaError_t launch_shared_attn(cudaStream_t s, int dtype, const SharedAttn& p, const SharedPlan& plan);

}  // namespace nfai

// Entry points of the operators of a step of several answers to one prompt. Arguments are checked before anything else, so that what
// is refused is refused without a device too.
#include <float.h>
#include <math.h>

#include "answers.h"
#include "model.h"

namespace {

// The context's device for the length of a call; the caller's current device is as it was afterwards. Set even where it is the current
// one already: in a thread that has not used the device yet, this is what makes its context current (tensor maps need one).
struct OnDevice {
  int before = -1;
  cudaError_t err;
  explicit OnDevice(int device) {
    err = cudaGetDevice(&before);
    if (err != cudaSuccess || before == device) before = -1;  // nothing to put back
    if (err == cudaSuccess) err = cudaSetDevice(device);
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

// `stream` null: the context's stream, and the result is there on return; else the work is put on that stream.
// waits: the kernels have waits that may give up, which they note in a word of the context (calls on a stream before this one, too).
cudaStream_t stream_of(nfai_ctx* c, void* stream) { return stream ? static_cast<cudaStream_t>(stream) : c->stream; }
int finish(nfai_ctx* c, void* stream, cudaError_t launched, bool waits) {
  if (launched != cudaSuccess)
    return fail(c, launched == cudaErrorInvalidValue ? NFAI_ERR_ARG : NFAI_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(launched));
  if (stream) return NFAI_OK;
  uint32_t err = 0;
  if (waits) CU(c, cudaMemcpyAsync(&err, c->answers_note(), 4, cudaMemcpyDeviceToHost, c->stream));
  CU(c, cudaStreamSynchronize(c->stream));
  if (!err) return NFAI_OK;
  CU(c, cudaMemsetAsync(c->answers_note(), 0, 4, c->stream));
  return fail(c, NFAI_ERR_TIMEOUT, "a bounded device-side wait gave up");
}
uint32_t budget(const nfai_ctx* c) { return 2 * (uint32_t)(c->wait_ns < 2000000000ull ? c->wait_ns : 2000000000ull); }  // in cycles
bool known_dtype(int t) { return t == NFAI_F32 || t == NFAI_F16 || t == NFAI_BF16; }
#define ON_DEVICE(c)                                        \
  if (!(c)) return fail(nullptr, NFAI_ERR_ARG, "ctx is null"); \
  OnDevice on_device((c)->device);                          \
  if (on_device.err != cudaSuccess) return fail((c), NFAI_ERR_CUDA, "cudaSetDevice: %s", cudaGetErrorString(on_device.err))

constexpr double kPi = 3.14159265358979323846, kLog2e = 1.4426950408889634;

}  // namespace

extern "C" {

int nfai_rope_frequencies(uint32_t dims, double base, int scaling, double factor, double a, double b, uint32_t trained, double* freqs,
                          float* magnitude) {
  if (!freqs || !dims || (dims & 1)) return fail(nullptr, NFAI_ERR_ARG, "freqs is null, or dims is not even");
  if (!(base > 1.0) || !isfinite(base)) return fail(nullptr, NFAI_ERR_ARG, "base must be above 1");
  if (scaling < NFAI_ROPE_PLAIN || scaling > NFAI_ROPE_YARN) return fail(nullptr, NFAI_ERR_ARG, "unknown scaling %d", scaling);
  if (scaling != NFAI_ROPE_PLAIN && (!(factor >= 1.0) || !isfinite(factor))) return fail(nullptr, NFAI_ERR_ARG, "factor must be at least 1");
  if (scaling == NFAI_ROPE_BANDS && (!(a > 0.0) || !(b > a) || !isfinite(b) || !trained))
    return fail(nullptr, NFAI_ERR_ARG, "bands need 0 < a < b and the context the model was trained with");
  if (scaling == NFAI_ROPE_YARN && (!(b > 0.0) || !(a > b) || !isfinite(a) || !trained))
    return fail(nullptr, NFAI_ERR_ARG, "yarn needs a > b > 0 and the context the model was trained with");
  double lo = 0.0, hi = 0.0;
  if (scaling == NFAI_ROPE_YARN) {
    // the pair (as an element count over the head) that turns `turns` times within the trained context
    auto place = [&](double turns) { return dims * log(trained / (turns * 2.0 * kPi)) / (2.0 * log(base)); };
    lo = fmax(0.0, floor(place(a)));
    hi = fmin(dims - 1.0, ceil(place(b)));
  }
  for (uint32_t i = 0; i < dims / 2; ++i) {
    double f = pow(base, -2.0 * i / dims);
    double keep = 1.0;  // of the frequency as it was trained
    if (scaling == NFAI_ROPE_LINEAR) keep = 0.0;
    if (scaling == NFAI_ROPE_BANDS) keep = fmin(1.0, fmax(0.0, (trained * f / (2.0 * kPi) - a) / (b - a)));
    if (scaling == NFAI_ROPE_YARN) keep = 1.0 - fmin(1.0, fmax(0.0, (i - lo) / fmax(hi - lo, 0.001)));
    freqs[i] = scaling == NFAI_ROPE_PLAIN ? f : keep * f + (1.0 - keep) * f / factor;
  }
  if (magnitude) *magnitude = scaling == NFAI_ROPE_YARN ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
  return NFAI_OK;
}

int nfai_op_rope_rows(nfai_ctx* c, const void* x, int x_dtype, uint64_t x_stride, uint32_t rows, uint32_t qH, uint32_t kvH, uint32_t d,
                      uint32_t dims, int layout, const double* freqs, float magnitude, const int32_t* positions, const int32_t* slots,
                      void* q_out, void* k_cache, void* v_cache, int out_dtype, uint64_t cache_rows, void* stream) {
  const uint64_t width = ((uint64_t)qH + 2ull * kvH) * d;
  if (!known_dtype(x_dtype) || !known_dtype(out_dtype)) return fail(c, NFAI_ERR_ARG, "unknown element type");
  if (qH > 65536 || kvH > 65536 || d > 65536 || !d || !(qH + kvH)) return fail(c, NFAI_ERR_ARG, "heads and their size must be in 1 .. 65536");
  if (dims > d || (dims & 1)) return fail(c, NFAI_ERR_ARG, "dims must be even and at most d");
  if (layout != NFAI_ROPE_PAIRS && layout != NFAI_ROPE_HALVES) return fail(c, NFAI_ERR_ARG, "unknown layout %d", layout);
  if (x_stride && x_stride < width) return fail(c, NFAI_ERR_ARG, "x_stride is shorter than a row");
  if (rows > 0x7fffffffu) return fail(c, NFAI_ERR_ARG, "too many rows");
  if (width > 0x7fffffffull) return fail(c, NFAI_ERR_ARG, "a row is too long");
  if (!x || (dims && (!freqs || !positions)) || (qH && !q_out) || (kvH && (!k_cache || !v_cache))) return fail(c, NFAI_ERR_ARG, "null argument");
  const size_t es = dtype_size(out_dtype), xs = dtype_size(x_dtype);
  if (((uintptr_t)q_out | (uintptr_t)k_cache | (uintptr_t)v_cache) % es || (uintptr_t)x % xs || (uintptr_t)freqs % 8 ||
      ((uintptr_t)positions | (uintptr_t)slots) % 4)
    return fail(c, NFAI_ERR_ARG, "a pointer is not aligned to its elements");
  ON_DEVICE(c);
  if (!rows) return NFAI_OK;
  RopeRows p;
  p.x = x; p.x_stride = x_stride ? x_stride : width; p.rows = rows; p.qH = qH; p.kvH = kvH; p.d = d; p.dims = dims;
  p.halves = layout == NFAI_ROPE_HALVES; p.freqs = freqs; p.magnitude = magnitude; p.positions = positions; p.slots = slots;
  p.cache_rows = cache_rows; p.q = q_out; p.k = k_cache; p.v = v_cache;
  return finish(c, stream, launch_rope_rows(stream_of(c, stream), x_dtype, out_dtype, p), false);
}

int nfai_op_logit_rules(nfai_ctx* c, const float* logits, uint32_t rows, uint32_t V, const uint32_t* history, uint32_t history_stride,
                        const int32_t* history_len, const float* repetition, const float* frequency, const float* presence,
                        const int32_t* bias_start, const uint32_t* bias_ids, const float* bias, uint32_t n_bias, const uint32_t* masks,
                        uint32_t n_masks, const int32_t* mask_rows, float* out, void* stream) {
  if (!logits || !out || !V) return fail(c, NFAI_ERR_ARG, "null argument, or no vocabulary");
  if (V > 0x7fffffffu - 4096 || rows > 0x7fffffffu) return fail(c, NFAI_ERR_ARG, "too many rows or tokens");
  if (n_bias > 0x7ffffffeu || (n_bias && (!bias_start || !bias_ids || !bias))) return fail(c, NFAI_ERR_ARG, "biases need their starts, ids and values");
  if (n_masks && !masks) return fail(c, NFAI_ERR_ARG, "masks is null");
  if (n_masks && !mask_rows && n_masks < rows) return fail(c, NFAI_ERR_ARG, "without mask_rows every row needs a mask of its own: %u masks, %u rows", n_masks, rows);
  if (((uintptr_t)logits | (uintptr_t)out | (uintptr_t)history | (uintptr_t)history_len | (uintptr_t)repetition | (uintptr_t)frequency |
       (uintptr_t)presence | (uintptr_t)bias_start | (uintptr_t)bias_ids | (uintptr_t)bias | (uintptr_t)masks | (uintptr_t)mask_rows) & 3)
    return fail(c, NFAI_ERR_ARG, "a pointer is not aligned to its elements");
  const uint64_t bytes = (uint64_t)rows * V * 4, at = (uintptr_t)logits, to = (uintptr_t)out;
  if (at != to && at < to + bytes && to < at + bytes) return fail(c, NFAI_ERR_ARG, "out overlaps logits without being the same buffer");
  ON_DEVICE(c);
  if (!rows) return NFAI_OK;
  LogitRules p;
  p.logits = logits; p.out = out; p.rows = rows; p.V = V;
  p.history = history; p.history_stride = history ? history_stride : 0; p.history_len = history_len;
  p.repetition = repetition; p.frequency = frequency; p.presence = presence;
  p.bias_start = bias_start; p.bias_ids = bias_ids; p.bias = bias; p.n_bias = n_bias;
  p.masks = masks; p.n_masks = n_masks; p.mask_rows = mask_rows; p.err = c->answers_note(); p.wait_cycles = budget(c);
  return finish(c, stream, launch_logit_rules(stream_of(c, stream), p), true);
}

// What is wrong with the sizes of an attention call; null: nothing.
static const char* bad_attn_sizes(int dtype, uint32_t B, uint32_t qH, uint32_t kvH, uint32_t d, uint32_t prefix, uint32_t capacity) {
  if (!known_dtype(dtype)) return "unknown element type";
  if (!qH || !kvH || qH % kvH || qH > 65536) return "query heads must be a multiple of the KV heads";
  if (!d || d % 8 || d > 256) return "the head size must be a multiple of 8 up to 256";
  if ((uint64_t)B * qH > 0x1000000ull) return "too many sequences times heads";
  if (prefix > 0x3fffffffu || capacity > 0x3fffffffu) return "too many rows";
  return nullptr;
}

size_t nfai_op_attn_shared_scratch_bytes(int dtype, uint32_t B, uint32_t qH, uint32_t kvH, uint32_t d, uint32_t prefix, uint32_t capacity) {
  if (!B || bad_attn_sizes(dtype, B, qH, kvH, d, prefix, capacity)) return 0;
  return shared_attn_scratch(dtype, B, qH, kvH, d, prefix, capacity);
}

int nfai_op_attn_shared(nfai_ctx* c, const void* q, const void* k_prefix, const void* v_prefix, uint32_t prefix, const void* k_own,
                        const void* v_own, uint32_t capacity, const int32_t* lens, int dtype, uint32_t B, uint32_t qH, uint32_t kvH,
                        uint32_t d, float scale, void* out, void* scratch, size_t scratch_bytes, void* stream) {
  if (const char* wrong = bad_attn_sizes(dtype, B, qH, kvH, d, prefix, capacity)) return fail(c, NFAI_ERR_ARG, "%s", wrong);
  if (!(scale >= 0.f) || scale * kLog2e > FLT_MAX) return fail(c, NFAI_ERR_ARG, "scale must be positive, or 0 for 1 / sqrt(d), and below 2^127.4");
  if (B) {
    if (!q || !out || !lens || !scratch || (prefix && (!k_prefix || !v_prefix)) || (capacity && (!k_own || !v_own)))
      return fail(c, NFAI_ERR_ARG, "null argument");
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_prefix | (uintptr_t)v_prefix | (uintptr_t)k_own | (uintptr_t)v_own) & 15 || (uintptr_t)lens & 3 ||
        (uintptr_t)scratch & 255)
      return fail(c, NFAI_ERR_ARG, "pointers must be 16-byte aligned, scratch 256");
  }
  const SharedPlan plan = B ? plan_shared_attn(dtype, B, qH, kvH, d, prefix, capacity) : SharedPlan();
  // (as much as ..scratch_bytes says, which is never less than the plan's: what is refused follows from the sizes in a way that a host can use)
  const size_t bound = B ? shared_attn_scratch(dtype, B, qH, kvH, d, prefix, capacity) : 0, need = plan.total > bound ? plan.total : bound;
  if (scratch_bytes < need) return fail(c, NFAI_ERR_ARG, "scratch too small: %zu < %zu", scratch_bytes, need);
  ON_DEVICE(c);
  if (!B) return NFAI_OK;
  SharedAttn p;
  char* const base = static_cast<char*>(scratch);
  p.q = q; p.kp = k_prefix; p.vp = v_prefix; p.ko = k_own; p.vo = v_own; p.lens = lens; p.prefix = prefix; p.capacity = capacity;
  p.B = B; p.qH = qH; p.kvH = kvH; p.d = d; p.out = out;
  p.scale2 = (float)((scale > 0.f ? (double)scale : 1.0 / sqrt((double)d)) * kLog2e);
  p.pre_o = (float*)(base + plan.pre_o); p.pre_ml = (float*)(base + plan.pre_ml);
  p.own_o = (float*)(base + plan.own_o); p.own_ml = (float*)(base + plan.own_ml);
  p.pre_splits = plan.pre_splits; p.pre_tiles = plan.pre_tiles; p.own_splits = plan.own_splits; p.own_least = plan.own_least; p.joined = plan.joined;
  p.err = c->answers_note(); p.wait_cycles = budget(c);
  return finish(c, stream, launch_shared_attn(stream_of(c, stream), dtype, p, plan), true);
}

}  // extern "C"

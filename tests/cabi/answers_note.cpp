// What becomes of the note of a bounded wait that gave up in attention over shared rows or rules on logits: the words of a context are
// written as the kernels write them, and the entry points are called. Exit code 0, or the line of the first check that does not hold.
#include <cstdio>

#include "model.h"

#define CHECK(x)                                   \
  do {                                             \
    if (!(x)) {                                    \
      printf("line %d: %s\n", __LINE__, #x);       \
      return __LINE__ & 0x7f ? __LINE__ & 0x7f : 1; \
    }                                              \
  } while (0)

int main() {
  nfai_ctx* c = nullptr;
  CHECK(nfai_ctx_create(0, &c) == NFAI_OK);
  // one float of each logit, and matrices and caches of zeros
  constexpr size_t kBytes = 1 << 20;
  char* mem = nullptr;
  CHECK(cudaMalloc((void**)&mem, kBytes) == cudaSuccess && cudaMemset(mem, 0, kBytes) == cudaSuccess);
  float *const logits = (float*)mem, *const out = (float*)(mem + 4096), *const product = (float*)(mem + 65536);
  void *const a = mem + 131072, *const w = mem + 196608, *const scratch = mem + 262144;
  const size_t need = nfai_op_attn_shared_scratch_bytes(NFAI_F32, 1, 2, 1, 32, 4, 0);
  CHECK(need && need < kBytes / 2);
  auto write = [&](uint32_t* word, uint32_t bits) { return cudaMemcpy(word, &bits, 4, cudaMemcpyHostToDevice) == cudaSuccess && cudaDeviceSynchronize() == cudaSuccess; };
  auto read = [&](const uint32_t* word) {
    uint32_t v = 0xdead;
    cudaMemcpy(&v, word, 4, cudaMemcpyDeviceToHost);
    return v;
  };
  auto rules = [&](void* stream) {
    return nfai_op_logit_rules(c, logits, 1, 100, nullptr, 0, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0, nullptr, 0, nullptr, out, stream);
  };
  auto attend = [&](void* stream) {  // (the lengths are zeros, the shared rows too)
    return nfai_op_attn_shared(c, a, w, w, 4, nullptr, nullptr, 0, (const int32_t*)logits, NFAI_F32, 1, 2, 1, 32, 0.f, out, scratch, need, stream);
  };
  auto gemm = [&]() { return nfai_op_gemm(c, a, w, NFAI_F16, 16, 64, 64, product); };
  auto rope = [&]() { return nfai_op_rope_rows(c, a, NFAI_F32, 0, 1, 2, 0, 32, 0, 0, nullptr, 1.f, nullptr, nullptr, out, nullptr, nullptr, NFAI_F32, 0, nullptr); };
  CHECK(rules(nullptr) == NFAI_OK && attend(nullptr) == NFAI_OK && gemm() == NFAI_OK && rope() == NFAI_OK);

  // A kernel gave up on a stream; a product, rotary rows and further work on the stream follow.
  for (int k = 0; k < 2; ++k) {
    CHECK(write(c->answers_note(), 4));
    CHECK(gemm() == NFAI_OK && rope() == NFAI_OK && rules(cudaStreamLegacy) == NFAI_OK && attend(cudaStreamLegacy) == NFAI_OK);
    CHECK(cudaDeviceSynchronize() == cudaSuccess && gemm() == NFAI_OK);
    CHECK((k ? rules(nullptr) : attend(nullptr)) == NFAI_ERR_TIMEOUT);
    CHECK(rules(nullptr) == NFAI_OK && attend(nullptr) == NFAI_OK && read(c->answers_note()) == 0);
  }
  // Another operator's word
  CHECK(write(c->dev_err, 4));
  CHECK(rules(nullptr) == NFAI_OK && attend(nullptr) == NFAI_OK && read(c->dev_err) == 4);
  CHECK(gemm() == NFAI_OK && read(c->dev_err) == 0);
  cudaFree(mem);
  CHECK(nfai_ctx_destroy(c) == NFAI_OK);
  puts("ok");
  return 0;
}

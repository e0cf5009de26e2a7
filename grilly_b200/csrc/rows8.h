// Shared by the 8-bit row kernels (rows8.cu) and their matrix products (gemm8.cu).
#pragma once
#include "internal.h"
#include <new>

namespace gb {

// Smallest scale of a row: 2^-126, the smallest normal fp32 number, so that 1 / scale is finite for every row.
constexpr float ROWS8_TINY = 1.17549435e-38f;

// Runs the body of an entry point under the context's lock, on the context's device (the caller's current device is
// put back), and turns what C++ would throw into a status: nothing may unwind into a C caller.
template <class F>
int rows8_entry(grilly_ctx* ctx, F&& body) noexcept {
  if (!ctx) return GRILLY_ERR_INVALID_ARG;
  int before = -1;
  int rc = GRILLY_ERR_CUDA;
  try {
    std::lock_guard<std::mutex> lock(ctx->mu);
    if (cudaGetDevice(&before) != cudaSuccess) before = -1;
    if (before != ctx->device && cudaSetDevice(ctx->device) != cudaSuccess) return set_error(ctx, GRILLY_ERR_CUDA, "cudaSetDevice failed");
    rc = body();
  } catch (const std::bad_alloc&) {
    rc = GRILLY_ERR_OOM;
  } catch (...) {
    rc = GRILLY_ERR_CUDA;
  }
  if (before >= 0 && before != ctx->device) cudaSetDevice(before);
  return rc;
}

// Scratch of one call from the stream-ordered pool: taken and given back on the context's stream, so calls on other
// streams and captured graphs never share it. One allocation a call: parts are reserved first, then take() gets them all.
class Rows8Scratch {
 public:
  explicit Rows8Scratch(grilly_ctx* c) : ctx(c) {}
  Rows8Scratch(const Rows8Scratch&) = delete;
  // offset of a part of `bytes` bytes, on a 256-byte boundary
  size_t reserve(size_t bytes) {
    const size_t at = total;
    total += (bytes + 255) / 256 * 256;
    return at;
  }
  int take() {
    if (!total) return GRILLY_OK;
    const cudaError_t e = cudaMallocAsync(&p, total, ctx->stream);
    if (e == cudaSuccess) return GRILLY_OK;
    cudaGetLastError();
    p = nullptr;
    return set_error(ctx, e == cudaErrorMemoryAllocation ? GRILLY_ERR_OOM : GRILLY_ERR_CUDA,
                     std::string("8-bit rows: scratch: ") + cudaGetErrorString(e));
  }
  template <class T>
  T* at(size_t offset) const { return reinterpret_cast<T*>(static_cast<char*>(p) + offset); }
  ~Rows8Scratch() { if (p) cudaFreeAsync(p, ctx->stream); }

 private:
  grilly_ctx* ctx;
  void* p = nullptr;
  size_t total = 0;
};

// Checks the geometry of an 8-bit row tensor. Indices within a row are 32-bit, with room for a block's stride above them.
constexpr long long ROWS8_MAX_FEATURES = 1ll << 30;
inline int rows8_check(grilly_ctx* ctx, const char* who, const void* q, const void* scale, long long rows, int features, long long ld) {
  if (rows < 0 || features < 1) return set_error(ctx, GRILLY_ERR_INVALID_ARG, std::string(who) + ": rows must not be negative and features must be positive");
  if (ld < features || ld % 16 != 0) return set_error(ctx, GRILLY_ERR_INVALID_ARG, std::string(who) + ": the rows' pitch must be a multiple of 16 and at least the features");
  if (features > ROWS8_MAX_FEATURES || ld > 2 * ROWS8_MAX_FEATURES || rows > (1ll << 60) / ld)
    return set_error(ctx, GRILLY_ERR_UNSUPPORTED, std::string(who) + ": more than 2^30 features, a pitch above 2^31, or too many rows");
  if (rows > 0 && (!q || !scale)) return set_error(ctx, GRILLY_ERR_INVALID_ARG, std::string(who) + ": null 8-bit rows");
  if (reinterpret_cast<uintptr_t>(q) & 15) return set_error(ctx, GRILLY_ERR_INVALID_ARG, std::string(who) + ": 8-bit rows must be 16-byte aligned");
  return GRILLY_OK;
}

// An operand's memory. `in_place`: number (from 1) of the output that may be this very memory. `align`: bytes of an element.
struct Rows8Span {
  const void* p;
  long long bytes;
  int in_place = 0;
  int align = 4;
};
// Every tensor starts on a boundary of its own type: the kernels load whole elements. Outputs may overlap neither each other
// nor an input, but for an input that is an output's very memory where that is offered: the kernels read inputs while other
// blocks write.
template <int OUTS, int INS>
int rows8_memory(grilly_ctx* ctx, const char* who, const Rows8Span (&outs)[OUTS], const Rows8Span (&ins)[INS]) {
  auto off = [](const Rows8Span& a) { return reinterpret_cast<uintptr_t>(a.p) % a.align != 0; };
  auto overlap = [](const Rows8Span& a, const Rows8Span& b) {
    const auto x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    return a.p && b.p && x < y + static_cast<uintptr_t>(b.bytes) && y < x + static_cast<uintptr_t>(a.bytes);
  };
  for (const Rows8Span& in : ins)
    if (off(in)) return set_error(ctx, GRILLY_ERR_INVALID_ARG, std::string(who) + ": an operand does not start on a boundary of its type");
  for (int i = 0; i < OUTS; ++i) {
    if (off(outs[i])) return set_error(ctx, GRILLY_ERR_INVALID_ARG, std::string(who) + ": a result does not start on a boundary of its type");
    for (int j = 0; j < i; ++j)
      if (overlap(outs[i], outs[j])) return set_error(ctx, GRILLY_ERR_INVALID_ARG, std::string(who) + ": two results share memory");
    for (const Rows8Span& in : ins)
      if (overlap(outs[i], in) && !(in.in_place == i + 1 && in.p == outs[i].p))
        return set_error(ctx, GRILLY_ERR_INVALID_ARG, std::string(who) + ": a result shares memory with an operand");
  }
  return GRILLY_OK;
}

}  // namespace gb

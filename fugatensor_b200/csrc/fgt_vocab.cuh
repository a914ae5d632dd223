// fgt_vocab.cuh — what the vocabulary operators share: element types, launch
// and argument checks (fgt_embedding.cu, fgt_loss.cu, fgt_logits.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <cstdlib>
#include <string>

#include "fgt.h"
#include "fgt_device.cuh"
#include "fgt_internal.h"

namespace fgt {

fgt_status record_error(fgt_status s, const std::string& m);  // fgt_runtime.cpp

// ------------------------------------------------------- element types ---
// Storage type and its exact f32 value; narrowing rounds to nearest even.
struct F32 {
  using S = float;
  FGT_DEV float get(S v) { return v; }
  FGT_DEV S put(float f) { return f; }
};
struct F16 {
  using S = fgt_u16;
  FGT_DEV float get(S v) { return fgt_f16_to_f32(v); }
  FGT_DEV S put(float f) { return fgt_f32_to_f16(f); }
};
struct BF16 {
  using S = fgt_u16;
  FGT_DEV float get(S v) { return fgt_bf16_to_f32(v); }
  FGT_DEV S put(float f) { return fgt_f32_to_bf16(f); }
};

// An i32 or i64 array of indices or lengths (one branch, the same for a warp).
struct Index {
  const void* p;
  bool wide;
  __device__ __forceinline__ fgt_i64 operator[](fgt_i64 i) const {
    return wide ? static_cast<const fgt_i64*>(p)[i] : (fgt_i64) static_cast<const int*>(p)[i];
  }
};

// ---------------------------------------------------------------- host ---
template <class F> fgt_status guarded_call(const char* name, F&& f) noexcept {
  try {
    f();
    return FGT_OK;
  } catch (const Error& e) {
    return record_error(e.status, std::string(name) + ": " + e.what());
  } catch (const std::exception& e) {
    return record_error(FGT_ERR_INVALID, std::string(name) + ": " + e.what());
  }
}

inline void cuda_check(cudaError_t e, const char* what) {
  if (e != cudaSuccess) fail(FGT_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

inline void check_buffer(const void* p, int64_t elements, const char* what) {
  if (elements == 0) return;
  require(p != nullptr, std::string(what) + " is NULL");
  require((uintptr_t)p % 16 == 0, std::string(what) + " must be 16-byte aligned");
}

inline void check_index_dtype(int dt, const char* what) {
  require(is_int(dt), std::string(what) + " must have dtype i32 or i64");
}

// a * b for sizes in [0, 2^62), refused where it passes 2^62
inline int64_t size_product(int64_t a, int64_t b, const char* what) {
  require(a >= 0 && b >= 0, std::string(what) + " must not be negative");
  require(a == 0 || b <= (INT64_C(1) << 62) / a, std::string(what) + " is too large");
  return a * b;
}

inline int sm_count() {
  static int cached[64] = {};
  int dev = 0;
  cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
  if (dev >= 0 && dev < 64 && cached[dev]) return cached[dev];
  int n = 0;
  cuda_check(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
  if (dev >= 0 && dev < 64) cached[dev] = n;
  return n;
}

// An error left pending on the thread by earlier work is reported as such.
inline void check_pending() {
  const cudaError_t e = cudaPeekAtLastError();
  if (e != cudaSuccess)
    fail(FGT_ERR_CUDA, std::string("an earlier CUDA error is pending on this thread (") + cudaGetErrorString(e) +
                           "); nothing was launched");
}

// Calls f(type tag) for a float dtype.
template <class F> void for_dtype(int dt, F&& f) {
  switch (dt) {
    case FGT_F32: f(F32{}); return;
    case FGT_F16: f(F16{}); return;
    case FGT_BF16: f(BF16{}); return;
  }
  fail(FGT_ERR_INVALID, "dtype must be f32, f16 or bf16");
}

inline unsigned blocks_for(int64_t work, int64_t per_block, const char* what) {
  const int64_t n = (work + per_block - 1) / per_block;
  require(n <= 0x7fffffff, std::string(what) + " is too large for one launch");
  return (unsigned)n;
}

}  // namespace fgt

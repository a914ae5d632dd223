// fgt_vocab.cuh — what the vocabulary operators share: element types, launch
// and argument checks (fgt_embedding.cu, fgt_loss.cu, fgt_logits.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <algorithm>
#include <cstdlib>
#include <map>
#include <mutex>
#include <string>
#include <tuple>

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
  FGT_DEV void split(unsigned w, float& lo, float& hi) {
    lo = fgt_f16_to_f32((fgt_u16)w);
    hi = fgt_f16_to_f32((fgt_u16)(w >> 16));
  }
  FGT_DEV unsigned pair(float lo, float hi) {
    unsigned u;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(hi), "f"(lo));
    return u;
  }
  FGT_DEV S put(float f) { return fgt_f32_to_f16(f); }
};
struct BF16 {
  using S = fgt_u16;
  FGT_DEV float get(S v) { return fgt_bf16_to_f32(v); }
  FGT_DEV void split(unsigned w, float& lo, float& hi) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
  }
  FGT_DEV unsigned pair(float lo, float hi) {
    unsigned u;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(hi), "f"(lo));
    return u;
  }
  FGT_DEV S put(float f) { return fgt_f32_to_bf16(f); }
};

// 16 bytes of storage as f32 values, and back.
template <class T> struct Vec {
  static constexpr int kN = 16 / (int)sizeof(typename T::S);
  static __device__ __forceinline__ void unpack(const uint4& u, float (&v)[kN]) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (sizeof(typename T::S) == 4) {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = __uint_as_float(w[k]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) T::split(w[k], v[2 * k], v[2 * k + 1]);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[kN]) {
    unsigned w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (sizeof(typename T::S) == 4)
        w[k] = __float_as_uint(v[k]);
      else
        w[k] = T::pair(v[2 * k], v[2 * k + 1]);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// Programmatic dependent launch: a kernel waits for its predecessor on the
// stream before it touches memory, and lets its successor be scheduled.
FGT_DEV void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
FGT_DEV void grid_release() { asm volatile("griddepcontrol.launch_dependents;"); }

FGT_DEV unsigned cluster_size() {
  unsigned n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}

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
  if (e == cudaSuccess) return;
  cudaGetLastError();  // this call reports it: it is not left pending on the thread
  fail(FGT_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
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

// FGT_PDL=0: plain stream order (as for the generated kernels); so is a stream that is being captured.
inline bool programmatic(cudaStream_t st) {
  static const bool on = [] {
    const char* e = std::getenv("FGT_PDL");
    return !(e && std::atoi(e) == 0);
  }();
  if (!on) return false;
  cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
  cuda_check(cudaStreamIsCapturing(st, &cs), "cudaStreamIsCapturing");
  return cs == cudaStreamCaptureStatusNone;
}

struct Launch {
  cudaStream_t stream;
  bool pdl;
};

// One launch; cluster > 1 groups that many CTAs. Kernels launched this way call grid_wait() first.
template <class... P, class... A>
void launch(const Launch& l, void (*kernel)(P...), unsigned grid, unsigned threads, size_t smem, unsigned cluster, A&&... args) {
  cudaLaunchAttribute at[2] = {};
  unsigned n = 0;
  if (l.pdl) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = cluster;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = l.stream;
  cfg.attrs = at;
  cfg.numAttrs = n;
  cuda_check(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...), "launch");
}

// How many clusters (CTAs, for a cluster of 1) of the kernel run at once on the
// current device, and leave for its dynamic shared memory (48 KB, static
// included, need none); asked once per kernel, device and launch shape.
template <class K> unsigned active_clusters(K kernel, unsigned threads, size_t smem, unsigned cluster) {
  static std::mutex mu;
  static std::map<std::tuple<const void*, int, size_t, unsigned>, unsigned> known;
  static std::map<std::pair<const void*, int>, size_t> allowed;  // one setting per kernel: it only grows
  int dev = 0;
  cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
  std::lock_guard<std::mutex> lock(mu);
  unsigned& n = known[{(const void*)kernel, dev, smem, cluster}];
  if (!n) {
    size_t& most = allowed[{(const void*)kernel, dev}];
    if (smem > 32 * 1024 && smem > most) {
      cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "cudaFuncSetAttribute");
      most = smem;
    }
    if (cluster > 8) cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "cudaFuncSetAttribute");
    int c = 0;
    if (cluster == 1) {
      cuda_check(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&c, kernel, (int)threads, smem), "cudaOccupancyMaxActiveBlocksPerMultiprocessor");
      c *= sm_count();
    } else {
      cudaLaunchAttribute at = {};
      at.id = cudaLaunchAttributeClusterDimension;
      at.val.clusterDim.x = cluster;
      at.val.clusterDim.y = at.val.clusterDim.z = 1;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(cluster);
      cfg.blockDim = dim3(threads);
      cfg.dynamicSmemBytes = smem;
      cfg.attrs = &at;
      cfg.numAttrs = 1;
      cuda_check(cudaOccupancyMaxActiveClusters(&c, kernel, &cfg), "cudaOccupancyMaxActiveClusters");
    }
    require(c > 0, "a kernel does not fit the device", FGT_ERR_CUDA);
    n = (unsigned)c;
  }
  return n;
}

inline unsigned blocks_for(int64_t work, int64_t per_block, const char* what) {
  const int64_t n = (work + per_block - 1) / per_block;
  require(n <= 0x7fffffff, std::string(what) + " is too large for one launch");
  return (unsigned)n;
}

}  // namespace fgt

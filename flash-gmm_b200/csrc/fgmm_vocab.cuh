// Shared by the vocabulary operators (fgmm_xent.cu, fgmm_embed.cu): element
// types and their conversions, and the argument checks of the entry points.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include <stdio.h>

#include <exception>
#include <string>

#include "../../include/flashgmm.h"
#include "fgmm_internal.cuh"

namespace fgmm {

constexpr int64_t kVocabMaxN = int64_t(1) << 30;
constexpr int32_t kVocabMaxV = 1 << 30;
constexpr int32_t kVocabMaxD = 1 << 16;

inline int type_size(int type) { return type == FGMM_T_F32 ? 4 : 2; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// VEC consecutive elements, moved as one access (VEC * sizeof(T) = 16, or one element).
template <class T, int VEC>
struct __align__(VEC * sizeof(T)) Pack {
  T v[VEC];
  __device__ __forceinline__ void load(const T* p) { *this = *reinterpret_cast<const Pack*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Pack*>(p) = *this; }
};

// Calls f with a null pointer of the element type (a type tag).
template <class F>
decltype(auto) with_type(int type, F&& f) {
  if (type == FGMM_T_BF16) return f(static_cast<__nv_bfloat16*>(nullptr));
  if (type == FGMM_T_F16) return f(static_cast<__half*>(nullptr));
  return f(static_cast<float*>(nullptr));
}

// Programmatic dependent launch: let the next kernel of the stream be set up, and wait
// for the end of the one before (no-ops in a launch without the attribute).
__device__ __forceinline__ void pdl_trigger() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void pdl_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Launches a kernel; `dependent`: it may be set up while the kernel before it (of this
// call, on the same stream) still runs, and waits for its end itself (pdl_wait).
template <class... P, class... A>
cudaError_t launch(void (*kernel)(P...), int64_t grid, int threads, size_t smem,
                   cudaStream_t stream, bool dependent, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = dependent ? 1 : 0;
  count_launches(1);
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// FGMM_OK, or the status of a refused type or shape with its message recorded.
inline int vocab_check_shape(const char* name, int type, int64_t N, int32_t V, int32_t D) {
  char buf[200];
  if (type != FGMM_T_F32 && type != FGMM_T_BF16 && type != FGMM_T_F16) {
    snprintf(buf, sizeof buf, "%s: unknown type %d", name, type);
    return entry_fail(FGMM_ERR_ARG, buf);
  }
  if (N < 0 || V < 1 || D < 1) {
    snprintf(buf, sizeof buf, "%s: invalid shape N=%lld V=%d D=%d", name, (long long)N, V, D);
    return entry_fail(FGMM_ERR_ARG, buf);
  }
  if (N >= kVocabMaxN || V >= kVocabMaxV || D > kVocabMaxD) {
    snprintf(buf, sizeof buf, "%s: N=%lld V=%d D=%d exceeds the supported N < 2^30, V < 2^30, "
             "D <= 65536", name, (long long)N, V, D);
    return entry_fail(FGMM_ERR_UNSUPPORTED, buf);
  }
  return FGMM_OK;
}

// Negative strides and pointers that are not aligned to their elements.
inline int vocab_check_array(const char* name, const char* what, const void* p, int size,
                             int64_t s0, int64_t s1) {
  if (s0 < 0 || s1 < 0)
    return entry_fail(FGMM_ERR_ARG, std::string(name) + ": negative stride of " + what);
  if (reinterpret_cast<uintptr_t>(p) % (unsigned)size)
    return entry_fail(FGMM_ERR_ARG, std::string(name) + ": " + what +
                                        " is not aligned to its elements");
  return FGMM_OK;
}

// Refuses an input (N rows of D elements at these strides) that shares bytes with an
// output of out_bytes: blocks read the input while others write.
inline int vocab_check_overlap(const char* name, const char* what, const void* p, int64_t N,
                               int64_t D, int64_t s0, int64_t s1, int size, const char* out_name,
                               const void* out, int64_t out_bytes) {
  if (N == 0) return FGMM_OK;
  const __int128 a = (__int128)reinterpret_cast<uintptr_t>(p);
  const __int128 b = (__int128)reinterpret_cast<uintptr_t>(out);
  const __int128 a_end = a + ((__int128)(N - 1) * s0 + (__int128)(D - 1) * s1 + 1) * size;
  if (a >= b + out_bytes || b >= a_end) return FGMM_OK;
  return entry_fail(FGMM_ERR_ARG, std::string(name) + ": " + out_name + " overlaps " + what);
}

inline int vocab_check_workspace(const char* name, const void* ws, size_t got, size_t need) {
  if (need > 0 && (ws == nullptr || got < need || (reinterpret_cast<uintptr_t>(ws) & 255))) {
    char buf[200];
    snprintf(buf, sizeof buf, "%s: workspace of %zu bytes (256-byte aligned) required, got %zu at %p",
             name, need, got, ws);
    return entry_fail(FGMM_ERR_WORKSPACE, buf);
  }
  return FGMM_OK;
}

// Runs an entry point's body; no C++ exception crosses the C ABI.
template <class F>
int vocab_entry(const char* name, F&& body) noexcept {
  try {
    entry_fail(FGMM_OK, "");
    return body();
  } catch (const std::exception& e) {
    try {
      return entry_fail(FGMM_ERR_CUDA, std::string(name) + ": " + e.what());
    } catch (...) {
      return FGMM_ERR_CUDA;
    }
  } catch (...) {
    return FGMM_ERR_CUDA;
  }
}

}  // namespace fgmm

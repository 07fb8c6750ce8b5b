// What the host sides of the C ABI share: the error of the last CUDA call, tensor maps, device attributes, launches.
#pragma once

#include <atomic>
#include <mutex>

#include "../../include/b200_trimul.h"
#include "ptx.cuh"

namespace trimul {

inline thread_local int tl_last_cuda_error = 0;

#define TRIMUL_CUDA(expr)                             \
  do {                                                \
    cudaError_t _e = (expr);                          \
    if (_e != cudaSuccess) {                          \
      tl_last_cuda_error = static_cast<int>(_e);      \
      return B200_TRIMUL_E_CUDA;                      \
    }                                                 \
  } while (0)

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn get_encode_fn() {
  static std::once_flag once;
  static EncodeTiledFn fn = nullptr;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qres) == cudaSuccess &&
        qres == cudaDriverEntryPointSuccess) {
      fn = reinterpret_cast<EncodeTiledFn>(p);
    }
  });
  return fn;
}

// bf16 tensor map with 128-byte swizzle. dims[0] is the contiguous dimension; strides (bytes) are for
// dims[1..rank-1].
inline int make_map(CUtensorMap* m, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                    const uint32_t* box) {
  EncodeTiledFn fn = get_encode_fn();
  if (fn == nullptr) {
    tl_last_cuda_error = static_cast<int>(cudaErrorNotSupported);
    return B200_TRIMUL_E_CUDA;
  }
  cuuint64_t d[5];
  cuuint64_t s[4];
  cuuint32_t b[5];
  cuuint32_t e[5];
  for (int i = 0; i < rank; ++i) {
    d[i] = dims[i];
    b[i] = box[i];
    e[i] = 1;
    if (i > 0) s[i - 1] = strides[i - 1];
  }
  CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, static_cast<cuuint32_t>(rank), const_cast<void*>(base), d, s,
                  b, e, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    tl_last_cuda_error = 100000 + static_cast<int>(r);
    return B200_TRIMUL_E_CUDA;
  }
  return B200_TRIMUL_OK;
}

struct DeviceInfo {
  int sms;
  int cc_major;
  int device;
};

constexpr int kMaxDevices = 64;

// SM count and compute capability of the current device; queried once per device and process.
inline int device_info(DeviceInfo* info) {
  static std::atomic<int> cached_sms[kMaxDevices];  // 0 = not queried yet
  static std::atomic<int> cached_cc[kMaxDevices];
  int dev = 0;
  TRIMUL_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return B200_TRIMUL_E_DEVICE;
  info->device = dev;
  int sms = cached_sms[dev].load(std::memory_order_acquire);
  if (sms == 0) {
    int cc = 0;
    TRIMUL_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    TRIMUL_CUDA(cudaDeviceGetAttribute(&cc, cudaDevAttrComputeCapabilityMajor, dev));
    cached_cc[dev].store(cc, std::memory_order_relaxed);
    cached_sms[dev].store(sms, std::memory_order_release);
  }
  info->sms = sms;
  info->cc_major = cached_cc[dev].load(std::memory_order_relaxed);
  if (info->cc_major != 10) return B200_TRIMUL_E_DEVICE;
  return B200_TRIMUL_OK;
}

// Opt a kernel in to its dynamic shared-memory size, once per kernel and device (the attribute belongs to the
// function in a device's context; setting it again is harmless, so a benign race between two threads is fine).
template <typename K>
inline int set_smem(K kernel, int bytes, int device) {
  struct Slot {
    std::atomic<const void*> fn{nullptr};
    std::atomic<unsigned long long> devices{0};
  };
  static Slot slots[64];
  const void* key = reinterpret_cast<const void*>(kernel);
  const unsigned long long bit = 1ull << device;
  for (Slot& s : slots) {
    const void* cur = s.fn.load(std::memory_order_acquire);
    if (cur == nullptr) {
      const void* expected = nullptr;
      if (!s.fn.compare_exchange_strong(expected, key, std::memory_order_acq_rel) && expected != key) continue;
      cur = key;
    }
    if (cur != key) continue;
    if (s.devices.load(std::memory_order_acquire) & bit) return B200_TRIMUL_OK;
    TRIMUL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    s.devices.fetch_or(bit, std::memory_order_release);
    return B200_TRIMUL_OK;
  }
  TRIMUL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));  // table full
  return B200_TRIMUL_OK;
}

// Launch a kernel whose blocks may be placed while the kernel before it on the stream finishes: it sets itself up and keeps the
// rules at grid_dependency_wait on what it touches before that. The kernels of a call are launched this way (but a backward's set-up),
// which takes the set-up (barriers, tensor memory, cluster start) and part of the tail off every boundary: the forward takes 26.6 us
// without and 21.8 us with it at N = 64, 91.9 / 88.7 us at N = 384, 339.3 / 333.7 us at N = 768 (one box, in turn).
template <typename... P, typename... A>
inline cudaError_t launch_overlapped(void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t stream, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }


}  // namespace trimul

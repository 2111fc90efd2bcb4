// Host-side helpers shared by the translation units of the C ABI: launch
// counting, the per-device cache, tensor maps, dependent launches, the pair
// occupancy query and workspace partitioning.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <mutex>
#include <utility>

#include "ethos_b200.h"
#include "kernel_table.h"

namespace ethos {

// Kernels this library has launched in this process (ethos_launch_count).
inline std::atomic<unsigned long long> g_launch_count{0};
inline void count_launch() { g_launch_count.fetch_add(1, std::memory_order_relaxed); }

// ------------------------------------------------------------ device cache --
struct DeviceInfo {
  int sm_count = 0;
  int major = 0;
  bool attrs_set = false;  // capi.cu: its kernels' shared-memory limits are set
};

// Record of the current device; ETHOS_ERR_NO_DEVICE unless it is an sm_100.
inline int base_device_info(DeviceInfo** out) {
  static std::mutex mu;
  static DeviceInfo devs[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return ETHOS_ERR_NO_DEVICE;
  std::lock_guard<std::mutex> lock(mu);
  DeviceInfo& d = devs[dev];
  if (d.sm_count == 0) {
    int sms = 0, major = 0;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return ETHOS_ERR_CUDA;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess) return ETHOS_ERR_CUDA;
    d.sm_count = sms;
    d.major = major;
  }
  if (d.major != 10) return ETHOS_ERR_NO_DEVICE;
  // cuTensorMapEncodeTiled needs a current context, and a thread that has made
  // no runtime call that binds one (an autograd worker whose allocations all
  // came from the cache) has none
  static thread_local int bound = -1;
  if (bound != dev) {
    if (cudaSetDevice(dev) != cudaSuccess) return ETHOS_ERR_CUDA;
    bound = dev;
  }
  *out = &d;
  return ETHOS_OK;
}

// Sets the dynamic shared-memory limit of a kernel once per device.
inline int smem_attr_once(const void* fn, int bytes) {
  int dev = 0, set = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return ETHOS_ERR_NO_DEVICE;
  static KernelTable<int> table;
  return table.get(dev, fn, &set, [&](int* v) {
    *v = bytes;
    return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
  }) ? ETHOS_OK : ETHOS_ERR_CUDA;
}

// ------------------------------------------------------------- tensor maps --
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = []() -> EncodeTiledFn {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

// Row-major bf16 matrix [rows, cols] (row pitch ld >= cols elements) read in
// boxes of 64 columns x box_rows rows with the 128-byte swizzle that the UMMA
// descriptors expect.
// box_cols 64, 32 or 16 (rows of 128, 64 or 32 bytes, with the swizzle of
// that width); the UMMA descriptor of the consuming kernel must match it.
inline int make_tmap_bf16(CUtensorMap* m, const void* ptr, int64_t rows, int64_t cols, int box_rows, int64_t ld = 0,
                   int box_cols = 64, CUtensorMapDataType dtype = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return ETHOS_ERR_TENSOR_MAP;
  if (ld == 0) ld = cols;
  if ((reinterpret_cast<uintptr_t>(ptr) & 15u) != 0 || (ld * 2) % 16 != 0) return ETHOS_ERR_ALIGNMENT;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld * 2)};
  if (box_cols != 64 && box_cols != 32 && box_cols != 16) return ETHOS_ERR_TENSOR_MAP;
  cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1u, 1u};
  CUresult r = fn(m, dtype, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE,
                  box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B
                                 : (box_cols == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B),
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? ETHOS_OK : ETHOS_ERR_TENSOR_MAP;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline int launch_status() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? ETHOS_OK : ETHOS_ERR_CUDA;
}

// Launch with programmatic stream serialization: the kernel may start while
// the previous kernel of the stream finishes (its set-up overlaps that tail)
// and waits in pdl_wait() for it before touching global memory.  Only kernels
// that call pdl_wait() before their first global access are launched so.
template <class... KArgs, class... Args>
int launch_pdl(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  if (cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...) != cudaSuccess) return ETHOS_ERR_CUDA;
  return launch_status();
}

// Clusters of two that can run at once for a 2-SM GEMM kernel (queried once
// per kernel and device: the SM-pair topology decides it, not the tile count).
inline int max_pair_clusters(const void* fn, int threads, int smem, const DeviceInfo& dev) {
  int d = 0, pairs = 0;
  if (cudaGetDevice(&d) != cudaSuccess) return 0;
  static KernelTable<int> table;
  table.get(d, fn, &pairs, [&](int* n) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(dev.sm_count & ~1));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(n, fn, &cfg) == cudaSuccess) return true;
    cudaGetLastError();
    *n = 0;
    return false;
  });
  return pairs;
}

// ------------------------------------------------------- workspace layout --
struct Carve {
  char* base;
  size_t off = 0;
  size_t cap;
  template <class T>
  T* take(size_t count) {
    off = (off + 255) & ~static_cast<size_t>(255);
    T* p = base ? reinterpret_cast<T*>(base + off) : nullptr;
    off += count * sizeof(T);
    return p;
  }
};

// Wait limit of the kernels in training.cu (each translation unit has its own
// device variable; ethos_set_wait_limit_ns sets both).
int training_set_wait_limit(unsigned long long limit_ns);

}  // namespace ethos

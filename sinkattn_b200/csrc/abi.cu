// abi.cu — host-side plumbing of the C ABI: thread-local error messages,
// the driver's cuTensorMapEncodeTiled resolved through the runtime (so the
// library needs no -lcuda), and cached per-device SM counts.

#include <stdarg.h>
#include <stdio.h>

#include <mutex>
#include <set>
#include <tuple>

#include "sa_common.cuh"

namespace sa {

namespace {
thread_local char g_err[512] = "";
std::mutex g_mu;
EncodeTiledFn g_encode = nullptr;
int g_sm_count[64] = {};
// (device, kernel, attribute, value) already applied by func_attr_once
std::set<std::tuple<int, const void*, int, int>> g_attrs;
}  // namespace

void set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
}

int cuda_fail(cudaError_t e, const char* what) {
  set_error("%s failed: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
  return SA_ECUDA;
}

EncodeTiledFn encode_tiled_fn() {
  std::lock_guard<std::mutex> lock(g_mu);
  if (g_encode != nullptr) return g_encode;
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult q;
  cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
  if (e != cudaSuccess || fn == nullptr || q != cudaDriverEntryPointSuccess) {
    set_error("cannot resolve cuTensorMapEncodeTiled (%s)",
              e != cudaSuccess ? cudaGetErrorString(e) : "symbol not found");
    return nullptr;
  }
  g_encode = reinterpret_cast<EncodeTiledFn>(fn);
  return g_encode;
}

int sm_count_current_device() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev >= 0 && dev < 64) {
    std::lock_guard<std::mutex> lock(g_mu);
    if (g_sm_count[dev] > 0) return g_sm_count[dev];
  }
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
    n = 148;
  if (dev >= 0 && dev < 64) {
    std::lock_guard<std::mutex> lock(g_mu);
    g_sm_count[dev] = n;
  }
  return n;
}

int func_attr_once(const void* func, cudaFuncAttribute attr, int value) {
  int dev = 0;
  SA_CUDA_TRY(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lock(g_mu);
  const auto key = std::make_tuple(dev, func, (int)attr, value);
  if (g_attrs.count(key) != 0) return SA_OK;
  SA_CUDA_TRY(cudaFuncSetAttribute(func, attr, value));
  g_attrs.insert(key);
  return SA_OK;
}

int tile_map_bhsd(CUtensorMap* map, const void* base, const int64_t st[4], int B, int H, int S,
                  int D) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (enc == nullptr) return SA_ECUDA;
  // dims innermost first: (D, S, H, B); strides in bytes for dims 1..3.
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)S, (cuuint64_t)H, (cuuint64_t)B};
  cuuint64_t strides[3] = {(cuuint64_t)st[2] * 2, (cuuint64_t)st[1] * 2, (cuuint64_t)st[0] * 2};
  cuuint32_t box[4] = {64, 128, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const auto encode = [&] {
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides,
               box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  if (r == CUDA_ERROR_INVALID_CONTEXT) {
    // a thread whose first CUDA call this is (an autograd worker): setting the
    // device that is current already binds its context to the thread
    int dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) r = encode();
  }
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (CUresult %d)", (int)r);
    return SA_ECUDA;
  }
  return SA_OK;
}

bool strides16_ok(const int64_t st[4]) {
  if (st[3] != 1) return false;
  for (int i = 0; i < 3; ++i)
    if (st[i] < 0 || (st[i] % 8) != 0) return false;
  return true;
}

}  // namespace sa

extern "C" const char* sa_last_error(void) { return sa::g_err; }

extern "C" int sa_version(void) { return 1; }

extern "C" int sa_device_sm_count(void) { return sa::sm_count_current_device(); }

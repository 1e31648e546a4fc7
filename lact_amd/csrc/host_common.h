// What the library's host code shares: the error message of a thread, the optional timing of launches, launch and argument checks.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>
#include <initializer_list>
#include <string>
#include <vector>

namespace lact {

inline thread_local std::string g_err;
inline int fail(const std::string& m) {
  g_err = m;
  return -1;
}

inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

inline int check_ptrs(std::initializer_list<const void*> ps, const char* what) {
  for (const void* p : ps)
    if (!p) return fail(std::string("null pointer: ") + what);
  return 0;
}

// ---- optional per-launch timing (HIP events on the caller's stream) ---------------------------------
struct ProfRec {
  const char* kernel;
  const char* site;
  double flops;
  hipStream_t stream;
  hipEvent_t e0, e1;
};
struct Profiler {
  bool on = false;
  std::vector<ProfRec> recs;
  std::vector<hipEvent_t> pool;
  hipEvent_t get() {
    if (!pool.empty()) {
      hipEvent_t e = pool.back();
      pool.pop_back();
      return e;
    }
    hipEvent_t e;
    (void)hipEventCreate(&e);
    return e;
  }
  void clear() {
    for (auto& r : recs) {
      pool.push_back(r.e0);
      pool.push_back(r.e1);
    }
    recs.clear();
  }
};
inline Profiler g_prof;
struct ProfScope {
  hipStream_t s;
  hipEvent_t e1 = nullptr;
  ProfScope(const char* kernel, const char* site, double flops, hipStream_t st) : s(st) {
    if (!g_prof.on) return;
    ProfRec r{kernel, site, flops, st, g_prof.get(), g_prof.get()};
    (void)hipEventRecord(r.e0, s);
    e1 = r.e1;
    g_prof.recs.push_back(r);
  }
  ~ProfScope() {
    if (e1) (void)hipEventRecord(e1, s);
  }
};
// kern may contain template commas: pass it parenthesised
#define LACT_LAUNCH(kname, site, flops, kern, grid, block, stream, ...)  \
  do {                                                                  \
    ProfScope ps_(kname, site, flops, stream);                          \
    hipLaunchKernelGGL(kern, grid, block, 0, stream, __VA_ARGS__);      \
  } while (0)

#define LACT_LAUNCH_SMEM(kname, site, flops, kern, grid, block, smem_bytes, stream, ...) \
  do {                                                                                   \
    ProfScope ps_(kname, site, flops, stream);                                           \
    hipLaunchKernelGGL(kern, grid, block, smem_bytes, stream, __VA_ARGS__);              \
  } while (0)

// Kernels whose ring exceeds the default dynamic LDS limit opt in once per call site (= instantiation) and device:
// the attribute belongs to the current device.
inline void allow_big_lds(std::atomic<uint64_t>& done, const void* kern, int bytes) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
  const uint64_t bit = 1ull << dev;
  if (done.load(std::memory_order_acquire) & bit) return;
  (void)hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  done.fetch_or(bit, std::memory_order_release);
}
#define LACT_BIG_LDS(kern, bytes)                                         \
  do {                                                                    \
    static std::atomic<uint64_t> done_{0};                                \
    allow_big_lds(done_, reinterpret_cast<const void*>(kern), bytes);     \
  } while (0)

template <typename T> const char* tname();
template <> inline const char* tname<uint16_t>() { return "bf16"; }
template <> inline const char* tname<float>() { return "f32"; }

#define LACT_CHECK_LAUNCH()                                                     \
  do {                                                                          \
    hipError_t e_ = hipGetLastError();                                          \
    if (e_ != hipSuccess) return fail(std::string("kernel launch failed: ") + hipGetErrorString(e_)); \
  } while (0)

}  // namespace lact

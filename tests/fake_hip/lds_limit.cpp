// Goes before the fake runtime: launches with more LDS than hipFuncSetAttribute last allowed
// the kernel (64 KB without it; 160 KB at most) are refused and counted.
#include <cstddef>
#include <cstdint>
#include <map>

namespace {
struct Dim3 {
  uint32_t x, y, z;
};
constexpr int kMaxDynamicSharedMemorySize = 8;  // hipFuncAttributeMaxDynamicSharedMemorySize
std::map<const void*, size_t> g_limit;
int g_last = 0, g_refused = 0, g_launches = 0;
size_t g_most = 0;
}  // namespace

extern "C" {
int hipFuncSetAttribute(const void* fn, int attribute, int value) {
  if (attribute != kMaxDynamicSharedMemorySize || value < 0 || value > 160 * 1024) return 1;
  g_limit[fn] = (size_t)value;
  return 0;
}
int hipLaunchKernel(const void* fn, Dim3, Dim3, void**, size_t lds, void*) {
  auto it = g_limit.find(fn);
  g_launches++;
  if (lds > g_most) g_most = lds;
  if (lds <= (it == g_limit.end() ? 64 * 1024 : it->second)) return 0;
  g_refused++;
  return g_last = 1;
}
int hipGetLastError() {
  const int e = g_last;
  g_last = 0;
  return e;
}
int lds_refused() { return g_refused; }
int lds_launches() { return g_launches; }
size_t lds_most() { return g_most; }
}

// The part of the health word (fs_device_error) that the products of routed experts and the orthogonal updates share. The kernels get its address with
// their arguments: a word of each source's own would be a copy of 12 us more wherever a solver reads the word. A source by itself, since
// looking for the address loads the module that the word is in, and one with kernels takes 10 ms for that.
#include <cuda_runtime.h>

#include <atomic>

namespace fs {
namespace ex {
namespace {

__device__ int g_products_error = 0;  // non-zero once a bounded wait gave up
std::atomic<bool> g_launched{false};  // whether this process has launched such a kernel: if not, the word is not looked at

}  // namespace

// The word on the current device, for a kernel that is about to be launched; null after an error of the runtime's.
int* products_health() {
  static std::atomic<int*> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return nullptr;
  int* at = dev < 64 ? known[dev].load(std::memory_order_relaxed) : nullptr;
  if (!at) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_products_error) != cudaSuccess) return nullptr;
    at = static_cast<int*>(p);
    if (dev < 64) known[dev].store(at, std::memory_order_relaxed);
  }
  g_launched.store(true, std::memory_order_relaxed);
  return at;
}

// Solvers read the health word where the host waits anyway: not this part of it in programs without products.
int products_error_flag() {
  if (!g_launched.load(std::memory_order_relaxed)) return 0;
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_products_error, sizeof(int)) != cudaSuccess) return -1;
  return v ? 1 : 0;
}
int clear_products_error_flag() {
  if (!g_launched.load(std::memory_order_relaxed)) return 0;
  const int zero = 0;
  return cudaMemcpyToSymbol(g_products_error, &zero, sizeof(int)) == cudaSuccess ? 0 : -1;
}

}  // namespace ex
}  // namespace fs

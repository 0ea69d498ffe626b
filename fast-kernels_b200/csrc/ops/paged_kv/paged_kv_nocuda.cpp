// The op surface of a build WITHOUT CUDA: same names, every call throws
// std::runtime_error("fast-kernels was built without CUDA support") -- there is no CPU path.
#include <stdexcept>

#include "ops/paged_kv/paged_kv.h"

namespace fast_kernels::paged_kv {
namespace {
[[noreturn]] void unavailable() { throw std::runtime_error("fast-kernels was built without CUDA support"); }
}  // namespace

using ptr = std::uintptr_t;
using stride = std::int64_t;

void paged_kv_append_forward(ptr, ptr, stride, stride, stride, stride, ptr, ptr, ptr, ptr, ptr, int, int, int, int, int,
                             int, int, int, float, ptr) {
  unavailable();
}

void paged_attention_forward(ptr, stride, stride, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, int, int, int, int, int,
                             int, int, int, int, int, int, float, float, ptr) {
  unavailable();
}
void shared_prefix_decode_forward(ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr, ptr,
                                  int, int, int, int, int, int, int, int, int, int, int, int, float, float, ptr) {
  unavailable();
}
int paged_kv_device_status() { unavailable(); }

}  // namespace fast_kernels::paged_kv

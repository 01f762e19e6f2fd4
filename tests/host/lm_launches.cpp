// Prints the kernels that calls of the language-model C ABI launch, on the host:
// the library's sources are compiled for the host only, and the HIP calls that a
// launch makes are answered here, so nothing runs and the addresses are never
// read. Without arguments it reads lines
//   masked <f16|f32> batch heads kv-heads sequence head-dim causal window capped biased
//   paged <f16|f32> batch heads kv-heads head-dim page-size max-pages pages
//   rope <f16|f32> tokens heads kv-heads head-dim rotary-dim interleaved offset
// and answers each with "status" and, for each launch, the kernel's mangled name.
// With an argument it prints the name of every kernel that was registered.

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstdio>
#include <cstring>
#include <map>
#include <string>

#include "operatorlib/lm_c.h"

namespace {

// Host-side handle of a kernel -> its device name, as registered at start-up.
std::map<const void*, std::string>& kernels() {
  static std::map<const void*, std::string> names;
  return names;
}

std::string launched;

hipError_t record(const void* kernel) {
  launched += " " + kernels()[kernel];
  return hipSuccess;
}

}  // namespace

extern "C" {
char __hip_fatbin;
void** __hipRegisterFatBinary(const void*) {
  static void* handle;
  return &handle;
}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*,
                           void*, void*, void*, int*) {
  kernels()[host] = name;
}
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}
void __hipUnregisterFatBinary(void**) {}
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* shared, hipStream_t* stream) {
  *grid = *block = dim3(1);
  *shared = 0;
  *stream = nullptr;
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void* kernel, dim3, dim3, void**, size_t, hipStream_t) {
  return record(kernel);
}
hipError_t hipGetLastError() { return hipSuccess; }
}

int main(int argc, char**) {
  if (argc > 1) {
    for (const auto& k : kernels()) std::printf("%s\n", k.second.c_str());
    return 0;
  }
  // aligned addresses, far apart
  auto f32 = [](int i, int offset = 0) {
    return reinterpret_cast<float*>(std::uintptr_t(i) << 40) + offset;
  };
  auto f16 = [](int i, int offset = 0) {
    return reinterpret_cast<operatorlib_half_t*>(std::uintptr_t(i) << 40) + offset;
  };
  auto i32 = [](int i) { return reinterpret_cast<int32_t*>(std::uintptr_t(i) << 40); };
  char op[16], type[8];
  while (std::scanf("%15s %7s", op, type) == 2) {
    const bool half = type[1] == '1';
    launched.clear();
    int status = -1;
    if (std::strcmp(op, "masked") == 0) {
      int b, h, hk, s, d, causal, window, capped, biased;
      if (std::scanf("%d %d %d %d %d %d %d %d %d", &b, &h, &hk, &s, &d, &causal, &window, &capped,
                     &biased) != 9)
        return 1;
      const operatorlib_strides_t q = {int64_t(h) * s * d, int64_t(s) * d, d};
      const operatorlib_strides_t k = {int64_t(hk) * s * d, int64_t(s) * d, d};
      const float* slopes = biased ? f32(5) : nullptr;
      const float cap = capped == 2 ? 1e6f : capped ? 30.0f : 0.0f;
      status = half ? operatorlib_masked_attention_f16(f16(1), q, f16(2), k, f16(3), k, slopes,
                                                       nullptr, nullptr, f16(4), q, b, h, hk, s, d,
                                                       0.1f, causal, window, cap, nullptr)
                    : operatorlib_masked_attention_f32(f32(1), q, f32(2), k, f32(3), k, slopes,
                                                       nullptr, nullptr, f32(4), q, b, h, hk, s, d,
                                                       0.1f, causal, window, cap, nullptr);
    } else if (std::strcmp(op, "paged") == 0) {
      int b, h, hk, d, page, width, pages;
      float cap;
      if (std::scanf("%d %d %d %d %d %d %d %f", &b, &h, &hk, &d, &page, &width, &pages, &cap) != 8)
        return 1;
      const size_t ws = size_t(1) << 40;
      status = half ? operatorlib_paged_attention_f16_ws(f16(1), int64_t(h) * d, f16(2), f16(3),
                                                         i32(6), width, i32(7), nullptr, f16(4), b,
                                                         h, hk, d, pages, page, width, 0.1f, 0,
                                                         cap, f32(9), ws, nullptr)
                    : operatorlib_paged_attention_f32_ws(f32(1), int64_t(h) * d, f32(2), f32(3),
                                                         i32(6), width, i32(7), nullptr, f32(4), b,
                                                         h, hk, d, pages, page, width, 0.1f, 0,
                                                         cap, f32(9), ws, nullptr);
    } else {
      int t, h, hk, d, rotary, interleaved, offset;
      if (std::scanf("%d %d %d %d %d %d %d", &t, &h, &hk, &d, &rotary, &interleaved, &offset) != 7)
        return 1;
      const int64_t qs = int64_t(h) * d, ks = int64_t(hk) * d;
      status = half ? operatorlib_rope_append_f16(f16(1, offset), qs, f16(2), ks, f16(3), ks,
                                                  i32(6), 1, nullptr, f32(8), i32(7), f16(4),
                                                  nullptr, f16(10), f16(11), t, h, hk, d, rotary,
                                                  interleaved, t + 1, 16, nullptr)
                    : operatorlib_rope_append_f32(f32(1, offset), qs, f32(2), ks, f32(3), ks,
                                                  i32(6), 1, nullptr, f32(8), i32(7), f32(4),
                                                  nullptr, f32(10), f32(11), t, h, hk, d, rotary,
                                                  interleaved, t + 1, 16, nullptr);
    }
    std::printf("%d%s\n", status, launched.c_str());
  }
  return 0;
}

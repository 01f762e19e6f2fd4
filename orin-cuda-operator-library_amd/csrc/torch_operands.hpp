#pragma once
// What the torch bindings share: checks of tensors, sizes as the C ABI takes
// them, scratch from torch's allocator, and the launch of one C ABI call.

#include <ATen/ATen.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include <cstddef>
#include <cstdint>
#include <initializer_list>
#include <limits>
#include <utility>
#include <vector>

#include "operatorlib/operatorlib_c.h"

namespace {

enum DTypes { kFloat32Only, kFloat32OrFloat16 };

inline const char* dtype_set_text(DTypes set) {
  return set == kFloat32Only ? "float32" : "float32 or float16";
}

class Operands {
 public:
  // `named` lists (tensor, argument name); the first tensor sets the device
  // and dtype the others must share. `dense`: every tensor must be dense
  // row-major; else the operator states its own stride rules.
  Operands(const char* op, DTypes allowed,
           std::initializer_list<std::pair<const at::Tensor*, const char*>> named,
           bool dense = true)
      : op_(op), list_(named) {
    const at::Tensor& lead = *list_.front().first;
    for (const auto& [t, name] : list_) {
      TORCH_CHECK(t->is_cuda(), op_, ": ", name,
                  " must live in HIP device memory (a CUDA-key tensor), got ",
                  t->device());
      TORCH_CHECK(!dense || t->is_contiguous(), op_, ": ", name,
                  " must be contiguous (dense row-major)");
      TORCH_CHECK(t->device() == lead.device(), op_, ": ", name, " is on ",
                  t->device(), " but ", list_.front().second, " is on ", lead.device());
      TORCH_CHECK(t->scalar_type() == lead.scalar_type(), op_, ": ", name,
                  " has dtype ", t->scalar_type(), " but ", list_.front().second,
                  " has dtype ", lead.scalar_type());
    }
    const at::ScalarType dt = lead.scalar_type();
    const bool ok = dt == at::kFloat || (allowed == kFloat32OrFloat16 && dt == at::kHalf);
    TORCH_CHECK(ok, op_, ": inputs must be ", dtype_set_text(allowed), ", got ", dt);
    half_ = dt == at::kHalf;
  }

  bool half() const { return half_; }
  const at::Tensor& lead() const { return *list_.front().first; }
  const char* op() const { return op_; }

 private:
  const char* op_;
  std::vector<std::pair<const at::Tensor*, const char*>> list_;
  bool half_ = false;
};

// A size the C ABI takes as int: positive and within int32.
inline int extent(const char* op, const char* what, std::int64_t value) {
  TORCH_CHECK(value > 0 && value <= std::numeric_limits<int>::max(), op, ": ",
              what, " = ", value, " is not a positive int32");
  return static_cast<int>(value);
}

inline void require_rank(const Operands& in, const at::Tensor& t, const char* name,
                         std::int64_t rank, const char* layout) {
  TORCH_CHECK(t.dim() == rank, in.op(), ": ", name, " must be ", layout, ", got ",
              t.dim(), " dimension(s)");
}

// Rows of a tensor read as [rows, size(-1)].
inline std::pair<int, int> rows_by_last(const Operands& in, const at::Tensor& t,
                                        const char* last_name) {
  TORCH_CHECK(t.dim() >= 1, in.op(), ": ", "input must have at least one dimension");
  const int last = extent(in.op(), last_name, t.size(-1));
  const int rows = extent(in.op(), "row count (numel / size(-1))", t.numel() / t.size(-1));
  return {rows, last};
}

inline const void* caddr(const at::Tensor& t) { return t.data_ptr(); }

// Scratch for a *_ws entry point: `bytes` from torch's caching allocator on
// the inputs' device, handed back to it when the operator returns. The
// allocator is stream-ordered (the block is reused only by later work on
// the current stream, which is where the call's kernels run) and
// capture-aware (under graph capture it comes from the graph's pool), so
// the library itself holds no memory for these calls.
struct Workspace {
  at::Tensor tensor;
  Workspace(const Operands& in, std::size_t bytes) {
    if (bytes > 0)
      tensor = at::empty({static_cast<std::int64_t>(bytes)},
                         in.lead().options().dtype(at::kByte));
  }
  void* data() const { return tensor.defined() ? tensor.data_ptr() : nullptr; }
  std::size_t bytes() const { return tensor.defined() ? tensor.numel() : 0; }
};

// Checks a tensor of another type that goes with the operands: on their
// device, of dtype `dt`, dense row-major.
inline void require_aux(const Operands& in, const at::Tensor& t, const char* name,
                        at::ScalarType dt) {
  TORCH_CHECK(t.device() == in.lead().device(), in.op(), ": ", name, " is on ", t.device(),
              " but the inputs are on ", in.lead().device());
  TORCH_CHECK(t.scalar_type() == dt, in.op(), ": ", name, " must be ", dt, ", got ",
              t.scalar_type());
  TORCH_CHECK(t.is_contiguous(), in.op(), ": ", name, " must be contiguous (dense row-major)");
}

// Runs `call(stream)` (one C ABI entry point) with the inputs' device
// current, on that device's current stream.
template <typename Call>
void launch(const Operands& in, Call&& call) {
  const c10::DeviceGuard guard(in.lead().device());
  void* stream = at::hip::getCurrentHIPStreamMasqueradingAsCUDA(
                     in.lead().get_device()).stream();
  const int status = call(stream);
  TORCH_CHECK(status == 0, in.op(), " launch failed: ",
              operatorlib_status_string(status));
}

}  // namespace

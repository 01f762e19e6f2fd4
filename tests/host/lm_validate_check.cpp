// Argument predicates of the language-model entry points
// (csrc/lm_validate.hpp) at boundary values, built with AddressSanitizer and
// UndefinedBehaviorSanitizer. Prints "failures=N"; exit status 0 only when
// every expectation holds.

#include <climits>
#include <cstdint>
#include <cstdio>
#include <initializer_list>
#include <limits>

#include "lm_validate.hpp"

namespace {

int failures = 0;

void expect(bool got, bool want, const char* what) {
  if (got != want) {
    std::printf("FAIL %s: got %d want %d\n", what, got, want);
    ++failures;
  }
}

}  // namespace

int main() {
  const std::int64_t far = std::numeric_limits<std::int64_t>::max();
  opl::RopeShape r = {512, 256, 256, 1, 3, 4, 2, 128, 128, 5, 16};
  expect(opl::rope_shape_ok(r), true, "rope");
  for (int big : {INT_MAX, 1 << 30, 1 << 16}) {
    opl::RopeShape x = r;
    x.q_heads = x.kv_heads = x.head_dim = big;
    x.q_stride = x.k_stride = x.v_stride = far;
    expect(opl::rope_shape_ok(x), false, "rope: a token past 32 bits");
    x = r;
    x.pages = x.page_size = big;
    expect(opl::rope_shape_ok(x), false, "rope: slots past 32 bits");
  }
  r.pages = INT_MAX / 16;
  expect(opl::rope_shape_ok(r), true, "rope: the most slots");
  r.pages += 1;
  expect(opl::rope_shape_ok(r), false, "rope: one more page");
  r = {512, 256, 256, 0, 3, 4, 2, 128, 0, 5, 16};
  expect(opl::rope_shape_ok(r), true, "rope: nothing rotates, no positions");

  opl::PagedShape p = {3, 4, 2, 128, 16, 9};
  expect(opl::paged_shape_ok(p, 2), true, "paged");
  p.head_dim = 4;
  expect(opl::paged_shape_ok(p, 4), true, "paged: fp32 head_dim 4");
  expect(opl::paged_shape_ok(p, 2), false, "paged: fp16 head_dim 4");
  p = {INT_MAX, INT_MAX, INT_MAX, 128, INT_MAX, INT_MAX};
  expect(opl::paged_shape_ok(p, 2), false, "paged: everything large");
  const int most_tokens = INT_MAX - 1024;
  p = {1, 1, 1, 128, most_tokens, 1};
  expect(opl::paged_shape_ok(p, 2), true, "paged: the largest page");
  p = {1, 1, 1, 128, most_tokens + 1, 1};
  expect(opl::paged_shape_ok(p, 2), false, "paged: one token more");
  p = {65, 1, 1, 128, most_tokens, 1};
  expect(opl::paged_shape_ok(p, 2), false, "paged: past 2^31 units");
  p = {64, 1, 1, 128, most_tokens, 1};
  expect(opl::paged_shape_ok(p, 2), true, "paged: just below 2^31 units");
  p = {33, 66, 2, 128, most_tokens, 1};
  expect(opl::paged_shape_ok(p, 2), false, "paged: two tiles of heads count");
  expect(opl::paged_cache_ok(INT_MAX, 2, 1), true, "cache: 2^32 - 2 rows");
  expect(opl::paged_cache_ok(INT_MAX, 3, 1), false, "cache: past 2^32 rows");
  expect(opl::paged_cache_ok(INT_MAX, INT_MAX, INT_MAX), false, "cache: everything large");

  const float inf = std::numeric_limits<float>::infinity();
  expect(opl::score_rules_ok(1.0f, 0, 0.0f), true, "rules");
  expect(opl::score_rules_ok(inf, 0, 0.0f), false, "rules: scale");
  expect(opl::score_rules_ok(1.0f, 0, -inf), false, "rules: softcap");
  expect(opl::score_rules_ok(1.0f, -1, 0.0f), false, "rules: window");
  expect(opl::score_rules_ok(0x1p-100f, 0, 0.0f), true, "rules: the least scale");
  expect(opl::score_rules_ok(0x1p-101f, 0, 0.0f), false, "rules: below the least scale");
  expect(opl::score_rules_ok(0x1p50f, 0, 0x1p-50f), true, "rules: the largest scale / softcap");
  expect(opl::score_rules_ok(0x1p50f, 0, 0x1p-51f), false, "rules: past the largest scale / softcap");
  expect(opl::score_rules_ok(0x1p-50f, 0, 0x1p51f), false, "rules: below the least scale / softcap");

  opl::MaskedShape m = {2, 4, 2, 80, 64};
  expect(opl::masked_shape_ok(m, 2), true, "masked");
  m = {INT_MAX, INT_MAX, INT_MAX, 1 << 20, 128};
  expect(opl::masked_shape_ok(m, 2), false, "masked: everything large");
  m = {1, 511, 511, 1 << 20, 128};
  expect(opl::masked_shape_ok(m, 2), true, "masked: just below 2^24 blocks");
  m = {1, 512, 512, 1 << 20, 128};
  expect(opl::masked_shape_ok(m, 2), false, "masked: 2^24 blocks");
  m = {1, 1, 1, 1 << 20, 64};
  alignas(16) static char memory[32];
  const opl::MaskedStrides at = {0, 0, 1016}, past = {0, 0, 1024}, most = {far & ~7, far & ~7, far & ~7};
  expect(opl::masked_strides_ok(memory, at, m, 2), true, "strides: just below 2^31 bytes");
  expect(opl::masked_strides_ok(memory, past, m, 2), false, "strides: 2^31 bytes");
  expect(opl::masked_strides_ok(memory, most, m, 2), false, "strides: the largest");
  expect(opl::masked_strides_ok(memory + 8, at, m, 2), false, "strides: base off 16 bytes");
  std::printf("failures=%d\n", failures);
  return failures == 0 ? 0 : 1;
}

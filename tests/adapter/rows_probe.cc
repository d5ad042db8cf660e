// Whether rows lie over each other, as the operators' entry points see it (operators_check.cc), against the bytes themselves: all small
// layouts of two sets of rows. Prints what is wrong and exits 1.
#include <cstdio>
#include <set>

#include "operators.h"

static int wrong = 0;
constexpr uint32_t kDim = 2;
static const uintptr_t kBase = 1u << 20;

static b2_rows Make(int64_t at, int64_t row, int64_t head) { return b2_rows{reinterpret_cast<void *>(kBase + 2 * at), row, head}; }
static std::set<int64_t> Elements(int64_t at, int64_t row, int64_t head, uint32_t n, uint32_t heads, bool *itself) {
  std::set<int64_t> s;
  *itself = false;
  for (uint32_t r = 0; r < n; ++r)
    for (uint32_t h = 0; h < heads; ++h)
      for (uint32_t d = 0; d < kDim; ++d)
        if (!s.insert(at + static_cast<int64_t>(r) * row + static_cast<int64_t>(h) * head + d).second) *itself = true;
  return s;
}

int main() {
  bool itself, ignored;
  for (uint32_t n = 1; n <= 4; ++n)
    for (uint32_t hy = 1; hy <= 3; ++hy)
      for (int64_t row = -9; row <= 9; ++row)
        for (int64_t head = -9; head <= 9; ++head) {
          const std::set<int64_t> y = Elements(0, row, head, n, hy, &itself);
          const b2_rows ry = Make(0, row, head);
          if (b2::CheckResult("y", &ry, n, hy, kDim, B2_BF16).empty() == itself) {
            std::printf("itself: %u rows, %u heads, strides %lld %lld\n", n, hy, (long long)row, (long long)head);
            ++wrong;
          }
          for (uint32_t hx = 1; hx <= 3; ++hx)
            for (int64_t at = -14; at <= 14; ++at) {
              const std::set<int64_t> x = Elements(at, row, head, n, hx, &ignored);
              bool meet = false;
              for (int64_t e : x) meet = meet || y.count(e);
              const b2_rows rx = Make(at, row, head);
              if (b2::CheckApart("y", &ry, hy, "x", &rx, hx, n, kDim, B2_BF16, false).empty() == meet) {
                std::printf("apart: %u rows, %u and %u heads, strides %lld %lld, %lld on\n", n, hy, hx, (long long)row, (long long)head, (long long)at);
                ++wrong;
              }
              if (at == 0 && hx == hy && !b2::CheckApart("y", &ry, hy, "x", &rx, hx, n, kDim, B2_BF16, true).empty()) ++wrong;      // the very same place
            }
        }
  // other strides: what is apart in memory is fine, what is not is refused
  const b2_rows a = Make(0, 8, 4), b = Make(60, 6, 2), c = Make(20, 6, 2), far = Make(0, int64_t(1) << 40, 2);
  if (!b2::CheckApart("y", &a, 2, "x", &b, 3, 7, kDim, B2_BF16, false).empty()) ++wrong;
  if (b2::CheckApart("y", &a, 2, "x", &c, 3, 7, kDim, B2_BF16, true).empty()) ++wrong;
  if (!b2::CheckResult("y", &far, 0x7fffffffu, 2, kDim, B2_BF16).empty()) ++wrong;
  if (!b2::CheckApart("y", &a, 2, "x", &far, 0, 7, kDim, B2_BF16, false).empty() || !b2::CheckResult("y", nullptr, 0, 2, kDim, B2_BF16).empty()) ++wrong;
  return wrong ? 1 : 0;
}

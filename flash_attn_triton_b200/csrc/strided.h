// Whether strided arrays share memory: for calls that write several of them at once (no CUDA).
#pragma once
#include <algorithm>
#include <cstdint>

namespace fa {

// Runs of `width` bytes at base + sum of i[d] * stride[d], 0 <= i[d] < size[d]; strides in bytes.
struct Strided {
  int64_t base, width;
  int64_t size[3], stride[3];
};
inline Strided strided(const void* base, int64_t width, int64_t bytes, const int64_t (&size)[3], const int64_t* stride) {
  Strided s = {(int64_t)reinterpret_cast<intptr_t>(base), width, {}, {}};
  for (int d = 0; d < 3; ++d) {
    s.size[d] = size[d];
    s.stride[d] = stride[d] * bytes;
    if (s.stride[d] < 0) {                       // the same runs from the other end
      s.base += (size[d] - 1) * s.stride[d];
      s.stride[d] = -s.stride[d];
    }
  }
  return s;
}
inline bool holds_nothing(const Strided& s) { return s.size[0] <= 0 || s.size[1] <= 0 || s.size[2] <= 0; }

// False only if no two runs of the array share a byte: each dimension steps over all that those of smaller strides reach.
inline bool may_overlap_itself(const Strided& s) {
  if (holds_nothing(s)) return false;
  int order[3] = {0, 1, 2};
  std::sort(order, order + 3, [&](int a, int b) { return s.stride[a] < s.stride[b]; });
  int64_t reach = s.width;
  for (int d : order) {
    if (s.size[d] <= 1) continue;
    if (s.stride[d] < reach) return true;
    reach += (s.size[d] - 1) * s.stride[d];
  }
  return false;
}

// False only if no run of a shares a byte with one of b.  Dimensions of the same stride in both (views of one tensor) are one dimension of
// differences; what is left is taken for an interval.
inline bool may_overlap(const Strided& a, const Strided& b) {
  if (holds_nothing(a) || holds_nothing(b)) return false;
  struct Steps {
    int64_t stride, lo, hi;
  } steps[3];
  int n = 0;
  int64_t lo = -a.width + 1, hi = b.width - 1;   // b's byte minus a's, beyond the starts of their runs
  bool used[3] = {};
  for (int d = 0; d < 3; ++d) {
    if (a.size[d] <= 1) continue;
    int e = 0;
    while (e < 3 && (used[e] || b.size[e] <= 1 || b.stride[e] != a.stride[d])) ++e;
    if (e < 3 && a.stride[d] > 0) {
      used[e] = true;
      steps[n++] = Steps{a.stride[d], -(a.size[d] - 1), b.size[e] - 1};
    } else {
      lo -= (a.size[d] - 1) * a.stride[d];
    }
  }
  for (int e = 0; e < 3; ++e)
    if (!used[e]) hi += (b.size[e] - 1) * b.stride[e];
  std::sort(steps, steps + n, [](const Steps& x, const Steps& y) { return x.stride < y.stride; });
  // Is a sum of steps[0 .. k) and a number in [lo, hi] equal to -delta?  From the largest stride down: few multiples of it are near enough.
  struct Search {
    const Steps* steps;
    int64_t lo, hi;
    bool found(int k, int64_t delta) const {
      int64_t low = lo, high = hi;
      for (int i = 0; i + 1 < k; ++i) {
        low += steps[i].lo * steps[i].stride;
        high += steps[i].hi * steps[i].stride;
      }
      if (k == 0) return delta + low <= 0 && delta + high >= 0;
      const Steps& s = steps[k - 1];
      auto down = [](int64_t x, int64_t y) { return x / y - (x % y != 0 && x < 0 ? 1 : 0); };
      const int64_t first = std::max(s.lo, -down(delta + high, s.stride)), last = std::min(s.hi, down(-delta - low, s.stride));
      if (last - first > 64) return true;        // (strides that do not nest)
      for (int64_t m = first; m <= last; ++m)
        if (found(k - 1, delta + m * s.stride)) return true;
      return false;
    }
  };
  return Search{steps, lo, hi}.found(n, b.base - a.base);
}

}  // namespace fa

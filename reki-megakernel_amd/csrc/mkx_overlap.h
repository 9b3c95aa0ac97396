// Views of one buffer that share elements: the check ahead of a launch whose outputs must not be its inputs.
#pragma once
#include <stdint.h>

namespace mkx {

struct View {  // [T, n, hd] 16-bit numbers at p, strides in elements
  const void* p;
  int64_t n, st, sh;
};

// Whether x and y, of T tokens each and 16-byte aligned, share an element. Views of the same strides are told exactly where the
// larger stride spans the other axis, as in a buffer of [T, N, hd] or [N, T, hd]; of other pairs nothing is said (false).
inline bool share_elements(View x, View y, int64_t T, int64_t hd) {
  auto most = [](int64_t a, int64_t b) { return a > b ? a : b; };
  // the stride of an axis of one entry says nothing
  if (x.n == 1) x.sh = y.n == 1 ? hd : y.sh;
  if (y.n == 1) y.sh = x.sh;
  if (T == 1) x.st = y.st = most(x.n, y.n) * most(x.sh, hd);
  if (x.st != y.st || x.sh != y.sh) return false;
  const bool by_token = x.st >= x.sh;
  struct Axis {
    int64_t stride, lo, hi, count;  // of x's index less y's
  } t = {x.st, -(T - 1), T - 1, T}, h = {x.sh, -(y.n - 1), x.n - 1, most(x.n, y.n)}, &outer = by_token ? t : h, &inner = by_token ? h : t;
  if (inner.stride < hd || outer.stride < (inner.count - 1) * inner.stride + hd) return false;
  const int64_t d = ((intptr_t)y.p - (intptr_t)x.p) / 2;  // = (outer) stride + (inner) stride + (column), each less y's
  for (int64_t o = d / outer.stride - 1; o <= d / outer.stride + 1; ++o) {
    const int64_t r = d - o * outer.stride;
    if (o < outer.lo || o > outer.hi) continue;
    for (int64_t i = r / inner.stride - 1; i <= r / inner.stride + 1; ++i)
      if (i >= inner.lo && i <= inner.hi && r - i * inner.stride < hd && i * inner.stride - r < hd) return true;
  }
  return false;
}

}  // namespace mkx

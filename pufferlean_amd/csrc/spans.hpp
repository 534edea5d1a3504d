// Memory that strided arrays take, on the host: whether two of them share an element, or one holds an element twice. Column slices of one
// buffer lie between each other without that, so bounds do not decide it; sums of strides do.
#pragma once
#include <cstdint>

namespace ph {

// w contiguous bytes at p + i0 s0 + i1 s1 + i2 s2 for every i < n, strides in bytes.
struct Span {
  const void* p;
  long w, n[3], s[3];
  bool empty() const { return !p || w <= 0 || n[0] <= 0 || n[1] <= 0 || n[2] <= 0; }
};
inline Span flat(const void* p, long bytes) { return {p, bytes, {1, 1, 1}, {0, 0, 0}}; }

// sum of c[k] x[k], lo[k] <= x[k] <= hi[k], the largest c first.
struct StrideSum {
  int k = 0;
  long c[6], lo[6], hi[6];
  int steps = 4096;  // nested strides leave two or three values each; whatever asks for more than these counts as apart

  void add(long stride, long from, long to) {
    if (stride == 0 || (from == 0 && to == 0)) return;
    if (stride < 0) {
      const long f = from;
      stride = -stride, from = -to, to = -f;
    }
    int i = 0;
    while (i < k && c[i] > stride) i++;
    if (i < k && c[i] == stride) {
      lo[i] += from, hi[i] += to;
      return;
    }
    for (int j = k++; j > i; j--) c[j] = c[j - 1], lo[j] = lo[j - 1], hi[j] = hi[j - 1];
    c[i] = stride, lo[i] = from, hi[i] = to;
  }
  // Whether the terms from i on reach from..to (other: not with all of them zero).
  bool reach(long from, long to, bool other, int i = 0) {
    if (i == k) return from <= 0 && to >= 0 && !other;
    if (--steps < 0) return false;
    long least = 0, most = 0;
    for (int j = i + 1; j < k; j++) least += c[j] * lo[j], most += c[j] * hi[j];
    auto down = [&](long v) { return v >= 0 ? v / c[i] : -((-v + c[i] - 1) / c[i]); };
    long a = -down(most - from), b = down(to - least);
    if (a < lo[i]) a = lo[i];
    if (b > hi[i]) b = hi[i];
    if (i == k - 1) return a <= b && !(other && a == 0 && b == 0);
    for (long x = a; x <= b && steps > 0; x++)
      if (reach(from - c[i] * x, to - c[i] * x, other && x == 0, i + 1)) return true;
    return false;
  }
};
inline bool meet(const Span& a, const Span& b) {
  if (a.empty() || b.empty()) return false;
  StrideSum t;
  for (int i = 0; i < 3; i++) {
    t.add(a.s[i], 0, a.n[i] - 1);
    t.add(b.s[i], -(b.n[i] - 1), 0);
  }
  const long d = (long)((intptr_t)b.p - (intptr_t)a.p);
  return t.reach(d - (a.w - 1), d + (b.w - 1), false);
}
inline bool folds(const Span& a) {
  if (a.empty()) return false;
  StrideSum t;
  for (int i = 0; i < 3; i++) {
    if (a.n[i] > 1 && a.s[i] == 0) return true;
    for (int j = 0; j < i; j++)
      if (a.n[i] > 1 && a.n[j] > 1 && (a.s[i] == a.s[j] || a.s[i] == -a.s[j])) return true;
    t.add(a.s[i], -(a.n[i] - 1), a.n[i] - 1);
  }
  return t.reach(-(a.w - 1), a.w - 1, true);
}

}  // namespace ph

// Whether two operands of a call share memory. An operand is `rows` x `heads` runs of `bytes` bytes, `row` and `head`
// bytes apart: what is written must not lie in what another workgroup reads, or writes, whatever the views' layout. Views
// of one allocation that interleave (q, k and v of one projection) share nothing, so extents alone do not tell.
// Host code only; no dependency.
#pragma once
#include <algorithm>
#include <cstdint>
#include <utility>

namespace nrse_overlap {

struct Area {
  const char* name;
  uintptr_t at;
  long long rows, row, heads, head, bytes;
};

inline Area flat(const char* name, const void* p, long long bytes) {
  return Area{name, (uintptr_t)p, 1, 0, 1, 0, bytes};
}

// An area with the larger of its strides outside: `n` groups `step` apart of `m` runs `gap` apart of `w` bytes.
struct Lattice {
  long long at, n, step, m, gap, w;
  long long group() const { return (m - 1) * gap + w; }
  long long extent() const { return (n - 1) * step + group(); }
};

inline Lattice lattice(const Area& a) {
  Lattice l{(long long)a.at, a.rows, a.row, a.heads, a.head, a.bytes};
  if (l.n == 1 || (l.m > 1 && l.gap > l.step)) {
    std::swap(l.n, l.m);
    std::swap(l.step, l.gap);
  }
  if (l.m == 1) l.gap = 0;
  else if (l.gap <= l.w) l.w = l.group(), l.m = 1, l.gap = 0;                // runs that touch are one
  if (l.n == 1) l.step = 0;
  else if (l.step < l.group() || (l.m == 1 && l.step == l.w))                // groups that interleave: the whole extent
    l.w = l.extent(), l.n = l.m = 1, l.step = l.gap = 0;
  return l;
}

inline long long ceil_div(long long a, long long b) { return a >= 0 ? (a + b - 1) / b : -(-a / b); }   // b > 0

// is there a j in [0, n) with lo < j step < hi (n == 1: j = 0)
inline bool between(long long lo, long long hi, long long n, long long step, long long& first, long long& last) {
  if (n == 1) {
    first = last = 0;
    return lo < 0 && 0 < hi;
  }
  first = std::max(0LL, ceil_div(lo + 1, step));
  last = std::min(n - 1, ceil_div(hi, step) - 1);
  return first <= last;
}

// one group of a against one of b that starts `shift` behind it
inline bool groups_meet(const Lattice& a, const Lattice& b, long long shift) {
  long long f, l;
  for (long long i = 0; i < a.m; ++i)
    if (between(i * a.gap - shift - b.w, i * a.gap - shift + a.w, b.m, b.gap, f, l)) return true;
  return false;
}

// (more than `limit` pairs to look at, which takes different strides and interleaved allocations: taken to meet)
inline bool meet(const Area& x, const Area& y, long long limit = 1 << 22) {
  if (x.rows <= 0 || x.heads <= 0 || x.bytes <= 0 || y.rows <= 0 || y.heads <= 0 || y.bytes <= 0) return false;
  Lattice a = lattice(x), b = lattice(y);
  long long d = b.at - a.at;
  if (d >= a.extent() || -d >= b.extent()) return false;
  if (a.n > 1 && b.n > 1 && a.step == b.step) {
    // groups i of a and i + k of b are all d + k step apart
    long long lo = ceil_div(-b.group() - d + 1, a.step), hi = ceil_div(a.group() - d, a.step) - 1;
    lo = std::max(lo, -(a.n - 1));
    hi = std::min(hi, b.n - 1);
    for (long long k = lo; k <= hi; ++k)
      if (groups_meet(a, b, d + k * a.step)) return true;
    return false;
  }
  if (a.step < b.step || a.n == 1) {   // a: the one whose groups are further apart
    std::swap(a, b);
    d = -d;
  }
  long long looked = 0, f, l, i0, i1;
  if (!between(d - a.group(), d + b.extent(), a.n, a.step, i0, i1)) return false;
  for (long long i = i0; i <= i1; ++i) {
    if (++looked > limit) return true;
    const long long at = i * a.step - d;   // from b's start
    if (!between(at - b.group(), at + a.group(), b.n, b.step, f, l)) continue;
    for (long long j = f; j <= l; ++j) {
      if (++looked > limit) return true;
      if (groups_meet(a, b, j * b.step - at)) return true;
    }
  }
  return false;
}

}  // namespace nrse_overlap

// Do operands (rows, heads, elements) lie over one another? Kernels whose threads
// write one while others read the next refuse that.
#pragma once
#include <torch/extension.h>

#include <algorithm>

namespace nk {

// The bytes of one operand: `outer` runs of `inner` items of `item` bytes, at strides.
struct Lattice {
  int64_t at, item, inner, inner_stride, outer, outer_stride;
  bool empty;

  explicit Lattice(const torch::Tensor& t)
      : at(int64_t(reinterpret_cast<uintptr_t>(t.data_ptr()))), item(t.size(2) * t.element_size()), inner(t.size(1)),
        inner_stride(t.stride(1) * t.element_size()), outer(t.size(0)), outer_stride(t.stride(0) * t.element_size()),
        empty(item == 0 || inner == 0 || outer == 0) {
    if (outer > 1 && inner > 1 && outer_stride < inner_stride) {  // heads before rows
      std::swap(outer, inner);
      std::swap(outer_stride, inner_stride);
    } else if (outer == 1 && inner > 1) {
      std::swap(outer, inner);
      std::swap(outer_stride, inner_stride);
    }
    if (inner == 1) inner_stride = item;
  }
  int64_t run() const { return (inner - 1) * inner_stride + item; }
  int64_t end() const { return at + (outer - 1) * outer_stride + run(); }
  // No byte of it is named twice.
  bool simple() const {
    return empty || ((inner == 1 || inner_stride >= item) && (outer == 1 || outer_stride >= run()));
  }
};

// Two runs of m and n bytes, `gap` apart, that both repeat every `period` bytes.
inline bool apart(int64_t gap, int64_t m, int64_t n, int64_t period) {
  gap = (gap % period + period) % period;
  return gap >= m && gap + n <= period;
}

// No byte is in both. Operands that share a period of rows (column blocks of one buffer)
// or of heads (heads of several operands in turn) are told apart; others that interleave
// count as lying over one another.
inline bool disjoint(const Lattice& a, const Lattice& b) {
  if (a.empty || b.empty || a.end() <= b.at || b.end() <= a.at) return true;
  const int64_t gap = b.at - a.at;
  const int64_t period = a.outer > 1 ? a.outer_stride : b.outer_stride;
  if (period > 0 && (a.outer == 1 || a.outer_stride == period) && (b.outer == 1 || b.outer_stride == period) &&
      apart(gap, a.run(), b.run(), period))
    return true;
  const int64_t step = a.inner > 1 ? a.inner_stride : b.inner_stride;
  auto repeats = [&](const Lattice& l) {
    return (l.inner == 1 || l.inner_stride == step) && (l.outer == 1 || l.outer_stride % step == 0);
  };
  return step > 0 && repeats(a) && repeats(b) && apart(gap, a.item, b.item, step);
}

// An operand of a call, for the checks below.
struct Operand {
  const torch::Tensor& t;
  const char* name;
  Lattice lies;
  Operand(const torch::Tensor& x, const char* n) : t(x), name(n), lies(x) {}
};

// `out` takes the result of `in`: in place, or in memory of its own.
inline void check_result(const Operand& in, const Operand& out) {
  TORCH_CHECK(out.lies.simple(), out.name, ": elements of the output share memory");
  const bool same = in.lies.at == out.lies.at && in.t.sizes() == out.t.sizes() && in.t.strides() == out.t.strides();
  TORCH_CHECK(same || disjoint(in.lies, out.lies), in.name, ": overlaps its output");
}

inline void check_disjoint(const Operand& x, const Operand& y) {
  TORCH_CHECK(disjoint(x.lies, y.lies), x.name, " overlaps ", y.name);
}

}  // namespace nk

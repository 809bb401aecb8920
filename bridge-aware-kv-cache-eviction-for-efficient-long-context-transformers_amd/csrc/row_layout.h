// Where the rows of a strided tensor lie, for calls that write several rows at once: rows
// that share memory would be written in any order (host code).
#pragma once

#include <cstdint>

namespace cab {

// Rows of `row` elements at three strides: the dims of more than one place, by falling stride.
// `extent`: elements from the first to behind the last. `apart`: each stride spans what the smaller ones cover, so that no two rows share an element.
// (Sufficient; of layouts that torch's views make, only overlapping ones fail it.)
struct RowLayout {
  int64_t st[3], size[3], row, low = 0, extent;  // elements; low: of the first one, from the pointer
  int dims = 0;
  bool empty = false, apart = true;

  RowLayout(const int64_t* strides, const int64_t* sizes, int64_t row_elements) : row(row_elements) {
    for (int d = 0; d < 3; ++d) {
      empty = empty || sizes[d] <= 0;
      if (sizes[d] <= 1) continue;
      const int64_t s = strides[d] < 0 ? -strides[d] : strides[d];
      int at = dims++;
      for (; at > 0 && st[at - 1] < s; --at) {
        st[at] = st[at - 1];
        size[at] = size[at - 1];
      }
      st[at] = s;
      size[at] = sizes[d];
    }
    // (past 2^60 elements nothing is addressed: counts as not apart)
    constexpr int64_t FAR = int64_t{1} << 60;
    extent = row;
    for (int d = dims - 1; d >= 0; --d) {
      const bool far = extent >= FAR || st[d] > (FAR - extent) / (size[d] - 1);
      apart = apart && !far && st[d] >= extent;
      extent = far ? FAR : extent + (size[d] - 1) * st[d];
    }
    for (int d = 0; d < 3 && extent < FAR; ++d)
      if (sizes[d] > 1 && strides[d] < 0) low += (sizes[d] - 1) * strides[d];
  }

  bool same_as(const RowLayout& o) const {
    bool same = dims == o.dims && row == o.row && low == o.low;
    for (int d = 0; d < dims && same; ++d) same = st[d] == o.st[d] && size[d] == o.size[d];
    return same;
  }

  // Whether rows of a tensor laid out so and of one `diff` elements further on share an element:
  // diff is then a sum of places times strides, less than a row off. As strides span what is
  // below them (the rows are apart), only the two nearest numbers of places can be it.
  bool meets(int64_t diff, int d = 0) const {
    if (d == dims) return diff < row && -diff < row;
    const int64_t k = diff / st[d] - (diff % st[d] < 0);
    for (int64_t i = k; i <= k + 1; ++i)
      if (i < size[d] && -i < size[d] && meets(diff - i * st[d], d + 1)) return true;
    return false;
  }
};

// Whether two tensors (a layout each, elements of es bytes) may share memory: exact for rows
// that are apart and laid out alike, else whether their spans meet.
inline bool rows_share(const void* a, const RowLayout& x, const void* b, const RowLayout& y, int64_t es) {
  if (x.empty || y.empty) return false;
  const int64_t from_a = static_cast<int64_t>(reinterpret_cast<uintptr_t>(a)) + x.low * es;
  const int64_t from_b = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b)) + y.low * es;
  if (from_a + x.extent * es <= from_b || from_b + y.extent * es <= from_a) return false;
  return !x.apart || !x.same_as(y) || x.meets((from_b - from_a) / es);
}

}  // namespace cab

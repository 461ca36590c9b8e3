// Row grids on the device (fd_rows as a kernel argument) and the row index
// split, shared by the row-wise kernels (fd_rows.cu, fd_quant.cu).
#pragma once

#include "fd_common.cuh"

namespace fd {

// Plain (coherent) 16-byte load without L1 allocation.  Used where an output
// may alias the input (in-place residual), so the non-coherent path is avoided.
FD_DEV uint4 ld_plain16(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

struct RowsArg {
  char* ptr;
  int64_t sa, sb, sc, col;
};

inline RowsArg rows_arg(const fd_rows* r) {
  RowsArg a;
  a.ptr = static_cast<char*>(r ? r->ptr : nullptr);
  a.sa = r ? r->sa : 0;
  a.sb = r ? r->sb : 0;
  a.sc = r ? r->sc : 0;
  a.col = r ? r->col : 0;
  return a;
}

template <typename T>
FD_DEV T* row_ptr(const RowsArg& g, int64_t row, int64_t B, int64_t C) {
  return reinterpret_cast<T*>(g.ptr) + row_base(row, B, C, g.sa, g.sb, g.sc);
}

// Element offset of row `row` in a row grid.  FLAT: a 2-D grid (one leading
// dimension).  Otherwise the (ia, ib, ic) split in 32-bit arithmetic (the host
// sends grids of 2^32 rows or more to the generic kernel).
struct RowIdx {
  uint32_t ia, ib, ic;
};
template <bool FLAT>
FD_DEV RowIdx split_row(int64_t row, int64_t B, int64_t C) {
  if (FLAT) return {0u, 0u, static_cast<uint32_t>(row)};
  const uint32_t r = static_cast<uint32_t>(row), c = static_cast<uint32_t>(C), b = static_cast<uint32_t>(B);
  const uint32_t t = r / c;
  return {t / b, t % b, r % c};
}
FD_DEV int64_t offset_of(const RowsArg& g, const RowIdx& i) {
  return i.ia * g.sa + i.ib * g.sb + static_cast<int64_t>(i.ic) * g.sc;
}

}  // namespace fd

// Checks of the operand descriptions that the recurrent-block operators share.
#pragma once

#include <initializer_list>

#include "host_support.hpp"

namespace tcu {

inline bool aligned_to(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
inline size_t element_bytes(int dtype) { return dtype == TCU_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == TCU_F16 || dtype == TCU_BF16 || dtype == TCU_F32; }
inline bool known_activation(int act) { return act >= TCU_ACT_NONE && act <= TCU_ACT_SIGMOID; }

// HIP launches fewer than 2^32 threads at a time.
inline bool launch_fits(size_t blocks, size_t threads) { return blocks <= 0xffffffffu / threads; }

// A matrix of `rows` x `width` elements whose rows are `stride` elements apart; clears *whole_chunks if its rows do not all
// begin on 16 bytes.
inline int check_matrix(const std::string &w, const char *name, const void *p, size_t stride, size_t rows, size_t width, int dtype, bool *whole_chunks) {
  if (!p) return report_failure(TCU_ERR_INVALID_ARG, w + ": " + name + " is null");
  if (rows > 1 && stride < width) return report_failure(TCU_ERR_INVALID_ARG, w + ": the rows of " + name + " overlap (its stride is below its width)");
  size_t elements = 0;
  const size_t e = element_bytes(dtype);
  if (rows && !product_fits(stride, rows - 1, &elements)) return report_failure(TCU_ERR_INVALID_ARG, w + ": " + name + ": stride * rows overflows");
  if (elements > (~(size_t)0) / e - width) return report_failure(TCU_ERR_INVALID_ARG, w + ": " + name + ": stride * rows overflows");
  if (!aligned_to(p, e)) return report_failure(TCU_ERR_INVALID_ARG, w + ": " + name + " is not aligned to its elements");
  if (!aligned_to(p, 16) || (rows > 1 && stride * e % 16 != 0)) *whole_chunks = false;
  return TCU_OK;
}
// a vector of `e`-byte elements that may be missing
inline int check_vector(const std::string &w, const char *name, const void *p, size_t e, bool *whole_chunks) {
  if (p && !aligned_to(p, e)) return report_failure(TCU_ERR_INVALID_ARG, w + ": " + name + " is not aligned to its elements");
  if (p && !aligned_to(p, 16)) *whole_chunks = false;
  return TCU_OK;
}
// What an operand takes of memory: `rows` rows of `width` elements of `bytes` bytes, `stride` elements apart.
struct Place {
  const char *name;
  const void *p;
  size_t stride, rows, width, bytes;
};
// whether two operands have an element in common; rows at the same distance may lie between each other (slices of one wider matrix)
inline bool places_meet(const Place &a, const Place &b) {
  if (!a.p || !b.p || a.rows * a.width == 0 || b.rows * b.width == 0) return false;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
  const size_t row_a = a.width * a.bytes, row_b = b.width * b.bytes, step = a.stride * a.bytes;
  if (pa + (a.rows - 1) * step + row_a <= pb || pb + (b.rows - 1) * b.stride * b.bytes + row_b <= pa) return false;
  if (a.rows == 1 || b.rows == 1 || step != b.stride * b.bytes) return true;
  const size_t of_b = pb >= pa ? (size_t)(pb - pa) % step : (step - (size_t)(pa - pb) % step) % step;  // from the beginning of a row of a to that of the next row of b
  return of_b < row_a || of_b + row_b > step;
}
inline bool same_place(const Place &a, const Place &b) { return a.p == b.p && a.bytes == b.bytes && a.rows == b.rows && a.width == b.width && (a.rows <= 1 || a.stride == b.stride); }
// An output that shares memory with another operand: it may stand in the very place of those of `replaceable`, and must lie apart from `others`.
inline int check_output_place(const std::string &w, const Place &out, std::initializer_list<Place> replaceable, std::initializer_list<Place> others) {
  for (const Place &q : replaceable)
    if (places_meet(out, q) && !same_place(out, q)) return report_failure(TCU_ERR_INVALID_ARG, w + ": " + out.name + " shares memory with " + q.name + " but is not in its place (address, size and stride)");
  for (const Place &q : others)
    if (places_meet(out, q)) return report_failure(TCU_ERR_INVALID_ARG, w + ": " + out.name + " shares memory with " + q.name);
  return TCU_OK;
}
// The size a call reports for a workspace of which it uses `used` bytes: 256 says that it uses none.
inline size_t smallest_workspace(size_t used) { return used == 0 ? 256 : used < 512 ? 512 : used; }
inline int check_workspace(const std::string &w, const void *workspace, size_t have, size_t need) {
  if (have < need) return report_failure(TCU_ERR_WORKSPACE, w + ": workspace of " + std::to_string(have) + " bytes, needs " + std::to_string(need));
  if (!aligned_to(workspace, 256)) return report_failure(TCU_ERR_INVALID_ARG, w + ": the workspace must be 256-byte aligned");
  return TCU_OK;
}

}  // namespace tcu

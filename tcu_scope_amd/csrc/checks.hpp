// Checks of the operand descriptions that the recurrent-block operators share.
#pragma once

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
// The size a call reports for a workspace of which it uses `used` bytes: 256 says that it uses none.
inline size_t smallest_workspace(size_t used) { return used == 0 ? 256 : used < 512 ? 512 : used; }
inline int check_workspace(const std::string &w, const void *workspace, size_t have, size_t need) {
  if (have < need) return report_failure(TCU_ERR_WORKSPACE, w + ": workspace of " + std::to_string(have) + " bytes, needs " + std::to_string(need));
  if (!aligned_to(workspace, 256)) return report_failure(TCU_ERR_INVALID_ARG, w + ": the workspace must be 256-byte aligned");
  return TCU_OK;
}

}  // namespace tcu

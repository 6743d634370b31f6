// C ABI of the fused product (declared in include/tcu_scope.h).
#include <hip/hip_runtime.h>

#include "fused_gemm_host.hpp"
#include "stream_device.hpp"

extern "C" {

int tcu_fused_gemm(const tcu_fused_gemm_shape *shape, const void *d_A, size_t lda, const void *d_B, size_t ldb, const void *d_bias, const void *d_C, size_t ldc, void *d_D, size_t ldd, void *d_Z, size_t ldz,
                   void *d_workspace, size_t *workspace_bytes, void *stream) {
  return tcu::on_stream_device("tcu_fused_gemm", stream,
                               [&] { return tcu::fused_gemm_dispatch(shape, d_A, lda, d_B, ldb, d_bias, d_C, ldc, d_D, ldd, d_Z, ldz, d_workspace, workspace_bytes, stream); });
}

int tcu_fused_gemm_backward(const tcu_fused_gemm_shape *shape, const void *d_dD, size_t lddd, const void *d_A, size_t lda, const void *d_B, size_t ldb, const void *d_Z, size_t ldz, void *d_dA, size_t ldda,
                            void *d_dB, size_t lddb, float *d_dbias, void *d_workspace, size_t *workspace_bytes, void *stream) {
  return tcu::on_stream_device("tcu_fused_gemm_backward", stream, [&] {
    return tcu::fused_gemm_backward_dispatch(shape, d_dD, lddd, d_A, lda, d_B, ldb, d_Z, ldz, d_dA, ldda, d_dB, lddb, d_dbias, d_workspace, workspace_bytes, stream);
  });
}

}  // extern "C"

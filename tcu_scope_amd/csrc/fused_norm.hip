// C ABI of the fused norm (declared in include/tcu_scope.h).
#include <hip/hip_runtime.h>

#include "fused_norm_host.hpp"
#include "stream_device.hpp"

extern "C" {

int tcu_fused_norm(const tcu_fused_norm_shape *shape, const void *d_x, size_t x_stride, const void *d_residual, size_t residual_stride, const void *d_gate, size_t gate_stride, const void *d_weight,
                   const void *d_bias, const void *d_channel_scale, void *d_out, size_t out_stride, void *d_residual_out, size_t residual_out_stride, void *stream) {
  return tcu::on_stream_device("tcu_fused_norm", stream, [&] {
    return tcu::fused_norm_dispatch(shape, d_x, x_stride, d_residual, residual_stride, d_gate, gate_stride, d_weight, d_bias, d_channel_scale, d_out, out_stride, d_residual_out, residual_out_stride, stream);
  });
}

int tcu_fused_norm_backward(const tcu_fused_norm_shape *shape, const void *d_dout, size_t dout_stride, const void *d_z, size_t z_stride, const void *d_gate, size_t gate_stride, const void *d_weight,
                            const void *d_bias, const void *d_channel_scale, const void *d_x, size_t x_stride, const void *d_dresidual_out, size_t dresidual_out_stride, void *d_dx, size_t dx_stride,
                            void *d_dgate, size_t dgate_stride, void *d_dresidual, size_t dresidual_stride, float *d_dweight, float *d_dbias, float *d_dchannel_scale, void *d_workspace,
                            size_t *workspace_bytes, void *stream) {
  return tcu::on_stream_device("tcu_fused_norm_backward", stream, [&] {
    return tcu::fused_norm_backward_dispatch(shape, d_dout, dout_stride, d_z, z_stride, d_gate, gate_stride, d_weight, d_bias, d_channel_scale, d_x, x_stride, d_dresidual_out, dresidual_out_stride, d_dx,
                                             dx_stride, d_dgate, dgate_stride, d_dresidual, dresidual_stride, d_dweight, d_dbias, d_dchannel_scale, d_workspace, workspace_bytes, stream);
  });
}

}  // extern "C"

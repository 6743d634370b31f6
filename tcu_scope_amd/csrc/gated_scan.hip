// C ABI of the gated scan (declared in include/tcu_scope.h).
#include <hip/hip_runtime.h>

#include "gated_scan_host.hpp"
#include "stream_device.hpp"

extern "C" {

int tcu_gated_scan(const tcu_gated_scan_shape *shape, const void *d_x, size_t x_stride, const void *d_g, size_t g_stride, void *d_h, size_t h_stride, const float *d_h0, float *d_h_last, void *d_workspace,
                   size_t *workspace_bytes, void *stream) {
  return tcu::on_stream_device("tcu_gated_scan", stream, [&] { return tcu::gated_scan_dispatch(shape, d_x, x_stride, d_g, g_stride, d_h, h_stride, d_h0, d_h_last, d_workspace, workspace_bytes, stream); });
}

int tcu_gated_scan_backward(const tcu_gated_scan_shape *shape, const void *d_dh, size_t dh_stride, const void *d_x, size_t x_stride, const void *d_g, size_t g_stride, const void *d_h, size_t h_stride,
                            const float *d_h0, const float *d_dh_last, void *d_dx, size_t dx_stride, void *d_dg, size_t dg_stride, float *d_dh0, void *d_workspace, size_t *workspace_bytes, void *stream) {
  return tcu::on_stream_device("tcu_gated_scan_backward", stream, [&] {
    return tcu::gated_scan_backward_dispatch(shape, d_dh, dh_stride, d_x, x_stride, d_g, g_stride, d_h, h_stride, d_h0, d_dh_last, d_dx, dx_stride, d_dg, dg_stride, d_dh0, d_workspace, workspace_bytes, stream);
  });
}

int tcu_gated_scan_step(int dtype, int gate, size_t channels, size_t num_rows, const void *d_x, size_t x_stride, const void *d_g, size_t g_stride, void *d_h, size_t h_stride, const float *d_state,
                        float *d_new_state, size_t num_slots, const int32_t *d_slots, int zero_padding, void *stream) {
  return tcu::on_stream_device("tcu_gated_scan_step", stream, [&] {
    return tcu::gated_scan_step_dispatch(dtype, gate, channels, num_rows, d_x, x_stride, d_g, g_stride, d_h, h_stride, d_state, d_new_state, num_slots, d_slots, zero_padding, stream);
  });
}

}  // extern "C"

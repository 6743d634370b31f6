// Argument checks, workspace layout and kernel selection of the fused norm's entry points.
#pragma once

#include "checks.hpp"
#include "column_sum.hpp"
#include "fused_norm.hpp"
#include "launch.hpp"

namespace tcu {

constexpr size_t kNormLaunchRows = (size_t)1 << 21;  // of one launch: up to 1024 threads a row, fewer than 2^32 in all
constexpr size_t kNormMaxDim = 16384;    // beyond it a block cannot hold a row and its columns' sums in registers
// Waves that share a row in the gradient's kernel, by the chunks per lane that one wave would need.
inline int norm_back_waves(size_t chunks) { return chunks <= 1 ? 1 : chunks <= 2 ? 2 : chunks <= 4 ? 4 : 8; }
// Its blocks, i.e. partial sums per column: as many as bring 8 waves to every compute unit (8192 x 4096 bf16 gated, 8 waves
// a row: 256 blocks 77 us + 4.7 for the sums, 512 blocks 85 + 7.5; 32768 x 1024: 227 us with half the waves).
constexpr size_t kNormBackWaves = 256 * 8;

inline int check_norm_shape(const std::string &w, const tcu_fused_norm_shape *s) {
  if (!s) return report_failure(TCU_ERR_INVALID_ARG, w + ": null shape");
  if (!known_dtype(s->dtype)) return report_failure(TCU_ERR_INVALID_ARG, w + ": dtype must be TCU_F16, TCU_BF16 or TCU_F32");
  if (s->norm != TCU_NORM_RMS && s->norm != TCU_NORM_LAYER) return report_failure(TCU_ERR_INVALID_ARG, w + ": unknown norm");
  if (s->order != TCU_ORDER_ADD_NORM && s->order != TCU_ORDER_NORM_ADD) return report_failure(TCU_ERR_INVALID_ARG, w + ": unknown order");
  if (!known_activation(s->activation)) return report_failure(TCU_ERR_INVALID_ARG, w + ": unknown activation");
  if (s->dim == 0) return report_failure(TCU_ERR_INVALID_ARG, w + ": dim is 0");
  if (s->dim > kNormMaxDim) return report_failure(TCU_ERR_UNSUPPORTED, w + ": dim is above 16384");
  if (s->rows >= ((size_t)1 << 31)) return report_failure(TCU_ERR_UNSUPPORTED, w + ": 2^31 rows or more");
  return TCU_OK;
}

// Waves that share a row, and chunks per lane: four waves as soon as the row has more than two chunks per lane of one (16384 x
// 4096 bf16 with residual: 4 waves 89.8 us, 1 wave with 8 chunks per lane 92.7; and the shorter way through a row counts where
// there are few).
template <int DT, bool ALIGNED>
inline void launch_fused_norm_rows(const FusedNormParams &p, void *stream) {
  const size_t ct = (p.dim + 64 * Elem<DT>::V - 1) / (64 * Elem<DT>::V);  // chunks per lane if one wave takes the row
  const size_t rows = p.rows, quads = (rows + 3) / 4;
#define TCU_NORM(W, C, BW, blocks) launch(fused_norm_kernel<DT, ALIGNED, W, C, BW>, (unsigned)(blocks), 64u * (BW), stream, p)
  if (ALIGNED && ct == 1) TCU_NORM(1, ALIGNED ? 1 : 2, 4, quads);
  else if (ct <= 2) TCU_NORM(1, 2, 4, quads);
  else if (ALIGNED && ct <= 4) TCU_NORM(4, ALIGNED ? 1 : 2, 4, rows);
  else if (ct <= 8) TCU_NORM(4, 2, 4, rows);
  else if (ALIGNED && ct <= 16) TCU_NORM(4, 4, 4, rows);
  else if (ct <= 32) TCU_NORM(8, 4, 8, rows);
  else TCU_NORM(16, 4, 16, rows);
#undef TCU_NORM
}
template <int DT, bool ALIGNED>
inline void launch_fused_norm(FusedNormParams p, void *stream) {
  for (size_t left = p.rows; left > 0; left -= p.rows) {
    p.rows = left < kNormLaunchRows ? left : kNormLaunchRows;
    launch_fused_norm_rows<DT, ALIGNED>(p, stream);
    auto ahead = [&](auto &q, size_t stride) {
      if (q) q = (char *)q + p.rows * stride * sizeof(typename Elem<DT>::word_t);
    };
    ahead(p.x, p.x_stride);
    ahead(p.residual, p.residual_stride);
    ahead(p.gate, p.gate_stride);
    ahead(p.out, p.out_stride);
    ahead(p.z_out, p.z_out_stride);
  }
}

inline int fused_norm_dispatch(const tcu_fused_norm_shape *s, const void *x, size_t x_stride, const void *residual, size_t residual_stride, const void *gate, size_t gate_stride, const void *weight,
                               const void *bias, const void *channel_scale, void *out, size_t out_stride, void *residual_out, size_t residual_out_stride, void *stream) {
  const std::string w("tcu_fused_norm");
  if (int rc = check_norm_shape(w, s)) return rc;
  if (!residual && s->order == TCU_ORDER_ADD_NORM && (channel_scale || s->scale != 1.0f)) return report_failure(TCU_ERR_INVALID_ARG, w + ": a scale of the residual branch without a residual");
  if (residual_out && (!residual || s->order != TCU_ORDER_ADD_NORM)) return report_failure(TCU_ERR_INVALID_ARG, w + ": d_residual_out goes with TCU_ORDER_ADD_NORM and a residual");
  if (!gate && s->activation != TCU_ACT_NONE) return report_failure(TCU_ERR_INVALID_ARG, w + ": an activation without a gate");
  if (s->rows == 0) return TCU_OK;
  const size_t e = element_bytes(s->dtype);
  bool aligned = s->dim * e % 16 == 0;
  auto matrix = [&](const char *name, const void *p, size_t stride) { return check_matrix(w, name, p, stride, s->rows, s->dim, s->dtype, &aligned); };
  if (int rc = matrix("d_x", x, x_stride)) return rc;
  if (int rc = residual ? matrix("d_residual", residual, residual_stride) : TCU_OK) return rc;
  if (int rc = gate ? matrix("d_gate", gate, gate_stride) : TCU_OK) return rc;
  if (int rc = matrix("d_out", out, out_stride)) return rc;
  if (int rc = residual_out ? matrix("d_residual_out", residual_out, residual_out_stride) : TCU_OK) return rc;
  if (int rc = check_vector(w, "d_weight", weight, e, &aligned)) return rc;
  if (int rc = check_vector(w, "d_bias", bias, e, &aligned)) return rc;
  if (int rc = check_vector(w, "d_channel_scale", channel_scale, e, &aligned)) return rc;
  if (residual_out == out) return report_failure(TCU_ERR_INVALID_ARG, w + ": d_out and d_residual_out are the same buffer");
  const Place px{"d_x", x, x_stride, s->rows, s->dim, e}, pr{"d_residual", residual, residual_stride, s->rows, s->dim, e}, pg{"d_gate", gate, gate_stride, s->rows, s->dim, e}, pw{"d_weight", weight, 0, 1, s->dim, e},
      pb{"d_bias", bias, 0, 1, s->dim, e}, pc{"d_channel_scale", channel_scale, 0, 1, s->dim, e}, po{"d_out", out, out_stride, s->rows, s->dim, e}, pz{"d_residual_out", residual_out, residual_out_stride, s->rows, s->dim, e};
  if (int rc = check_output_place(w, po, {px, pr, pg}, {pw, pb, pc, pz})) return rc;
  if (int rc = check_output_place(w, pz, {px, pr, pg}, {pw, pb, pc})) return rc;
  const FusedNormParams p{x, residual, gate, weight, bias, channel_scale, out, residual_out, x_stride, residual_stride, gate_stride, out_stride, residual_out_stride, s->rows, (unsigned)s->dim, s->eps, s->scale, s->norm, s->order, s->activation};
#define TCU_NORM_TYPE(DT) (aligned ? launch_fused_norm<DT, true>(p, stream) : launch_fused_norm<DT, false>(p, stream))
  if (s->dtype == TCU_F16) TCU_NORM_TYPE(kF16);
  else if (s->dtype == TCU_BF16) TCU_NORM_TYPE(kBF16);
  else TCU_NORM_TYPE(kF32);
#undef TCU_NORM_TYPE
  return TCU_OK;
}

// blocks of the gradient's kernel and partial sums per column
struct NormBackPlan {
  size_t blocks = 0, parts = 0, vectors = 0, bytes = 256;
};
inline NormBackPlan plan_norm_backward(const tcu_fused_norm_shape *s, size_t vectors) {
  NormBackPlan plan;
  const size_t per_wave = 64 * 16 / element_bytes(s->dtype), waves = norm_back_waves((s->dim + per_wave - 1) / per_wave);
  const size_t rows_per_block = waves == 1 ? 4 : 1, block_waves = waves == 1 ? 4 : waves;
  const size_t wanted = (s->rows + rows_per_block - 1) / rows_per_block, most = kNormBackWaves / block_waves;
  plan.blocks = wanted < most ? wanted : most;
  plan.parts = plan.blocks * rows_per_block;
  plan.vectors = vectors;
  const size_t bytes = plan.parts * vectors * s->dim * 4;
  plan.bytes = smallest_workspace(bytes);
  return plan;
}

// A lane has one chunk of the row up to 8 waves: the column sums, the row, the next row and the gate's factors are then all in
// registers.  Longer rows take the lean form.
template <int DT, bool ALIGNED, bool GATE, bool STREAM>
inline void launch_fused_norm_backward(const FusedNormBackParams &p, size_t blocks, void *stream) {
  const size_t ct = (p.dim + 64 * Elem<DT>::V - 1) / (64 * Elem<DT>::V);
#define TCU_NORM(LEAN, W, C, BW) launch(fused_norm_backward_kernel<DT, ALIGNED, GATE, STREAM, LEAN, W, C, BW>, (unsigned)blocks, 64u * (BW), stream, p)
  if (ct <= 1) TCU_NORM(false, 1, 1, 4);
  else if (ct <= 2) TCU_NORM(false, 2, 1, 2);
  else if (ct <= 4) TCU_NORM(false, 4, 1, 4);
  else if (ct <= 8) TCU_NORM(false, 8, 1, 8);
  else if (ct <= 16) TCU_NORM(DT != kF32, 8, 2, 8);  // two chunks of fp32 are as many values as one of 16 bits
  else if (ct <= 32) TCU_NORM(true, 8, 4, 8);
  else TCU_NORM(true, 8, DT == kF32 ? 8 : 4, 8);  // 16-bit types end at ct = 32
#undef TCU_NORM
}
template <int DT>
inline void launch_fused_norm_backward_typed(bool aligned, const FusedNormBackParams &p, size_t blocks, void *stream) {
  const bool streams = p.dstream != nullptr || (p.want_scale && p.order == kOrderAddNorm);
  if (!aligned) launch_fused_norm_backward<DT, false, true, true>(p, blocks, stream);
  else if (p.gate && streams) launch_fused_norm_backward<DT, true, true, true>(p, blocks, stream);
  else if (p.gate) launch_fused_norm_backward<DT, true, true, false>(p, blocks, stream);
  else if (streams) launch_fused_norm_backward<DT, true, false, true>(p, blocks, stream);
  else launch_fused_norm_backward<DT, true, false, false>(p, blocks, stream);
}

inline int fused_norm_backward_dispatch(const tcu_fused_norm_shape *s, const void *dout, size_t dout_stride, const void *z, size_t z_stride, const void *gate, size_t gate_stride, const void *weight,
                                        const void *bias, const void *channel_scale, const void *x, size_t x_stride, const void *dresidual_out, size_t dresidual_out_stride, void *dx, size_t dx_stride,
                                        void *dgate, size_t dgate_stride, void *dresidual, size_t dresidual_stride, float *dweight, float *dbias, float *dchannel_scale, void *workspace,
                                        size_t *workspace_bytes, void *stream) {
  const std::string w("tcu_fused_norm_backward");
  if (int rc = check_norm_shape(w, s)) return rc;
  const bool add_norm = s->order == TCU_ORDER_ADD_NORM;
  const NormBackPlan plan = plan_norm_backward(s, (dweight != nullptr) + (dbias != nullptr) + (dchannel_scale != nullptr));
  if (!workspace_bytes) return report_failure(TCU_ERR_INVALID_ARG, w + ": workspace_bytes is null");
  if (!workspace) {
    *workspace_bytes = plan.bytes;
    return TCU_OK;
  }
  if (int rc = check_workspace(w, workspace, *workspace_bytes, plan.bytes)) return rc;
  if (!gate && s->activation != TCU_ACT_NONE) return report_failure(TCU_ERR_INVALID_ARG, w + ": an activation without a gate");
  if (dgate && !gate) return report_failure(TCU_ERR_INVALID_ARG, w + ": d_dgate without a gate");
  if (!add_norm && (dresidual_out || dresidual)) return report_failure(TCU_ERR_INVALID_ARG, w + ": with TCU_ORDER_NORM_ADD the residual's gradient is d_dout itself");
  if (dchannel_scale && add_norm && !x) return report_failure(TCU_ERR_INVALID_ARG, w + ": d_dchannel_scale needs d_x");
  const size_t e = element_bytes(s->dtype);
  bool aligned = s->dim * e % 16 == 0;
  if (s->rows) {
    auto matrix = [&](const char *name, const void *p, size_t stride) { return check_matrix(w, name, p, stride, s->rows, s->dim, s->dtype, &aligned); };
    if (int rc = matrix("d_dout", dout, dout_stride)) return rc;
    if (int rc = matrix("d_z", z, z_stride)) return rc;
    if (int rc = gate ? matrix("d_gate", gate, gate_stride) : TCU_OK) return rc;
    if (int rc = dchannel_scale && add_norm ? matrix("d_x", x, x_stride) : TCU_OK) return rc;
    if (int rc = dresidual_out ? matrix("d_dresidual_out", dresidual_out, dresidual_out_stride) : TCU_OK) return rc;
    if (int rc = matrix("d_dx", dx, dx_stride)) return rc;
    if (int rc = dgate ? matrix("d_dgate", dgate, dgate_stride) : TCU_OK) return rc;
    if (int rc = dresidual ? matrix("d_dresidual", dresidual, dresidual_stride) : TCU_OK) return rc;
    if (dx == dgate || dx == dresidual || (dgate && dgate == dresidual)) return report_failure(TCU_ERR_INVALID_ARG, w + ": two gradients in the same buffer");
  }
  if (int rc = check_vector(w, "d_weight", weight, e, &aligned)) return rc;
  if (int rc = check_vector(w, "d_bias", bias, e, &aligned)) return rc;
  if (int rc = check_vector(w, "d_channel_scale", channel_scale, e, &aligned)) return rc;
  bool ignored = true;  // these are written element by element
  if (int rc = check_vector(w, "d_dweight", dweight, 4, &ignored)) return rc;
  if (int rc = check_vector(w, "d_dbias", dbias, 4, &ignored)) return rc;
  if (int rc = check_vector(w, "d_dchannel_scale", dchannel_scale, 4, &ignored)) return rc;
  const size_t n = s->rows, d = s->dim;
  const Place pd{"d_dout", dout, dout_stride, n, d, e}, pz{"d_z", z, z_stride, n, d, e}, pg{"d_gate", gate, gate_stride, n, d, e}, px{"d_x", dchannel_scale && add_norm ? x : nullptr, x_stride, n, d, e},
      ps{"d_dresidual_out", dresidual_out, dresidual_out_stride, n, d, e}, pw{"d_weight", weight, 0, 1, d, e}, pb{"d_bias", bias, 0, 1, d, e}, pc{"d_channel_scale", channel_scale, 0, 1, d, e},
      odx{"d_dx", dx, dx_stride, n, d, e}, odg{"d_dgate", dgate, dgate_stride, n, d, e}, odr{"d_dresidual", dresidual, dresidual_stride, n, d, e}, odw{"d_dweight", dweight, 0, 1, d, 4}, odb{"d_dbias", dbias, 0, 1, d, 4},
      odc{"d_dchannel_scale", dchannel_scale, 0, 1, d, 4};
  if (int rc = check_output_place(w, odx, {pd, pz, pg, px, ps}, {pw, pb, pc, odg, odr, odw, odb, odc})) return rc;
  if (int rc = check_output_place(w, odg, {pd, pz, pg, px, ps}, {pw, pb, pc, odr, odw, odb, odc})) return rc;
  if (int rc = check_output_place(w, odr, {pd, pz, pg, px, ps}, {pw, pb, pc, odw, odb, odc})) return rc;
  if (int rc = check_output_place(w, odw, {}, {pd, pz, pg, px, ps, pw, pb, pc, odb, odc})) return rc;
  if (int rc = check_output_place(w, odb, {}, {pd, pz, pg, px, ps, pw, pb, pc, odc})) return rc;
  if (int rc = check_output_place(w, odc, {}, {pd, pz, pg, px, ps, pw, pb, pc})) return rc;
  if (s->rows) {
    FusedNormBackParams p{};
    p.dout = dout;
    p.z = z;
    p.gate = gate;
    p.weight = weight;
    p.bias = bias;
    p.channel_scale = channel_scale;
    p.x = x;
    p.dstream = dresidual_out;
    p.dx = dx;
    p.dgate = dgate;
    p.dresidual = dresidual;
    p.dout_stride = dout_stride;
    p.z_stride = z_stride;
    p.gate_stride = gate_stride;
    p.x_stride = x_stride;
    p.dstream_stride = dresidual_out_stride;
    p.dx_stride = dx_stride;
    p.dgate_stride = dgate_stride;
    p.dresidual_stride = dresidual_stride;
    p.partial = static_cast<float *>(workspace);
    p.rows = s->rows;
    p.dim = (unsigned)s->dim;
    p.eps = s->eps;
    p.scale = s->scale;
    p.norm = s->norm;
    p.order = s->order;
    p.act = s->activation;
    p.want_weight = dweight != nullptr;
    p.want_bias = dbias != nullptr;
    p.want_scale = dchannel_scale != nullptr;
#define TCU_NORM_TYPE(DT) launch_fused_norm_backward_typed<DT>(aligned, p, plan.blocks, stream)
    if (s->dtype == TCU_F16) TCU_NORM_TYPE(kF16);
    else if (s->dtype == TCU_BF16) TCU_NORM_TYPE(kBF16);
    else TCU_NORM_TYPE(kF32);
#undef TCU_NORM_TYPE
  }
  if (plan.vectors) {
    ColumnSumParams q{};
    q.partial = static_cast<const float *>(workspace);
    q.parts = plan.parts;
    q.columns = (unsigned)s->dim;
    for (float *v : {dweight, dbias, dchannel_scale})
      if (v) q.out[q.vectors++] = v;
    launch(column_sum_kernel, (unsigned)((plan.vectors * s->dim + 63) / 64), 64u * kColumnSumWaves, stream, q);
  }
  return TCU_OK;
}

}  // namespace tcu

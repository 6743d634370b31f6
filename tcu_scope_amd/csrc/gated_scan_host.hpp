// Argument checks, workspace layout and kernel selection of the gated scan's entry points.
#pragma once

#include "checks.hpp"
#include "gated_scan.hpp"
#include "launch.hpp"

namespace tcu {

// Tiles: 16 lanes (256 bytes of a row) x 16 or 32 groups of so many places per thread, whose (a, b) stay in registers (two
// waves per SIMD).  Places: 8 | 4 forwards 65536 x 2048 fp16 187 | 228 us (both before the
// kernel loaded ahead of its masks: 8 then takes 173), 4 | 2 | 8 backwards 32768 x 2048 bf16 164 | 223 | 227.
// Blocks of 512 threads where there are few tiles, i.e. where the waits for each other count: 8191 x 1000 bf16 packed 22.5 ->
// 19.1 us, backwards 4099 x 769 fp32 30.2 -> 23.7; from about 1024 tiles on 256 threads are as fast or faster (backwards
// 32768 x 2048 bf16 164 | 178).
constexpr int kScanLanes = 16, kScanPlaces = 8, kScanBackPlaces = 4;
constexpr size_t kScanManyTiles = 1024;
inline unsigned scan_tile_channels(int dtype) { return (unsigned)(kScanLanes * 16 / element_bytes(dtype)); }

struct GatedScanPlan {
  size_t rows = 0, strips = 0, chunks = 0;
  size_t rows_at = 0, entries_at = 0, entries_bytes = 0, bytes = 0;  // workspace: 64 words, the rows' sequences, the entries
  int threads = 256;
  bool chained = false;                                        // several chunks of places: ticket and entries
};

inline int plan_gated_scan(const char *what, const tcu_gated_scan_shape *s, int places, GatedScanPlan *plan) {
  const std::string w(what);
  if (!s) return report_failure(TCU_ERR_INVALID_ARG, w + ": null shape");
  if (!known_dtype(s->dtype)) return report_failure(TCU_ERR_INVALID_ARG, w + ": dtype must be TCU_F16, TCU_BF16 or TCU_F32");
  if (s->gate != TCU_GATE_DECAY && s->gate != TCU_GATE_LOG && s->gate != TCU_GATE_SIGMOID) return report_failure(TCU_ERR_INVALID_ARG, w + ": unknown gate");
  if (s->channels == 0 || s->channels > ((size_t)1 << 28)) return report_failure(TCU_ERR_INVALID_ARG, w + ": channels must be 1 ... 2^28");
  if (s->num_sequences >= ((size_t)1 << 31)) return report_failure(TCU_ERR_UNSUPPORTED, w + ": 2^31 sequences or more");
  if (s->d_offsets) {
    if (s->offset_bits != 32 && s->offset_bits != 64) return report_failure(TCU_ERR_INVALID_ARG, w + ": offset_bits must be 32 or 64");
    if (!aligned_to(s->d_offsets, (size_t)s->offset_bits / 8)) return report_failure(TCU_ERR_INVALID_ARG, w + ": d_offsets is not aligned to its integers");
    plan->rows = s->num_rows;
  } else {
    if (!product_fits(s->num_sequences, s->sequence_length, &plan->rows)) return report_failure(TCU_ERR_INVALID_ARG, w + ": num_sequences * sequence_length overflows");
    if (s->num_rows != plan->rows) return report_failure(TCU_ERR_INVALID_ARG, w + ": num_rows must be num_sequences * sequence_length");
  }
  // place numbers and their successors are 32-bit
  if (plan->rows > ((size_t)1 << 31) - 4096) return report_failure(TCU_ERR_UNSUPPORTED, w + ": more than 2^31 - 4096 rows");
  const unsigned tc = scan_tile_channels(s->dtype);
  plan->strips = (s->channels + tc - 1) / tc;
  auto chunks = [&](int threads) { return (plan->rows + threads / kScanLanes * places - 1) / (threads / kScanLanes * places); };
  if (plan->strips * chunks(256) < kScanManyTiles) plan->threads = 512;
  plan->chunks = chunks(plan->threads);
  if (!launch_fits(plan->strips * plan->chunks, plan->threads)) return report_failure(TCU_ERR_UNSUPPORTED, w + ": rows and channels take more tiles than a launch can have");
  plan->chained = plan->chunks > 1;
  plan->rows_at = 256;
  plan->entries_at = plan->rows_at + (s->d_offsets ? (plan->rows * 4 + 255) / 256 * 256 : 0);
  plan->entries_bytes = plan->chained ? plan->strips * (plan->chunks + plan->chunks / kScanGroup + plan->chunks / (kScanGroup * kScanGroup)) * tc * 8 : 0;
  plan->bytes = plan->entries_at + plan->entries_bytes;
  if (plan->rows == 0 || s->d_offsets || plan->chained) plan->bytes = plan->bytes < 512 ? 512 : plan->bytes;  // the setup kernel runs
  return TCU_OK;
}

template <int DT, int GATE, bool BACK, bool ALIGNED>
inline void launch_gated_scan_kernel(unsigned grid, int threads, void *stream, const GatedScanParams &p) {
  constexpr int PLACES = BACK ? kScanBackPlaces : kScanPlaces;
  if (threads == 512) launch(gated_scan_kernel<DT, GATE, BACK, ALIGNED, kScanLanes, PLACES, 512>, grid, 512u, stream, p);
  else launch(gated_scan_kernel<DT, GATE, BACK, ALIGNED, kScanLanes, PLACES, 256>, grid, 256u, stream, p);
}
template <int DT, bool BACK>
inline void launch_gated_scan_typed(int gate, bool aligned, unsigned grid, int threads, void *stream, const GatedScanParams &p) {
#define TCU_SCAN_GATE(G_) aligned ? launch_gated_scan_kernel<DT, G_, BACK, true>(grid, threads, stream, p) : launch_gated_scan_kernel<DT, G_, BACK, false>(grid, threads, stream, p)
  if (gate == TCU_GATE_DECAY) TCU_SCAN_GATE(kGateDecay);
  else if (gate == TCU_GATE_LOG) TCU_SCAN_GATE(kGateLog);
  else TCU_SCAN_GATE(kGateSigmoid);
#undef TCU_SCAN_GATE
}

// setup (where something has to be cleared or looked up) and scan
template <bool BACK>
inline int run_gated_scan(const tcu_gated_scan_shape *s, const GatedScanPlan &plan, GatedScanParams p, bool aligned, void *workspace, void *stream) {
  unsigned *head = static_cast<unsigned *>(workspace);
  char *base = static_cast<char *>(workspace);
  p.rows = (unsigned)plan.rows;
  p.sequence_rows = (unsigned)s->sequence_length;
  p.channels = (unsigned)s->channels;
  p.zero_outside = s->zero_outside != 0;
  p.near_rows = true;
  for (size_t stride : {p.x_stride, p.g_stride, p.h_stride, p.dh_stride, p.out_stride, p.out_g_stride}) p.near_rows = p.near_rows && stride < ((size_t)1 << 23);
  p.strips = (unsigned)plan.strips;
  p.chunks = (unsigned)plan.chunks;
  p.ticket = plan.chained ? head : nullptr;
  p.expired = head + 1;
  p.entries = reinterpret_cast<unsigned long long *>(base + plan.entries_at);
  p.poll_limit = shared_poll_limit();
  p.mute_tile = shared_mute_partition();
  p.row_sequence = s->d_offsets ? reinterpret_cast<const int *>(base + plan.rows_at) : nullptr;
  if (plan.chained || s->d_offsets || (plan.rows == 0 && p.last)) {
    GatedScanSetup q{};
    q.head = head;
    q.clear = reinterpret_cast<uint4_t *>(base + plan.entries_at);
    q.clear_chunks = plan.entries_bytes / 16;
    q.offsets = s->d_offsets;
    q.offset_bits = s->offset_bits;
    q.sequences = (unsigned)s->num_sequences;
    q.rows = (unsigned)plan.rows;
    q.channels = (unsigned)s->channels;
    q.row_sequence = reinterpret_cast<int *>(base + plan.rows_at);
    q.seed = p.seed;
    q.last = p.last;
    size_t work = q.clear_chunks > plan.rows ? q.clear_chunks : plan.rows;
    if (q.last && (q.offsets || plan.rows == 0) && (size_t)q.sequences * 256 > work) work = (size_t)q.sequences * 256;
    size_t blocks = (work + 255) / 256;
    blocks = blocks < 1 ? 1 : (blocks > 2048 ? 2048 : blocks);
    launch(gated_scan_setup_kernel, (unsigned)blocks, 256u, stream, q);
  }
  if (plan.rows == 0) return TCU_OK;
  const unsigned grid = (unsigned)(plan.strips * plan.chunks);
  if (s->dtype == TCU_F16) launch_gated_scan_typed<kF16, BACK>(s->gate, aligned, grid, plan.threads, stream, p);
  else if (s->dtype == TCU_BF16) launch_gated_scan_typed<kBF16, BACK>(s->gate, aligned, grid, plan.threads, stream, p);
  else launch_gated_scan_typed<kF32, BACK>(s->gate, aligned, grid, plan.threads, stream, p);
  return TCU_OK;
}

inline int gated_scan_dispatch(const tcu_gated_scan_shape *s, const void *x, size_t x_stride, const void *g, size_t g_stride, void *h, size_t h_stride, const void *h0, void *h_last, void *workspace,
                               size_t *workspace_bytes, void *stream) {
  const char *what = "tcu_gated_scan";
  const std::string w(what);
  GatedScanPlan plan;
  if (int rc = plan_gated_scan(what, s, kScanPlaces, &plan)) return rc;
  if (!workspace_bytes) return report_failure(TCU_ERR_INVALID_ARG, w + ": workspace_bytes is null");
  if (!workspace) {
    *workspace_bytes = plan.bytes;
    return TCU_OK;
  }
  if (int rc = check_workspace(w, workspace, *workspace_bytes, plan.bytes)) return rc;
  bool aligned = s->channels % (16 / element_bytes(s->dtype)) == 0;
  if (plan.rows) {
    if (int rc = check_matrix(w, "d_x", x, x_stride, plan.rows, s->channels, s->dtype, &aligned)) return rc;
    if (int rc = check_matrix(w, "d_g", g, g_stride, plan.rows, s->channels, s->dtype, &aligned)) return rc;
    if (int rc = check_matrix(w, "d_h", h, h_stride, plan.rows, s->channels, s->dtype, &aligned)) return rc;
  }
  if (int rc = check_vector(w, "d_h0", h0, 4, &aligned)) return rc;
  if (int rc = check_vector(w, "d_h_last", h_last, 4, &aligned)) return rc;
  const size_t e = element_bytes(s->dtype), n = plan.rows, c = s->channels, states = s->num_sequences;
  const Place px{"d_x", x, x_stride, n, c, e}, pg{"d_g", g, g_stride, n, c, e}, ph{"d_h", h, h_stride, n, c, e}, p0{"d_h0", h0, c, states, c, 4}, pl{"d_h_last", h_last, c, states, c, 4};
  if (int rc = check_output_place(w, ph, {px, pg}, {p0, pl})) return rc;
  if (int rc = check_output_place(w, pl, {p0}, {px, pg})) return rc;
  if (s->num_sequences == 0 && (plan.rows == 0 || !s->zero_outside)) return TCU_OK;
  GatedScanParams p{};
  p.x = x;
  p.x_stride = x_stride;
  p.g = g;
  p.g_stride = g_stride;
  p.out = h;
  p.out_stride = h_stride;
  p.seed = static_cast<const float *>(h0);
  p.last = static_cast<float *>(h_last);
  return run_gated_scan<false>(s, plan, p, aligned, workspace, stream);
}

inline int gated_scan_backward_dispatch(const tcu_gated_scan_shape *s, const void *dh, size_t dh_stride, const void *x, size_t x_stride, const void *g, size_t g_stride, const void *h, size_t h_stride,
                                        const void *h0, const void *dh_last, void *dx, size_t dx_stride, void *dg, size_t dg_stride, void *dh0, void *workspace, size_t *workspace_bytes, void *stream) {
  const char *what = "tcu_gated_scan_backward";
  const std::string w(what);
  GatedScanPlan plan;
  if (int rc = plan_gated_scan(what, s, kScanBackPlaces, &plan)) return rc;
  if (!workspace_bytes) return report_failure(TCU_ERR_INVALID_ARG, w + ": workspace_bytes is null");
  if (!workspace) {
    *workspace_bytes = plan.bytes;
    return TCU_OK;
  }
  if (int rc = check_workspace(w, workspace, *workspace_bytes, plan.bytes)) return rc;
  bool aligned = s->channels % (16 / element_bytes(s->dtype)) == 0;
  if (plan.rows) {
    if (int rc = check_matrix(w, "d_dh", dh, dh_stride, plan.rows, s->channels, s->dtype, &aligned)) return rc;
    if (s->gate == TCU_GATE_SIGMOID)
      if (int rc = check_matrix(w, "d_x", x, x_stride, plan.rows, s->channels, s->dtype, &aligned)) return rc;
    if (int rc = check_matrix(w, "d_g", g, g_stride, plan.rows, s->channels, s->dtype, &aligned)) return rc;
    if (int rc = check_matrix(w, "d_h", h, h_stride, plan.rows, s->channels, s->dtype, &aligned)) return rc;
    if (int rc = check_matrix(w, "d_dx", dx, dx_stride, plan.rows, s->channels, s->dtype, &aligned)) return rc;
    if (int rc = check_matrix(w, "d_dg", dg, dg_stride, plan.rows, s->channels, s->dtype, &aligned)) return rc;
    if (dx == h || dg == h) return report_failure(TCU_ERR_INVALID_ARG, w + ": a gradient must not take the place of d_h (other tiles still read it)");
    if (dx == dg) return report_failure(TCU_ERR_INVALID_ARG, w + ": d_dx and d_dg are the same buffer");
  }
  if (int rc = check_vector(w, "d_h0", h0, 4, &aligned)) return rc;
  if (int rc = check_vector(w, "d_dh_last", dh_last, 4, &aligned)) return rc;
  if (int rc = check_vector(w, "d_dh0", dh0, 4, &aligned)) return rc;
  const size_t e = element_bytes(s->dtype), n = plan.rows, c = s->channels, states = s->num_sequences;
  const Place pd{"d_dh", dh, dh_stride, n, c, e}, px{"d_x", s->gate == TCU_GATE_SIGMOID ? x : nullptr, x_stride, n, c, e}, pg{"d_g", g, g_stride, n, c, e}, ph{"d_h", h, h_stride, n, c, e},
      p0{"d_h0", h0, c, states, c, 4}, pl{"d_dh_last", dh_last, c, states, c, 4}, odx{"d_dx", dx, dx_stride, n, c, e}, odg{"d_dg", dg, dg_stride, n, c, e}, od0{"d_dh0", dh0, c, states, c, 4};
  if (int rc = check_output_place(w, odx, {pd, px, pg}, {ph, p0, pl, odg, od0})) return rc;
  if (int rc = check_output_place(w, odg, {pd, px, pg}, {ph, p0, pl, od0})) return rc;
  if (int rc = check_output_place(w, od0, {p0, pl}, {pd, px, pg, ph})) return rc;
  if (s->num_sequences == 0 && (plan.rows == 0 || !s->zero_outside)) return TCU_OK;
  GatedScanParams p{};
  p.dh = dh;
  p.dh_stride = dh_stride;
  p.x = x;
  p.x_stride = x_stride;
  p.g = g;
  p.g_stride = g_stride;
  p.h = h;
  p.h_stride = h_stride;
  p.h0 = static_cast<const float *>(h0);
  p.seed = static_cast<const float *>(dh_last);
  p.out = dx;
  p.out_stride = dx_stride;
  p.out_g = dg;
  p.out_g_stride = dg_stride;
  p.last = static_cast<float *>(dh0);
  return run_gated_scan<true>(s, plan, p, aligned, workspace, stream);
}

inline int gated_scan_step_dispatch(int dtype, int gate, size_t channels, size_t rows, const void *x, size_t x_stride, const void *g, size_t g_stride, void *h, size_t h_stride, const void *state,
                                    void *new_state, size_t num_slots, const void *slots, int zero_padding, void *stream) {
  const char *what = "tcu_gated_scan_step";
  const std::string w(what);
  tcu_gated_scan_shape s{};
  s.dtype = dtype;
  s.gate = gate;
  s.channels = channels;
  s.num_sequences = 1;
  s.sequence_length = s.num_rows = rows;
  GatedScanPlan plan;
  if (int rc = plan_gated_scan(what, &s, kScanPlaces, &plan)) return rc;
  if (rows == 0) return TCU_OK;
  if (num_slots == 0 || num_slots >= ((size_t)1 << 31)) return report_failure(TCU_ERR_INVALID_ARG, w + ": num_slots must be 1 ... 2^31 - 1");
  if (!slots && num_slots < rows) return report_failure(TCU_ERR_INVALID_ARG, w + ": fewer slots than rows, and no d_slots to say which");
  if (slots && !aligned_to(slots, 4)) return report_failure(TCU_ERR_INVALID_ARG, w + ": d_slots is not aligned to its integers");
  bool aligned = channels % (16 / element_bytes(dtype)) == 0;
  if (int rc = check_matrix(w, "d_x", x, x_stride, rows, channels, dtype, &aligned)) return rc;
  if (int rc = check_matrix(w, "d_g", g, g_stride, rows, channels, dtype, &aligned)) return rc;
  if (int rc = check_matrix(w, "d_h", h, h_stride, rows, channels, dtype, &aligned)) return rc;
  if (!state || !new_state) return report_failure(TCU_ERR_INVALID_ARG, w + ": d_state or d_new_state is null");
  if (int rc = check_vector(w, "d_state", state, 4, &aligned)) return rc;
  if (int rc = check_vector(w, "d_new_state", new_state, 4, &aligned)) return rc;
  GatedStepParams p{};
  p.x = x;
  p.g = g;
  p.out = h;
  p.state = static_cast<const float *>(state);
  p.new_state = static_cast<float *>(new_state);
  p.slots = static_cast<const int *>(slots);
  p.x_stride = x_stride;
  p.g_stride = g_stride;
  p.out_stride = h_stride;
  p.rows = (unsigned)rows;
  p.num_slots = (unsigned)num_slots;
  p.zero_padding = zero_padding != 0;
  p.channels = (unsigned)channels;
  const size_t per_block = (size_t)kStepThreads * (16 / element_bytes(dtype));
  p.chunks = (unsigned)((channels + per_block - 1) / per_block);
  size_t grid = 0;
  if (!product_fits(rows, p.chunks, &grid) || !launch_fits(grid, kStepThreads)) return report_failure(TCU_ERR_UNSUPPORTED, w + ": rows and channels take more blocks than a launch can have");
  const size_t e = element_bytes(dtype);
  const Place px{"d_x", x, x_stride, rows, channels, e}, pg{"d_g", g, g_stride, rows, channels, e}, ph{"d_h", h, h_stride, rows, channels, e}, ps{"d_state", state, channels, num_slots, channels, 4},
      pn{"d_new_state", new_state, channels, num_slots, channels, 4}, pi{"d_slots", slots, rows, 1, rows, 4};
  if (int rc = check_output_place(w, ph, {px, pg}, {ps, pn, pi})) return rc;
  if (int rc = check_output_place(w, pn, {ps}, {px, pg, pi})) return rc;
#define TCU_STEP(DT_, G_) (aligned ? launch(gated_scan_step_kernel<DT_, G_, true>, (unsigned)grid, (unsigned)kStepThreads, stream, p) : launch(gated_scan_step_kernel<DT_, G_, false>, (unsigned)grid, (unsigned)kStepThreads, stream, p))
#define TCU_STEP_GATES(DT_) (gate == TCU_GATE_DECAY ? TCU_STEP(DT_, kGateDecay) : gate == TCU_GATE_LOG ? TCU_STEP(DT_, kGateLog) : TCU_STEP(DT_, kGateSigmoid))
  if (dtype == TCU_F16) TCU_STEP_GATES(kF16);
  else if (dtype == TCU_BF16) TCU_STEP_GATES(kBF16);
  else TCU_STEP_GATES(kF32);
#undef TCU_STEP_GATES
#undef TCU_STEP
  return TCU_OK;
}

}  // namespace tcu

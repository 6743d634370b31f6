// Builds the recurrent-block operators of tcu_scope_amd/csrc against the CPU lane emulator (TEST INFRASTRUCTURE ONLY).
#include "wave_ops_emu.hpp"
//
#include "block_ops_emu.hpp"
//
#include "../../tcu_scope_amd/csrc/gated_scan_host.hpp"

namespace tcu {
static std::string g_error;
static unsigned g_poll_limit = 1u << 20, g_mute = 0;
int report_failure(int code, const std::string &message) {
  g_error = message;
  return code;
}
unsigned shared_poll_limit() { return g_poll_limit; }
unsigned shared_mute_partition() { return g_mute; }
}  // namespace tcu

extern "C" {
const char *emu_last_error() { return tcu::g_error.c_str(); }
void emu_waits(unsigned poll_limit, unsigned mute) {
  tcu::g_poll_limit = poll_limit;
  tcu::g_mute = mute;
}
int emu_gated_scan(const tcu_gated_scan_shape *s, const void *x, size_t xs, const void *g, size_t gs, void *h, size_t hs, const void *h0, void *h_last, void *ws, size_t *wb) {
  return tcu::gated_scan_dispatch(s, x, xs, g, gs, h, hs, h0, h_last, ws, wb, nullptr);
}
int emu_gated_scan_backward(const tcu_gated_scan_shape *s, const void *dh, size_t dhs, const void *x, size_t xs, const void *g, size_t gs, const void *h, size_t hs, const void *h0, const void *dh_last, void *dx,
                            size_t dxs, void *dg, size_t dgs, void *dh0, void *ws, size_t *wb) {
  return tcu::gated_scan_backward_dispatch(s, dh, dhs, x, xs, g, gs, h, hs, h0, dh_last, dx, dxs, dg, dgs, dh0, ws, wb, nullptr);
}
int emu_gated_scan_step(int dtype, int gate, size_t channels, size_t rows, const void *x, size_t xs, const void *g, size_t gs, void *h, size_t hs, const void *state, void *new_state, size_t num_slots,
                        const void *slots, int zero_padding) {
  return tcu::gated_scan_step_dispatch(dtype, gate, channels, rows, x, xs, g, gs, h, hs, state, new_state, num_slots, slots, zero_padding, nullptr);
}
}
#include "../../tcu_scope_amd/csrc/fused_norm_host.hpp"

extern "C" {
int emu_fused_norm(const tcu_fused_norm_shape *s, const void *x, size_t xs, const void *res, size_t rs, const void *gate, size_t gs, const void *w, const void *b, const void *cs, void *out, size_t os, void *zo,
                   size_t zs) {
  return tcu::fused_norm_dispatch(s, x, xs, res, rs, gate, gs, w, b, cs, out, os, zo, zs, nullptr);
}
int emu_fused_norm_backward(const tcu_fused_norm_shape *s, const void *dout, size_t dos, const void *z, size_t zs, const void *gate, size_t gs, const void *w, const void *b, const void *cs, const void *x,
                            size_t xs, const void *dro, size_t dros, void *dx, size_t dxs, void *dg, size_t dgs, void *dr, size_t drs, float *dw, float *db, float *dcs, void *ws, size_t *wb) {
  return tcu::fused_norm_backward_dispatch(s, dout, dos, z, zs, gate, gs, w, b, cs, x, xs, dro, dros, dx, dxs, dg, dgs, dr, drs, dw, db, dcs, ws, wb, nullptr);
}
}
#include "../../tcu_scope_amd/csrc/fused_gemm_host.hpp"

extern "C" {
int emu_fused_gemm(const tcu_fused_gemm_shape *s, const void *A, size_t lda, const void *B, size_t ldb, const void *bias, const void *C, size_t ldc, void *D, size_t ldd, void *Z, size_t ldz, void *ws, size_t *wb) {
  return tcu::fused_gemm_dispatch(s, A, lda, B, ldb, bias, C, ldc, D, ldd, Z, ldz, ws, wb, nullptr);
}
int emu_fused_gemm_backward(const tcu_fused_gemm_shape *s, const void *dD, size_t lddd, const void *A, size_t lda, const void *B, size_t ldb, const void *Z, size_t ldz, void *dA, size_t ldda, void *dB,
                            size_t lddb, float *dbias, void *ws, size_t *wb) {
  return tcu::fused_gemm_backward_dispatch(s, dD, lddd, A, lda, B, ldb, Z, ldz, dA, ldda, dB, lddb, dbias, ws, wb, nullptr);
}
}

namespace {
template <int DT, int W8>
void emu_tiles(tcu::FusedGemmParams p) {
  const size_t tile = 32 * W8;
  p.tiles = (unsigned)((p.M + tile - 1) / tile * ((p.N + tile - 1) / tile));
  if (p.K % 64) tcu::launch(tcu::fused_gemm_tile_kernel<DT, false, W8, true>, p.tiles * p.splits, 256u, nullptr, p);
  else tcu::launch(tcu::fused_gemm_tile_kernel<DT, false, W8, false>, p.tiles * p.splits, 256u, nullptr, p);
  if (p.splits > 1) tcu::launch(tcu::fused_gemm_join_kernel<DT, false>, (unsigned)((p.M * (p.share_ld / 8) + 255) / 256), 256u, nullptr, p);
}
template <int DT, int W8, int LAYOUT>
void emu_down(tcu::FusedGemmParams p) {
  const size_t tile = 32 * W8;
  p.tiles = (unsigned)((p.M + tile - 1) / tile * ((p.N + tile - 1) / tile));
  tcu::launch(tcu::fused_gemm_tile_kernel<DT, true, W8, true, LAYOUT>, p.tiles * p.splits, 256u, nullptr, p);
  if (p.splits > 1) tcu::launch(tcu::fused_gemm_join_kernel<DT, true>, (unsigned)((p.M * (p.share_ld / 8) + 255) / 256), 256u, nullptr, p);
}
}  // namespace

extern "C" {
// the same with K down the rows of B (layout 1) or of both operands (2)
int emu_fused_gemm_down(int w8, int layout, unsigned splits, int dtype, size_t M, size_t N, size_t K, const void *A, size_t lda, const void *B, size_t ldb, void *D, size_t ldd, float *shares) {
  tcu::FusedGemmParams p{};
  p.A = A; p.lda = lda; p.B = B; p.ldb = ldb; p.D = D; p.ldd = ldd; p.M = M; p.N = N; p.K = K; p.splits = splits; p.share_ld = tcu::up_to(N, 8);
  p.shares = splits > 1 ? shares : nullptr;
#define EMU_DOWN(DT, W8) (layout == 1 ? emu_down<DT, W8, tcu::kDownB>(p) : emu_down<DT, W8, tcu::kDownBoth>(p))
  if (dtype == TCU_F16) w8 == 8 ? EMU_DOWN(tcu::kF16, 8) : w8 == 6 ? EMU_DOWN(tcu::kF16, 6) : EMU_DOWN(tcu::kF16, 4);
  else w8 == 8 ? EMU_DOWN(tcu::kBF16, 8) : w8 == 6 ? EMU_DOWN(tcu::kBF16, 6) : EMU_DOWN(tcu::kBF16, 4);
#undef EMU_DOWN
  return 0;
}
// the tile kernels at sizes at which the library would not take them; rows of A and B begin on 16 bytes, K is at least 64 for every split
int emu_fused_gemm_tiles(int w8, unsigned splits, int dtype, int act, size_t M, size_t N, size_t K, float beta, const void *A, size_t lda, const void *B, size_t ldb, const void *bias, const void *C, size_t ldc,
                         void *D, size_t ldd, void *Z, size_t ldz, float *shares) {
  tcu::FusedGemmParams p{};
  p.A = A; p.lda = lda; p.B = B; p.ldb = ldb; p.bias = bias; p.C = C; p.ldc = ldc; p.D = D; p.ldd = ldd; p.Z = Z; p.ldz = ldz;
  p.M = M; p.N = N; p.K = K; p.beta = beta; p.act = act; p.splits = splits; p.share_ld = tcu::up_to(N, 8);
  p.shares = splits > 1 ? shares : nullptr;
  if (dtype == TCU_F16) w8 == 8 ? emu_tiles<tcu::kF16, 8>(p) : w8 == 6 ? emu_tiles<tcu::kF16, 6>(p) : emu_tiles<tcu::kF16, 4>(p);
  else w8 == 8 ? emu_tiles<tcu::kBF16, 8>(p) : w8 == 6 ? emu_tiles<tcu::kBF16, 6>(p) : emu_tiles<tcu::kBF16, 4>(p);
  return 0;
}
}

// which kernels the library takes
extern "C" {
int emu_scan_threads(const tcu_gated_scan_shape *s, int back) {
  tcu::GatedScanPlan plan;
  return tcu::plan_gated_scan("plan", s, back ? tcu::kScanBackPlaces : tcu::kScanPlaces, &plan) == 0 ? plan.threads : 0;
}
// layout: 0 K along the rows of both operands, 1 down the rows of B, 2 down those of both; 0 for the form of few rows, else tiles of 32 times the result
int emu_gemm_tile(size_t M, size_t N, size_t K, int layout, size_t *splits) {
  const tcu::GemmPlan g = tcu::plan_gemm(M, N, K, layout);
  *splits = g.splits;
  return g.few_rows ? 0 : g.w8;
}
}

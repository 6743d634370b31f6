// Argument checks, workspace layout and kernel selection of the fused product's entry points.
#pragma once

#include <utility>

#include "checks.hpp"
#include "column_sum.hpp"
#include "fused_gemm.hpp"
#include "launch.hpp"

namespace tcu {

// Up to this many rows the product is bound by reading B.  Beyond it every block reading all of A costs more than the tile
// kernels' empty rows (33 x 8192 x 4096 bf16: 31.7 us, tiles with split K 18.5; 16 x 4096 x 8192: 20.6).
constexpr size_t kGemmFewRows = 32;
constexpr size_t kGemmMaxInner = (size_t)1 << 22; // a tile's rows of an operand lie within 32-bit byte offsets: 256 * 2^22 * 2 < 2^32

constexpr size_t kGemmMaxLd = (size_t)1 << 28;    // 8 rows of an output lie within 32-bit offsets

inline size_t up_to(size_t n, size_t step) { return (n + step - 1) / step * step; }
// bytes of a part of a workspace
inline size_t part_bytes(size_t bytes) { return up_to(bytes, 256); }

// How one product M x N over K runs, and what it takes of the workspace.
struct GemmPlan {
  bool few_rows = false;
  int few_tiles = 1;  // few rows: 16-row tiles
  int w8 = 8;         // block tiles of 32 w8 rows and columns
  int layout = kAlong;
  size_t tiles = 0, splits = 1;
  size_t share_ld = 0, share_bytes = 0;
};
// The time of a tiling in microseconds: rounds of blocks over the compute units, each as long as its K steps (64 elements)
// plus what a block spends before and after them, and the pass that joins split sums.  Measured with 8192 x 8192 x 4096 and
// 4001 x 2056 x 4096 bf16: a step of a 256 x 256 tile takes a compute unit 1.5 us, of 192 x 192 0.9, and of two 128 x 128
// tiles side by side 0.95; and with few steps, i.e. mostly what stands around them: 256 | 192 | 128 tiles 7616 x 4120 x 130 40 | 52 | 34 us,
// 8192 x 8192 x 200 79 | 107 | 71, 4032 x 3112 x 283 24 | 30 | 22.
inline double gemm_tiling_us(size_t tiles, size_t splits, int w8, size_t M, size_t N, size_t K) {
  const double step = w8 == 8 ? 1.5 : w8 == 6 ? 0.9 : 0.95, around = w8 == 8 ? 15.0 : w8 == 6 ? 10.0 : 5.5;
  const size_t at_once = w8 == 4 ? 512 : 256, blocks = tiles * splits;
  const double steps = (double)((K + 63) / 64 + splits - 1) / (double)splits;
  const double alone = w8 == 4 && blocks <= 256 ? 0.65 : 1.0;  // a 128 x 128 tile that has its compute unit to itself
  double us = (double)((blocks + at_once - 1) / at_once) * (steps * step * alone + around);
  if (splits > 1) us += 5.0 + (double)splits * (double)M * (double)N * 8.0 / 4.0e6;
  return us;
}
inline GemmPlan plan_gemm(size_t M, size_t N, size_t K, int layout = kAlong) {
  GemmPlan g;
  g.layout = layout;
  g.share_ld = up_to(N, 8);
  if (M <= kGemmFewRows && layout == kAlong) {
    g.few_rows = true;
    g.few_tiles = M <= 16 ? 1 : 2;
    g.tiles = (N + 15) / 16;
    // a block per compute unit: below that the waves of one compute unit cannot keep its share of the memory's bandwidth in flight
    const size_t steps = K / 1024;
    while (g.tiles * g.splits < 256 && g.splits * 2 <= steps) g.splits *= 2;
  } else {
    double best = 0.0;
    for (int w8 : {8, 6, 4}) {
      const size_t t = 32 * (size_t)w8, tiles = (M + t - 1) / t * ((N + t - 1) / t);
      for (size_t splits = 1; splits <= 16 && (splits == 1 || (splits * 4 <= K / 64 && tiles * splits <= 512)); splits++) {
        const double us = gemm_tiling_us(tiles, splits, w8, M, N, K);
        if (g.tiles != 0 && us >= best) continue;
        best = us;
        g.w8 = w8;
        g.tiles = tiles;
        g.splits = splits;
      }
    }
  }
  if (g.splits > 1) g.share_bytes = part_bytes(g.splits * M * g.share_ld * 4);
  return g;
}

// One product on operands that are ready for it.
template <int DT, bool WHOLE>
inline void launch_gemm(const GemmPlan &g, FusedGemmParams p, float *shares, bool whole_inner, void *stream) {
  p.splits = (unsigned)g.splits;
  p.tiles = (unsigned)g.tiles;
  p.share_ld = g.share_ld;
  p.shares = g.splits > 1 ? shares : nullptr;
  const unsigned grid = (unsigned)(g.tiles * g.splits);
  if (p.K == 0) {  // nothing to add up: the epilogue over a sum of no shares
    p.splits = 0;
  } else if (g.few_rows) {
#define TCU_FEW(MT, UNROLL) \
  (WHOLE && whole_inner ? launch(fused_gemm_few_rows_kernel<DT, WHOLE, MT, 8, UNROLL>, grid, 512u, stream, p) : launch(fused_gemm_few_rows_kernel<DT, false, MT, 8, UNROLL>, grid, 512u, stream, p))
    if (g.few_tiles == 1) TCU_FEW(1, 4);
    else TCU_FEW(2, 4);
#undef TCU_FEW
  } else {
#define TCU_TILE(W8, TAIL, LAYOUT) launch(fused_gemm_tile_kernel<DT, WHOLE || LAYOUT != kAlong, W8, TAIL, LAYOUT>, grid, 256u, stream, p)
#define TCU_TILES(TAIL, LAYOUT) (g.w8 == 8 ? TCU_TILE(8, TAIL, LAYOUT) : g.w8 == 6 ? TCU_TILE(6, TAIL, LAYOUT) : TCU_TILE(4, TAIL, LAYOUT))
    if (g.layout == kDownB) TCU_TILES(true, kDownB);  // taken for whole chunks only
    else if (g.layout == kDownBoth) TCU_TILES(true, kDownBoth);
    else if (p.K % 64) TCU_TILES(true, kAlong);
    else TCU_TILES(false, kAlong);
#undef TCU_TILE
#undef TCU_TILES
  }
  if (p.splits != 1) launch(fused_gemm_join_kernel<DT, WHOLE>, (unsigned)((p.M * (g.share_ld / 8) + 255) / 256), 256u, stream, p);
}
inline void run_gemm(int dtype, bool whole, const GemmPlan &g, const FusedGemmParams &p, float *shares, bool whole_inner, void *stream) {
  if (dtype == TCU_F16) {
    if (whole) launch_gemm<kF16, true>(g, p, shares, whole_inner, stream);
    else launch_gemm<kF16, false>(g, p, shares, whole_inner, stream);
  } else {
    if (whole) launch_gemm<kBF16, true>(g, p, shares, whole_inner, stream);
    else launch_gemm<kBF16, false>(g, p, shares, whole_inner, stream);
  }
}

// rows of 16 bits that the transfers of the tile kernel can take as they are
inline bool rows_ready(const void *p, size_t ld) { return aligned_to(p, 16) && ld % 8 == 0 && ld <= kGemmMaxInner; }

inline int check_gemm_shape(const std::string &w, const tcu_fused_gemm_shape *s) {
  if (!s) return report_failure(TCU_ERR_INVALID_ARG, w + ": null shape");
  if (s->dtype != TCU_F16 && s->dtype != TCU_BF16) return report_failure(TCU_ERR_INVALID_ARG, w + ": dtype must be TCU_F16 or TCU_BF16");
  if (!known_activation(s->activation)) return report_failure(TCU_ERR_INVALID_ARG, w + ": unknown activation");
  if (s->M >= (size_t)1 << 31 || s->N > kGemmMaxLd || s->K > kGemmMaxInner) return report_failure(TCU_ERR_UNSUPPORTED, w + ": M from 2^31 on, N above 2^28, or K above 2^22");
  return TCU_OK;
}
inline int check_output(const std::string &w, const char *name, const void *p, size_t ld, size_t rows, size_t width, int dtype, bool *whole) {
  if (ld > kGemmMaxLd) return report_failure(TCU_ERR_UNSUPPORTED, w + ": the leading dimension of " + name + " is above 2^28");
  return check_matrix(w, name, p, ld, rows, width, dtype, whole);
}
// a launch with one thread for each chunk of 8 elements of a matrix
inline int check_gemm_grid(const std::string &w, size_t M, size_t N) {
  size_t chunks = 0;
  if (!product_fits(M, up_to(N, 8) / 8, &chunks) || !launch_fits((chunks + 255) / 256, 256)) return report_failure(TCU_ERR_UNSUPPORTED, w + ": a matrix of 2^35 elements or more");
  return TCU_OK;
}
inline int check_gemm_tiles(const std::string &w, const GemmPlan &g) {
  if (!launch_fits(g.tiles * g.splits, g.few_rows ? 512 : 256)) return report_failure(TCU_ERR_UNSUPPORTED, w + ": the output takes more tiles than a launch can have");
  return TCU_OK;
}

// padded: a multiple of 8 from the width up to to_ld; the rows end in zeros up to there
inline void pack_rows(const void *from, size_t from_ld, void *to, size_t to_ld, size_t rows, size_t width, size_t padded, void *stream) {
  const PackRowsParams q{static_cast<const uint16_t *>(from), static_cast<uint16_t *>(to), rows, width, padded, from_ld, to_ld};
  launch(pack_rows_kernel, (unsigned)((rows * (padded / 8) + 255) / 256), 256u, stream, q);
}

inline int fused_gemm_dispatch(const tcu_fused_gemm_shape *s, const void *A, size_t lda, const void *B, size_t ldb, const void *bias, const void *C, size_t ldc, void *D, size_t ldd, void *Z, size_t ldz,
                               void *workspace, size_t *workspace_bytes, void *stream) {
  const std::string w("tcu_fused_gemm");
  if (int rc = check_gemm_shape(w, s)) return rc;
  if (int rc = check_gemm_grid(w, s->M, s->N)) return rc;
  const size_t M = s->M, N = s->N, K = s->K;
  const GemmPlan g = plan_gemm(M, N, K);
  if (int rc = check_gemm_tiles(w, g)) return rc;
  const bool few_k = K > 0 && K < 64;  // the tile kernels want a whole step
  const bool odd_k = few_k || K % 8 != 0;     // nor a part of a chunk
  const bool pack_a = !g.few_rows && K && (odd_k || !rows_ready(A, M > 1 ? lda : 8)), pack_b = !g.few_rows && K && (odd_k || !rows_ready(B, N > 1 ? ldb : 8));
  if (pack_a)
    if (int rc = check_gemm_grid(w, M, K)) return rc;
  if (pack_b)
    if (int rc = check_gemm_grid(w, N, K)) return rc;
  const size_t ldk = few_k ? 64 : up_to(K, 8), a_bytes = pack_a ? part_bytes(M * ldk * 2) : 0, b_bytes = pack_b ? part_bytes(N * ldk * 2) : 0;
  const size_t bytes = g.share_bytes + a_bytes + b_bytes, need = smallest_workspace(bytes);
  if (!workspace_bytes) return report_failure(TCU_ERR_INVALID_ARG, w + ": workspace_bytes is null");
  if (!workspace) {
    *workspace_bytes = need;
    return TCU_OK;
  }
  if (int rc = check_workspace(w, workspace, *workspace_bytes, need)) return rc;
  if (M == 0 || N == 0) return TCU_OK;
  const bool use_c = s->beta != 0.0f;
  if (use_c && !C) return report_failure(TCU_ERR_INVALID_ARG, w + ": beta without d_C");
  bool whole = N % 8 == 0, whole_inner = K % 8 == 0;
  if (K)
    if (int rc = check_matrix(w, "d_A", A, lda, M, K, s->dtype, &whole_inner)) return rc;
  if (K)
    if (int rc = check_matrix(w, "d_B", B, ldb, N, K, s->dtype, &whole_inner)) return rc;
  if (int rc = check_output(w, "d_D", D, ldd, M, N, s->dtype, &whole)) return rc;
  if (int rc = use_c ? check_output(w, "d_C", C, ldc, M, N, s->dtype, &whole) : TCU_OK) return rc;
  if (int rc = Z ? check_output(w, "d_Z", Z, ldz, M, N, s->dtype, &whole) : TCU_OK) return rc;
  if (int rc = check_vector(w, "d_bias", bias, 2, &whole)) return rc;
  if (D == A || D == B || D == Z || (Z && (Z == A || Z == B || (use_c && Z == C)))) return report_failure(TCU_ERR_INVALID_ARG, w + ": an output in the place of an operand other tiles still read, or of another output");
  const Place pa{"d_A", A, lda, M, K, 2}, pb{"d_B", B, ldb, N, K, 2}, pbias{"d_bias", bias, 0, 1, N, 2}, pc{"d_C", use_c ? C : nullptr, ldc, M, N, 2}, pd{"d_D", D, ldd, M, N, 2}, pz{"d_Z", Z, ldz, M, N, 2};
  if (int rc = check_output_place(w, pd, {pc}, {pa, pb, pbias, pz})) return rc;
  if (int rc = check_output_place(w, pz, {}, {pa, pb, pbias, pc})) return rc;
  char *at = static_cast<char *>(workspace) + g.share_bytes;
  FusedGemmParams p{};
  p.A = A;
  p.lda = lda;
  if (pack_a) {
    pack_rows(A, lda, at, ldk, M, K, few_k ? 64 : up_to(K, 8), stream);
    p.A = at;
    p.lda = ldk;
    at += a_bytes;
  }
  p.B = B;
  p.ldb = ldb;
  if (pack_b) {
    pack_rows(B, ldb, at, ldk, N, K, few_k ? 64 : up_to(K, 8), stream);
    p.B = at;
    p.ldb = ldk;
  }
  p.bias = bias;
  p.C = use_c ? C : nullptr;
  p.ldc = ldc;
  p.D = D;
  p.ldd = ldd;
  p.Z = Z;
  p.ldz = ldz;
  p.M = M;
  p.N = N;
  p.K = !g.few_rows && odd_k ? ldk : K;
  p.beta = s->beta;
  p.act = s->activation;
  run_gemm(s->dtype, whole, g, p, static_cast<float *>(workspace), whole_inner, stream);
  return TCU_OK;
}

inline int fused_gemm_backward_dispatch(const tcu_fused_gemm_shape *s, const void *dD, size_t lddd, const void *A, size_t lda, const void *B, size_t ldb, const void *Z, size_t ldz, void *dA, size_t ldda,
                                        void *dB, size_t lddb, float *dbias, void *workspace, size_t *workspace_bytes, void *stream) {
  const std::string w("tcu_fused_gemm_backward");
  if (int rc = check_gemm_shape(w, s)) return rc;
  const size_t M = s->M, N = s->N, K = s->K;
  if (M > kGemmMaxInner || N > kGemmMaxInner) return report_failure(TCU_ERR_UNSUPPORTED, w + ": M or N above 2^22");
  size_t tiles = 0;  // of 64 x 64 elements, of all that may have to be laid out anew in one launch
  for (auto mn : {std::make_pair(M, N), std::make_pair(M, K), std::make_pair(N, K)}) {
    if (int rc = check_gemm_grid(w, mn.first, mn.second)) return rc;
    tiles += (mn.first + 63) / 64 * ((mn.second + 63) / 64);
  }
  if (!launch_fits(tiles, 256)) return report_failure(TCU_ERR_UNSUPPORTED, w + ": the matrices take more tiles than a launch can have");
  const bool act = s->activation != TCU_ACT_NONE;
  if (act && !Z) return report_failure(TCU_ERR_INVALID_ARG, w + ": the gradient of an activation needs d_Z");
  // the copies' rows end in zeros up to a whole step of the tile kernels
  const size_t ldm = up_to(M, 64), ldn = up_to(N, 64);
  // the operands along whose rows the sums do not run, as they are: whole chunks, and a whole step of rows at least
  // (also where M is small enough for the few-row kernel, which would need B turned: 20 x 8192 x 8192 bf16 83 us, turned 149;
  // 8 x 4096 x 4096 39 | 37)
  const bool down_a = dA && N >= 64 && K % 8 == 0 && rows_ready(B, ldb) && rows_ready(dA, M > 1 ? ldda : 8);
  const bool down_b = dB && M >= 64 && K % 8 == 0 && rows_ready(A, lda) && rows_ready(dB, N > 1 ? lddb : 8);
  const GemmPlan ga = plan_gemm(M, K, N, down_a ? kDownB : kAlong), gb = plan_gemm(N, K, M, down_b ? kDownBoth : kAlong);
  if (int rc = dA ? check_gemm_tiles(w, ga) : TCU_OK) return rc;
  if (int rc = dB ? check_gemm_tiles(w, gb) : TCU_OK) return rc;
  // the gradient of the activation's argument: dD itself where there is no activation and its rows are ready
  const bool own_dz = (dA || down_b) && (act || N % (dA && !down_a ? 64 : 8) != 0 || !rows_ready(dD, M > 1 ? lddd : 8));
  const bool turn_a = dB && !down_b, turn_b = dA && !down_a;  // A and dZ; B
  const size_t dz_bytes = own_dz ? part_bytes(M * ldn * 2) : 0, dzt_bytes = turn_a ? part_bytes(N * ldm * 2) : 0, at_bytes = turn_a ? part_bytes(K * ldm * 2) : 0, bt_bytes = turn_b ? part_bytes(K * ldn * 2) : 0;
  const size_t strips = (M + 63) / 64, sums_bytes = dbias ? part_bytes(strips * N * 4) : 0;
  const size_t share_bytes = (dA ? ga.share_bytes : 0) > (dB ? gb.share_bytes : 0) ? ga.share_bytes : (dB ? gb.share_bytes : 0);
  const size_t bytes = share_bytes + dz_bytes + dzt_bytes + at_bytes + bt_bytes + sums_bytes, need = smallest_workspace(bytes);
  if (!workspace_bytes) return report_failure(TCU_ERR_INVALID_ARG, w + ": workspace_bytes is null");
  if (!workspace) {
    *workspace_bytes = need;
    return TCU_OK;
  }
  if (int rc = check_workspace(w, workspace, *workspace_bytes, need)) return rc;
  bool ignored = true, whole_a = K % 8 == 0, whole_b = K % 8 == 0;
  if (M && N)
    if (int rc = check_matrix(w, "d_dD", dD, lddd, M, N, s->dtype, &ignored)) return rc;
  if (M && N && act)
    if (int rc = check_matrix(w, "d_Z", Z, ldz, M, N, s->dtype, &ignored)) return rc;
  if (dB && M && K)
    if (int rc = check_matrix(w, "d_A", A, lda, M, K, s->dtype, &ignored)) return rc;
  if (dA && N && K)
    if (int rc = check_matrix(w, "d_B", B, ldb, N, K, s->dtype, &ignored)) return rc;
  if (dA && M && K)
    if (int rc = check_output(w, "d_dA", dA, ldda, M, K, s->dtype, &whole_a)) return rc;
  if (dB && N && K)
    if (int rc = check_output(w, "d_dB", dB, lddb, N, K, s->dtype, &whole_b)) return rc;
  if (int rc = check_vector(w, "d_dbias", dbias, 4, &ignored)) return rc;
  if ((dA && (dA == dD || dA == A || dA == B || dA == Z || dA == dB)) || (dB && (dB == dD || dB == A || dB == B || dB == Z)))
    return report_failure(TCU_ERR_INVALID_ARG, w + ": a gradient in the place of an operand, or of another gradient");
  const Place pd{"d_dD", dD, lddd, M, N, 2}, pz{"d_Z", act ? Z : nullptr, ldz, M, N, 2}, pa{"d_A", dB ? A : nullptr, lda, M, K, 2}, pb{"d_B", dA ? B : nullptr, ldb, N, K, 2}, oa{"d_dA", dA, ldda, M, K, 2},
      ob{"d_dB", dB, lddb, N, K, 2}, obias{"d_dbias", dbias, 0, 1, N, 4};
  if (int rc = check_output_place(w, oa, {}, {pd, pz, pa, pb, ob, obias})) return rc;
  if (int rc = check_output_place(w, ob, {}, {pd, pz, pa, pb, obias})) return rc;
  if (int rc = check_output_place(w, obias, {}, {pd, pz, pa, pb})) return rc;
  char *at = static_cast<char *>(workspace) + share_bytes;
  auto take = [&](size_t n) {
    char *q = at;
    at += n;
    return static_cast<void *>(q);
  };
  void *dz = take(dz_bytes), *dzt = take(dzt_bytes), *a_t = take(at_bytes), *b_t = take(bt_bytes);
  float *sums = static_cast<float *>(take(sums_bytes));
  float *shares = static_cast<float *>(workspace);
  TransposeParams q{};
  auto job = [&](int i, const void *from, size_t from_ld, void *to, size_t to_ld, size_t rows, size_t columns) {
    const unsigned column_tiles = (unsigned)((columns + 63) / 64);
    q.job[i] = TransposeJob{from, to, rows, columns, from_ld, to_ld, column_tiles, (unsigned)((rows + 63) / 64 * column_tiles)};
  };
  if (M && N && (own_dz || turn_a || dbias)) job(0, dD, lddd, turn_a ? dzt : nullptr, ldm, M, N);
  if (turn_a && M && K) job(1, A, lda, a_t, ldm, M, K);
  if (turn_b && N && K) job(2, B, ldb, b_t, ldn, N, K);
  q.Z = act ? Z : nullptr;
  q.z_ld = ldz;
  q.dz = own_dz ? dz : nullptr;
  q.dz_ld = ldn;
  q.partial = dbias ? sums : nullptr;
  q.act = s->activation;
  if (const unsigned grid = q.job[0].tiles + q.job[1].tiles + q.job[2].tiles) {
    if (s->dtype == TCU_F16) launch(gradient_layout_kernel<kF16>, grid, 256u, stream, q);
    else launch(gradient_layout_kernel<kBF16>, grid, 256u, stream, q);
  }
  if (dbias && N) {
    ColumnSumParams q{};
    q.partial = sums;
    q.out[0] = dbias;
    q.parts = strips;
    q.columns = (unsigned)N;
    q.vectors = 1;
    launch(column_sum_kernel, (unsigned)((N + 63) / 64), 64u * kColumnSumWaves, stream, q);
  }
  FusedGemmParams p{};
  p.act = TCU_ACT_NONE;
  p.N = K;
  if (dA && M && K) {
    p.A = own_dz ? dz : dD;
    p.lda = own_dz ? ldn : lddd;
    p.B = down_a ? B : b_t;
    p.ldb = down_a ? ldb : ldn;
    p.D = dA;
    p.ldd = ldda;
    p.M = M;
    p.K = down_a ? N : ldn;
    run_gemm(s->dtype, whole_a, ga, p, shares, true, stream);
  }
  if (dB && N && K) {
    p.A = !down_b ? dzt : own_dz ? dz : dD;
    p.lda = !down_b ? ldm : own_dz ? ldn : lddd;
    p.B = down_b ? A : a_t;
    p.ldb = down_b ? lda : ldm;
    p.D = dB;
    p.ldd = lddb;
    p.M = N;
    p.K = down_b ? M : ldm;
    run_gemm(s->dtype, whole_b, gb, p, shares, true, stream);
  }
  return TCU_OK;
}

}  // namespace tcu

// Matrix product with its epilogue, in fp16 or bf16:  D = act(A B + bias) + beta C,  and Z = A B + bias where a backward
// pass will want it.  A: M x K row-major, B: K x N given as N rows of K (a weight matrix as models hold it), bias: N.
//
// Gradient: dZ = dD * act'(Z) element by element, dA = dZ B^T (M x K), dB = dZ^T A (N rows of K), dbias = the column sums of
// dZ, dC = beta dD.  The two products sum over N and over M, along which B and A (and dZ for the second) are not contiguous:
// the tile kernel takes such operands as they are, rows of K one below the other, and turns them on the way from LDS to registers.
// Where their rows are no whole chunks, or fewer than a step, it runs on transposed copies in the workspace instead.  One launch
// writes those, dZ, and its column sums.
//
//   fused_gemm_tile_kernel : many rows.  256 x 256, 192 x 192 or 128 x 128 block tiles on 16x16x32 MFMAs, K steps of 64, operands
//                moved global -> LDS by transfers that run two steps ahead (three buffers for A, two for B; three for B too where
//                they fit), the loop of gemm_dlds_a3b2_m16_kernel.  M and N may be anything (rows beyond the last one are read
//                as the last one and not stored), K a multiple of 8 (a step with what is left of K goes through registers,
//                zero-filled; operands of another K are copied to padded rows first).
//                Bound by the matrix unit: 8192 x 8192 x 4096 bf16 with bias, silu and Z 431 us = 1.28 PFLOP/s.
//                Where the tiles are fewer than the compute units, several blocks share a tile's K steps and
//                fused_gemm_join_kernel adds their fp32 shares in a fixed order.
//   fused_gemm_few_rows_kernel : up to 32 rows.  Bound by reading B once: a block takes 16 columns of the output and all rows,
//                its waves share K and meet in LDS.  5 x 4096 x 8192 fp16 (67 MB) 16 us = 4.1 TB/s, launch included.
//   gradient_layout_kernel : dZ and what has to be transposed, bound by HBM traffic.  4001 x 4096 x 2056 bf16 with silu: 17 us, and the
//                products 74 and 77 (0.9 PFLOP/s); on transposed copies 38, 67 and 66.  Whole calls with silu and bias: 4001 x 4096 x 2056
//                161 us, 8192 x 8192 x 2048 490 (389 without an activation), 130 x 7616 x 4120 70, 20 x 8192 x 8192 82.
// Sums are fp32; the epilogue is applied to the fp32 sum and each result rounded once.  dZ is rounded to the operands' type,
// because the matrix unit takes operands of 16 bits; its column sums are taken before that.  dA and dB are 1.4 times as far from the
// formula as their own rounding alone leaves them (4001 x 4096 x 2056 bf16: 0.0023 of their norm, where one rounding is 0.0017); two
// products with dZ in two parts would halve the rate for that.
#pragma once

#include "elements.hpp"
#include "gemm.hpp"

namespace tcu {

struct FusedGemmParams {
  const void *A, *B, *bias, *C;  // bias, C may be null
  void *D, *Z;                   // Z may be null
  size_t lda, ldb, ldc, ldd, ldz;
  size_t M, N, K;
  float beta;
  int act;
  float *shares;           // null: the blocks finish their tiles; else raw sums, [split][M][share_ld]
  size_t share_ld;
  unsigned splits, tiles;  // blocks: splits * tiles, the splits of K outermost
};

// z = sum + bias, d = act(z) + beta c for the 8 columns at (row + lane_row, col + lane_col), of which `count` exist; row and col are
// the same for the whole wave, so that a lane's address is a scalar base and one offset per matrix.
template <int DT, bool WHOLE>
TCU_DEVICE void fused_gemm_finish(const FusedGemmParams &p, size_t row, size_t col, unsigned lane_row, unsigned lane_col, int count, float (&v)[8], const float (&bias)[8]) {
  auto base = [&](const void *q, size_t ld) { return static_cast<const uint16_t *>(q) + row * ld + col; };
  auto offset = [&](size_t ld) { return lane_row * (unsigned)ld + lane_col; };
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] += bias[e];
  if (p.Z) store_chunk_of<DT, WHOLE>(const_cast<uint16_t *>(base(p.Z, p.ldz)), offset(p.ldz), count, v);
  activate<false>(p.act, v);
  if (p.C) {
    float c[8];
    unpack_chunk<DT>(load_chunk_of<DT, WHOLE>(base(p.C, p.ldc), offset(p.ldc), count), c);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = __builtin_fmaf(p.beta, c[e], v[e]);
  }
  store_chunk_of<DT, WHOLE>(const_cast<uint16_t *>(base(p.D, p.ldd)), offset(p.ldd), count, v);
}

// One block tile (W8 = 8: 256 x 256, 6: 192 x 192, 4: 128 x 128; waves of 16 W8 x 16 W8).  Rows of A and B begin on 16 bytes; a tile's
// rows of either lie within 4 GiB.  A 192 x 192 tile has room for three buffers of B as well: the tiles of step s + 3 go out
// behind the barrier of step s, into its buffers, and have two steps to arrive.  The product is formed transposed (B fragment first), so a lane owns row (lane & 15)
// and four adjacent columns of every 16 x 16 tile.
constexpr int kAlong = 0, kDownB = 1, kDownBoth = 2;  // LAYOUT: K along the rows of both operands, down the rows of B, of both
// Where a tile of 16 U columns and 64 rows of K holds its 32-byte unit u of row k in LDS.  Two groups of 16 lanes read at a time, rows
// 8 g + 4 h + 0 ... 3 of two neighbouring g; the units of one column in those 8 rows lie in different banks (U = 12: in four of
// twelve columns pairs of them share banks).  Its own inverse.
template <unsigned U>
TCU_DEVICE unsigned unit_place(unsigned k, unsigned u) {
  const unsigned odd = (k >> 3) & 1;
  if constexpr (U == 12) return ((u & 3) ^ (k & 3)) | (((u >> 2) < 2 ? (u >> 2) ^ odd : u >> 2) << 2);
  return u ^ ((k & 3) | odd << 2);
}

template <int DT, bool WHOLE, int W8, bool TAIL, int LAYOUT>
TCU_DEVICE void fused_gemm_tile(const FusedGemmParams &p, size_t tile_m, size_t tile_n, size_t step0, size_t steps, bool tail, float *share) {
  constexpr int BK = 64, ROWH = BK, CPR = 8, RPT = 8, RS = 1, SUB = 2, NA = 3, NB = W8 == 6 ? 3 : 2;
  constexpr int TILE = 32 * W8, WT = 16 * W8;
  constexpr int NM = W8 * W8;
  constexpr int OPH = TILE * ROWH;
  constexpr int TPW = TILE / RPT / 4;
  constexpr int TEVERY = NM / 2 / TPW;
  constexpr bool BF16 = DT == kBF16;
  static_assert((W8 == 8 || W8 == 6 || W8 == 4) && 4 * W8 <= NM && (NM / 2) % TPW == 0, "fragment reads and transfers must fit a substep");
  __shared__ __attribute__((aligned(1024))) half_t lds_a[NA][OPH];
  __shared__ __attribute__((aligned(1024))) half_t lds_b[NB][OPH];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave >> 1, wn = wave & 1;
  const size_t row0 = tile_m * TILE, col0 = tile_n * TILE;
  constexpr bool DOWN_A = LAYOUT == kDownBoth, DOWN_B = LAYOUT != kAlong;
  constexpr unsigned UNITS = 2 * W8, CHUNKS = 2 * UNITS;  // of a row of the tile of an operand whose K runs down the rows
  // the last row of the tile that exists; of an operand whose K runs down the rows, where the last chunk of 8 columns begins
  auto last_of = [](size_t left, bool down) { return down ? (unsigned)((left < TILE ? left : TILE) + 7) / 8 * 8 - 8 : (unsigned)(left < TILE ? left : TILE) - 1; };
  const unsigned last_a = last_of(p.M - row0, DOWN_A), last_b = last_of(p.N - col0, DOWN_B);
  const char *A = static_cast<const char *>(p.A) + row0 * (DOWN_A ? 1 : p.lda) * 2, *B = static_cast<const char *>(p.B) + col0 * (DOWN_B ? 1 : p.ldb) * 2;

  float4_t acc[W8][W8];
#pragma unroll
  for (int i = 0; i < W8; i++)
#pragma unroll
    for (int j = 0; j < W8; j++) {
      // (of 192 x 192 tiles the compiler keeps known zeros apart from the loop's values, and copies those every step)
      if constexpr (W8 == 6 && !TAIL) acc[i][j] = opaque_zero();
      else acc[i][j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }

  const int frow = lane & 15, kq = lane >> 4, fsw = (frow >> RS) & (CPR - 1);
  const int fa0 = (wm * WT + frow) * ROWH, fb0 = (wn * WT + frow) * ROWH;
  int ko[SUB];
#pragma unroll
  for (int kk = 0; kk < SUB; kk++) ko[kk] = ((4 * kk + kq) ^ fsw) * 8;
  // operands whose K runs down the rows: the lane's piece of unit w W8 + i
  int da[W8], db[W8];
#pragma unroll
  for (int i = 0; i < W8; i++) {
    const unsigned k = (unsigned)(8 * kq + (frow >> 2));
    da[i] = (int)(k * TILE + unit_place<UNITS>(k, wm * W8 + i) * 16) + 4 * (frow & 3);
    db[i] = (int)(k * TILE + unit_place<UNITS>(k, wn * W8 + i) * 16) + 4 * (frow & 3);
  }
  auto fragment = [](const half_t *q) { return *reinterpret_cast<const uint4_t *>(q); };
  auto turned = [](const half_t *q) {  // 8 elements of K in two blocks of four rows
    const uint2_t lo = read_column_of_four(q), hi = read_column_of_four(q + 4 * TILE);
    return uint4_t{lo[0], lo[1], hi[0], hi[1]};
  };
  auto fragment_a = [&](int buf, int i, int kk) {
    if constexpr (DOWN_A) return turned(&lds_a[buf][da[i] + kk * 32 * TILE]);
    else return fragment(&lds_a[buf][fa0 + i * 16 * ROWH + ko[kk]]);
  };
  auto fragment_b = [&](int buf, int i, int kk) {
    if constexpr (DOWN_B) return turned(&lds_b[buf][db[i] + kk * 32 * TILE]);
    else return fragment(&lds_b[buf][fb0 + i * 16 * ROWH + ko[kk]]);
  };

  // What is left of K behind the last whole step, zero-filled, through registers into the first buffers.  It comes first, so that
  // the accumulators run through the loop below and into the epilogue without a branch between them (with one, the compiler
  // copies all of them every step: 4001 x 2056 x 4096 98 us instead of 75).
  if (TAIL && tail) {  // the same for the whole block
    const size_t k0 = p.K / BK * BK;
    const int left = (int)(p.K - k0);
#pragma unroll
    for (int t = 0; t < TILE * CPR / 256; t++) {
      // along the rows, K is a multiple of 8 or its rows go on in zeros up to one, so a chunk is there or is not; one that is not
      // reads the first of the step instead
      auto move = [&](const char *from, size_t ld, unsigned last, bool down, half_t *to) {
        const int at = t * 256 + tid, row = down ? at / (int)CHUNKS : at / CPR, place = down ? at % (int)CHUNKS : at % CPR;
        const bool there = (down ? row : place * 8) < left;
        size_t r, c;
        int slot;
        if (down) {
          const unsigned column = unit_place<UNITS>(row, place / 2) * 16 + (place & 1) * 8;
          r = k0 + (there ? row : 0);
          c = column < last ? column : last;
          slot = at * 8;
        } else {
          r = (unsigned)row < last ? (unsigned)row : last;
          c = k0 + (there ? place * 8 : 0);
          slot = row * ROWH + (place ^ ((row >> RS) & (CPR - 1))) * 8;
        }
        const uint4_t chunk = *reinterpret_cast<const uint4_t *>(from + (r * ld + c) * 2), none = {0u, 0u, 0u, 0u};
        *reinterpret_cast<uint4_t *>(to + slot) = there ? chunk : none;
      };
      move(A, p.lda, last_a, DOWN_A, lds_a[0]);
      move(B, p.ldb, last_b, DOWN_B, lds_b[0]);
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < SUB; kk++) {
      uint4_t fa[W8], fb[W8];
#pragma unroll
      for (int i = 0; i < W8; i++) {
        fa[i] = fragment_a(0, i, kk);
        fb[i] = fragment_b(0, i, kk);
      }
#pragma unroll
      for (int t = 0; t < NM; t++) acc[t / W8][t % W8] = mfma_16x16x32_chunks<BF16>(fb[t % W8], fa[t / W8], acc[t / W8][t % W8]);
    }
    __syncthreads();  // the buffers are free again
  }
  {
    uint32_t off_a[TPW], off_b[TPW];
#pragma unroll
    for (int t = 0; t < TPW; t++) {
      auto offset = [&](size_t ld, unsigned last, bool down) {
        const unsigned at = (unsigned)((wave * TPW + t) * 64 + lane);
        if (down) {
          const unsigned row = at / CHUNKS, place = at % CHUNKS, column = unit_place<UNITS>(row, place / 2) * 16 + (place & 1) * 8;
          return (uint32_t)((row * ld + (column < last ? column : last)) * 2);
        }
        const unsigned row = at / CPR, chunk = at % CPR ^ ((row >> RS) & (CPR - 1));
        return (uint32_t)(((row < last ? row : last) * ld + chunk * 8) * 2);
      };
      off_a[t] = offset(p.lda, last_a, DOWN_A);
      off_b[t] = offset(p.ldb, last_b, DOWN_B);
    }
    constexpr lds_addr_t STAGE = OPH * 2, TBYTES = 1024;
    const size_t step_a = BK * 2 * (DOWN_A ? p.lda : 1), step_b = BK * 2 * (DOWN_B ? p.ldb : 1);
    const char *ga = A + step0 * step_a, *gb = B + step0 * step_b;
    const lds_addr_t ta = wave_uniform(lds_address_of(&lds_a[0][0]) + wave * TPW * TBYTES);
    const lds_addr_t tb = wave_uniform(lds_address_of(&lds_b[0][0]) + wave * TPW * TBYTES);
    // steps past the end: a harmless re-read of the last step into a free buffer
    auto issue_a = [&](size_t step, int buf, int t) { load_chunk_to_lds(ga + (step < steps ? step : steps - 1) * step_a, off_a[t], ta + buf * STAGE + t * TBYTES); };
    auto issue_b = [&](size_t step, int buf, int t) { load_chunk_to_lds(gb + (step < steps ? step : steps - 1) * step_b, off_b[t], tb + buf * STAGE + t * TBYTES); };
    // in flight at the first barrier: A0 B0 | A1 B1 (| A2 B2) (the wave's counter returns in issue order)
#pragma unroll
    for (int d = 0; d < NB; d++) {
#pragma unroll
      for (int t = 0; t < TPW; t++) issue_a(d, d, t);
#pragma unroll
      for (int t = 0; t < TPW; t++) issue_b(d, d, t);
    }
    wait_vector_loads<2 * TPW * (NB - 1)>();
    block_barrier_lds_only();
    uint4_t fa[2][W8], fb[2][W8];
#pragma unroll
    for (int i = 0; i < W8; i++) {
      fa[0][i] = fragment_a(0, i, 0);
      fb[0][i] = fragment_b(0, i, 0);
    }
    int ca = 0, cb = 0;  // s % NA, s % NB
    for (size_t s = 0; s < steps; s++) {
      const int na = ca + 1 == NA ? 0 : ca + 1, nb = cb + 1 == NB ? 0 : cb + 1;
      const int fill_a = ca == 0 ? NA - 1 : ca - 1;  // A buffer of step s - 1 = of step s + 2
      // substep 0: MFMA t works on tile (t / W8, t % W8); the fragments of substep 1 are read under it, the A tile of
      // step s + 2 goes out under its second half
#pragma unroll
      for (int t = 0; t < NM; t++) {
        if (t < 4 * W8 && t % 2 == 0) {
          const int k = t / 2;
          if (k == 0) fa[1][0] = fragment_a(ca, 0, 1);
          else if (k <= W8) fb[1][k - 1] = fragment_b(cb, k - 1, 1);
          else fa[1][k - W8] = fragment_a(ca, k - W8, 1);
        }
        if (NB == 2 && t >= NM / 2 && (t - NM / 2) % TEVERY == 0) issue_a(s + 2, fill_a, (t - NM / 2) / TEVERY);
        acc[t / W8][t % W8] = mfma_16x16x32_chunks<BF16>(fb[0][t % W8], fa[0][t / W8], acc[t / W8][t % W8]);
        sched_fence();
      }
      // substep 1: own transfers of step s + 1 done (the A tile of step s + 2 may still fly), barrier, fragments of step
      // s + 1; the B tile of step s + 2 into the B buffer of step s
      wait_vector_loads<NB == 2 ? TPW : 2 * TPW>();
      block_barrier_lds_only();
      sched_fence();
#pragma unroll
      for (int t = 0; t < NM; t++) {
        if (t < 4 * W8 && t % 2 == 0) {
          const int k = t / 2;
          if (k == 0) fa[0][0] = fragment_a(na, 0, 0);
          else if (k <= W8) fb[0][k - 1] = fragment_b(nb, k - 1, 0);
          else fa[0][k - W8] = fragment_a(na, k - W8, 0);
        }
        if (NB == 2 && t >= NM / 2 && (t - NM / 2) % TEVERY == 0) issue_b(s + 2, cb, (t - NM / 2) / TEVERY);
        if (NB == 3 && t % TEVERY == 0) {  // the buffers of step s are free behind the barrier
          if (t < NM / 2) issue_a(s + 3, ca, t / TEVERY);
          else issue_b(s + 3, cb, (t - NM / 2) / TEVERY);
        }
        acc[t / W8][t % W8] = mfma_16x16x32_chunks<BF16>(fb[1][t % W8], fa[1][t / W8], acc[t / W8][t % W8]);
        sched_fence();
      }
      ca = na;
      cb = nb;
    }
    wait_vector_loads<0>();  // the re-reads past the last step must land before the buffers are used for anything else
  }
  // Epilogue: a row of W8 tiles (16 rows x 16 W8 columns) is turned through LDS, so that a lane finishes 8 adjacent columns of
  // a row and global memory sees whole rows of the wave's tile.
  constexpr int SROW = 16 * W8 + 4, LPR = 2 * W8;                    // floats per parked row, lanes per row
  constexpr int RPA = 64 / LPR >= 8 ? 8 : 64 / LPR >= 4 ? 4 : 2;     // rows per access; 192 x 192 tiles leave 16 lanes idle
  static_assert(4 * 2 * 16 * SROW * sizeof(float) <= sizeof(lds_a), "parking area of four waves");
  block_barrier_lds_only();  // the other waves have read their last fragments
  float *park = reinterpret_cast<float *>(&lds_a[0][0]) + wave * (2 * 16 * SROW);
  const bool active = RPA * LPR == 64 || lane < RPA * LPR;
  const unsigned rr = active ? lane / LPR : 0, rc = (lane % LPR) * 8;
  const size_t wave_row = row0 + wave_uniform(wm * WT), wave_col = col0 + wave_uniform(wn * WT);
  const size_t col = wave_col + rc;
  const int count = active && col < p.N ? (int)(p.N - col < 8 ? p.N - col : 8) : 0;
  const bool inside = wave_row + WT <= p.M && wave_col + WT <= p.N;  // the same for the whole wave
  float bias[8] = {};
  if (p.bias && !share) unpack_chunk<DT>(load_chunk_of<DT, WHOLE, false>(p.bias, col, count), bias);
  static_for<W8>([&](auto index) {  // unrolled whatever its size: the accumulators are registers
    constexpr int i = decltype(index)::value;
    float *buf = park + (i & 1) * (16 * SROW);
#pragma unroll
    for (int j = 0; j < W8; j++) *reinterpret_cast<float4_t *>(buf + frow * SROW + 16 * j + 4 * kq) = acc[i][j];
    wave_lds_fence();
    auto finish = [&](int t, int n) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const float4_t q = *reinterpret_cast<const float4_t *>(buf + (t * RPA + rr) * SROW + rc + e);
        v[e] = q[0];
        v[e + 1] = q[1];
        v[e + 2] = q[2];
        v[e + 3] = q[3];
      }
      if (share)
        store_floats<8, true>(share + (wave_row + 16 * i + t * RPA) * p.share_ld + wave_col, rr * (unsigned)p.share_ld + rc, n > 0 ? 8 : 0, v);  // share_ld: N up to a multiple of 8
      else
        fused_gemm_finish<DT, WHOLE>(p, wave_row + 16 * i + t * RPA, wave_col, rr, rc, n, v, bias);
    };
    if (inside) {
      if (active) {
#pragma unroll
        for (int t = 0; t < 16 / RPA; t++) finish(t, 8);
      }
    } else {
#pragma unroll
      for (int t = 0; t < 16 / RPA; t++)
        if (wave_row + 16 * i + t * RPA + rr < p.M) finish(t, count);
    }
  });
}

// K is at least 64, and each split has a whole step at least.  TAIL: K may be no multiple of 64.  (Where K runs down the rows of B the
// kernels all have the tail's code: without it the compiler copies the accumulators of 256 x 256 tiles every step, 3 times slower.)
template <int DT, bool WHOLE, int W8, bool TAIL, int LAYOUT = kAlong>
__global__ __launch_bounds__(256, W8 == 4 ? 2 : 1) void fused_gemm_tile_kernel(FusedGemmParams p) {
  constexpr int TILE = 32 * W8;
  const unsigned split = blockIdx.x / p.tiles, tile = blockIdx.x % p.tiles;
  size_t tile_m, tile_n;
  gemm_tile_of_block((p.M + TILE - 1) / TILE, (p.N + TILE - 1) / TILE, tile, &tile_m, &tile_n);
  const size_t full = p.K / 64, step0 = split * full / p.splits, end = (split + 1) * full / p.splits;
  fused_gemm_tile<DT, WHOLE, W8, TAIL, LAYOUT>(p, tile_m, tile_n, step0, end - step0, split + 1 == p.splits && p.K % 64 != 0, p.shares ? p.shares + (size_t)split * p.M * p.share_ld : nullptr);
}

// The epilogue over the sum of the shares, one thread per 8 adjacent columns, the shares in order.
template <int DT, bool WHOLE>
__global__ __launch_bounds__(256) void fused_gemm_join_kernel(FusedGemmParams p) {
  const size_t chunks = p.share_ld / 8, at = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= p.M * chunks) return;
  const size_t row = at / chunks, col = at % chunks * 8;
  const int count = p.N - col < 8 ? (int)(p.N - col) : 8;
  float v[8] = {}, bias[8] = {};
  for (unsigned s = 0; s < p.splits; s++) {
    float w[8];
    load_floats<8, true>(p.shares, ((size_t)s * p.M + row) * p.share_ld + col, 8, w);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] += w[e];
  }
  if (p.bias) unpack_chunk<DT>(load_chunk_of<DT, WHOLE, false>(p.bias, col, count), bias);
  fused_gemm_finish<DT, WHOLE>(p, row, col, 0u, 0u, count, v, bias);
}

// Up to 16 * MT rows: a block of WAVES waves takes 16 columns; wave w takes the K steps of 32 * UNROLL elements w, w + WAVES, ...
// of its split (a lane reads row (lane & 15) of 16 rows of B, 16 bytes at k = 8 (lane >> 4): 64 bytes of each row per
// instruction, UNROLL instructions in flight).
template <int DT, bool WHOLE, int MT, int WAVES, int UNROLL>
__global__ __launch_bounds__(64 * WAVES) void fused_gemm_few_rows_kernel(FusedGemmParams p) {
  constexpr bool BF16 = DT == kBF16;
  constexpr int STEP = 32 * UNROLL;
  __shared__ __attribute__((aligned(16))) float lds[WAVES][MT][16][20];  // [row of the output][column], padded
  const int lane = lane_id(), wave = wave_in_block(), frow = lane & 15, kq = lane >> 4;
  const unsigned split = blockIdx.x / p.tiles;
  const size_t col0 = (size_t)(blockIdx.x % p.tiles) * 16;
  const size_t n = col0 + frow < p.N ? col0 + frow : p.N - 1;
  const size_t steps = (p.K + STEP - 1) / STEP, per = (steps + p.splits - 1) / p.splits;
  const size_t end = (split + 1) * per < steps ? (split + 1) * per : steps;
  float4_t acc[MT];
#pragma unroll
  for (int i = 0; i < MT; i++) acc[i] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  uint4_t b[2][UNROLL], a[2][MT][UNROLL];
  auto load = [&](size_t s, int to) {
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
      const size_t k = s * STEP + 32 * u + 8 * kq;
      const int count = k < p.K ? (int)(p.K - k < 8 ? p.K - k : 8) : 0;
      b[to][u] = load_chunk_of<DT, WHOLE>(p.B, n * p.ldb + k, count);
#pragma unroll
      for (int i = 0; i < MT; i++) a[to][i][u] = load_chunk_of<DT, WHOLE, false>(p.A, (16 * i + frow) * p.lda + k, (size_t)(16 * i + frow) < p.M ? count : 0);
    }
  };
  auto multiply = [&](int from) {
#pragma unroll
    for (int u = 0; u < UNROLL; u++)
#pragma unroll
      for (int i = 0; i < MT; i++) acc[i] = mfma_16x16x32_chunks<BF16>(b[from][u], a[from][i][u], acc[i]);  // lane: row (lane & 15), columns 4 (lane >> 4) ...
  };
  // The wave's steps are numbered 0 ... count - 1 and begin at another one in every block: with all blocks at the same place
  // along K, rows that are a large power of two apart would all be read from a few memory channels.
  const size_t first = split * per + wave;
  const unsigned steps_here = first < end ? (unsigned)((end - first + WAVES - 1) / WAVES) : 0u, turn = steps_here ? blockIdx.x % steps_here : 0u;
  auto step_at = [&](unsigned i) { return first + (size_t)(i + turn < steps_here ? i + turn : i + turn - steps_here) * WAVES; };
  if (steps_here) load(step_at(0), 0);
  for (unsigned i = 0; i < steps_here; i += 2) {  // the next step's chunks are on their way during a step
    if (i + 1 < steps_here) load(step_at(i + 1), 1);
    multiply(0);
    if (i + 2 < steps_here) load(step_at(i + 2), 0);
    if (i + 1 < steps_here) multiply(1);
  }
#pragma unroll
  for (int i = 0; i < MT; i++) *reinterpret_cast<float4_t *>(&lds[wave][i][frow][4 * kq]) = acc[i];
  __syncthreads();
  // 2 * 16 * MT chunks of 8 columns
  for (int q = (int)threadIdx.x; q < 32 * MT; q += 64 * WAVES) {
    const int r = q / 2, c = (q % 2) * 8;
    const size_t row = r, col = col0 + c;
    const int count = col < p.N ? (int)(p.N - col < 8 ? p.N - col : 8) : 0;
    if (row >= p.M || count == 0) continue;
    float v[8] = {}, bias[8] = {};
#pragma unroll
    for (int w = 0; w < WAVES; w++)
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] += lds[w][r / 16][r % 16][c + e];
    if (p.shares) {
      store_floats<8, true>(p.shares, ((size_t)split * p.M + row) * p.share_ld + col, 8, v);
    } else {
      if (p.bias) unpack_chunk<DT>(load_chunk_of<DT, WHOLE, false>(p.bias, col, count), bias);
      fused_gemm_finish<DT, WHOLE>(p, row, col, 0u, 0u, count, v, bias);
    }
  }
}

// `rows` x `width` elements of 16 bits to rows of `to_ld` elements, 16-byte aligned (for operands whose rows are not)
struct PackRowsParams {
  const uint16_t *from;
  uint16_t *to;
  size_t rows, width, padded, from_ld, to_ld;  // padded: a multiple of 8; zeros from the width up to there
};
__global__ __launch_bounds__(256) inline void pack_rows_kernel(PackRowsParams p) {
  const size_t chunks = p.padded / 8, at = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= p.rows * chunks) return;
  const size_t row = at / chunks, col = at % chunks * 8;
  const int count = col < p.width ? (p.width - col < 8 ? (int)(p.width - col) : 8) : 0;
  const uint4_t c = load_chunk_of<kF16, false>(p.from, count ? row * p.from_ld + col : 0, count);
  *reinterpret_cast<uint4_t *>(p.to + row * p.to_ld + col) = c;
}

// 64 x 64 tiles turned through LDS.  The first job turns dZ = dD act'(Z), which is written
// as it stands as well (dz, which may be null), and adds up the columns of each 64-row strip of it before it is rounded.
struct TransposeJob {
  const void *from;
  void *to;                      // null: nothing is turned
  size_t rows, columns, from_ld, to_ld;  // to_ld: a multiple of 64; the rows of the transpose end in zeros up to that
  unsigned column_tiles, tiles;
};
struct TransposeParams {
  TransposeJob job[3];  // dD (of bf16 or fp16), then A and B, whose bits move as they are
  const void *Z;        // null: no activation
  void *dz;
  float *partial;       // [row strip][columns of dD], or null
  size_t z_ld, dz_ld;   // dz_ld: a multiple of 64
  int act;
};

template <int DT, bool GRAD>
TCU_DEVICE void transpose_tile(const TransposeParams &p, const TransposeJob &j, unsigned tile, uint16_t *lds, float *sums) {
  constexpr int LD = 66;  // 16-bit elements per LDS row: 33 words, so a column of 16-bit pairs falls into different banks
  const size_t row0 = (size_t)(tile / j.column_tiles) * 64, col0 = (size_t)(tile % j.column_tiles) * 64;
  const int tid = (int)threadIdx.x, tr = tid / 8, tc = (tid % 8) * 8;  // 32 rows of 8 chunks a round
  float s[8] = {};
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int r = h * 32 + tr;
    const size_t row = row0 + r, col = col0 + tc;
    const int count = row < j.rows && col < j.columns ? (j.columns - col < 8 ? (int)(j.columns - col) : 8) : 0;
    uint4_t c = load_chunk_of<DT, false>(j.from, count ? row * j.from_ld + col : 0, count);
    if constexpr (GRAD) {
      float d[8];
      unpack_chunk<DT>(c, d);
      if (p.Z) {
        float z[8], value[8], slope[8];
        unpack_chunk<DT>(load_chunk_of<DT, false>(p.Z, count ? row * p.z_ld + col : 0, count), z);
        activate_slope<false>(p.act, z, value, slope);
#pragma unroll
        for (int e = 0; e < 8; e++) d[e] = e < count ? d[e] * slope[e] : 0.0f;
        c = pack_chunk<DT>(d);
      }
      if (p.dz && row < j.rows) store_packed<DT, true>(p.dz, row * p.dz_ld + col, 8, c);  // its rows end in zeros
#pragma unroll
      for (int e = 0; e < 8; e++) s[e] += d[e];
    }
#pragma unroll
    for (int e = 0; e < 4; e++) *reinterpret_cast<uint32_t *>(&lds[r * LD + tc + 2 * e]) = c[e];
  }
  if constexpr (GRAD) {
#pragma unroll
    for (int e = 0; e < 8; e++) sums[tr * 64 + tc + e] = s[e];
  }
  __syncthreads();
  if constexpr (GRAD) {
    if (p.partial && tid < 64 && col0 + tid < j.columns) {
      float t = 0.0f;
#pragma unroll
      for (int r = 0; r < 32; r++) t += sums[r * 64 + tid];
      p.partial[row0 / 64 * j.columns + col0 + tid] = t;
    }
  }
  if (!j.to) return;
#pragma unroll
  for (int h = 0; h < 2; h++) {  // row tr (+ 32) of the transpose: 8 chunks of 8 of the tile's rows
    const int r = h * 32 + tr;
    const size_t row = col0 + r, col = row0 + tc;
    if (row >= j.columns) continue;
    uint4_t c;
#pragma unroll
    for (int e = 0; e < 4; e++) c[e] = (unsigned)lds[(tc + 2 * e) * LD + r] | (unsigned)lds[(tc + 2 * e + 1) * LD + r] << 16;
    *reinterpret_cast<uint4_t *>(static_cast<uint16_t *>(j.to) + row * j.to_ld + col) = c;
  }
}

// All that the gradient's products need laid out anew, in one launch (three transposes of 4001 x 4096 x 2056 bf16 one by one 27 + 10 + 10 us,
// together 38).
template <int DT>
__global__ __launch_bounds__(256) void gradient_layout_kernel(TransposeParams p) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[64 * 66];
  __shared__ float sums[32 * 64];
  unsigned tile = blockIdx.x;
  if (tile < p.job[0].tiles) {
    transpose_tile<DT, true>(p, p.job[0], tile, lds, sums);
    return;
  }
  tile -= p.job[0].tiles;
  const bool second = tile >= p.job[1].tiles;
  transpose_tile<kF16, false>(p, second ? p.job[2] : p.job[1], second ? tile - p.job[1].tiles : tile, lds, sums);
}

}  // namespace tcu

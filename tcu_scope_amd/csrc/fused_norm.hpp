// Norm of every row fused with the residual addition, the scale of the residual branch and a gate:
//
//   add_norm:  z = residual + s x (z = x without a residual),  out = act(gate) y(z),  z is written too (the residual stream)
//   norm_add:  out = residual + s act(gate) y(x)
//   y(z) = n weight + bias,  n = (z - mean) rho;  rms: mean = 0, rho = 1 / sqrt(mean z^2 + eps);
//   layer: mean of the row, rho = 1 / sqrt(mean (z - mean)^2 + eps);  s = scale * channel_scale, one number per channel.
//
// Gradient, with d the gradient with respect to act(gate) y (norm_add: s dout; add_norm: dout):
//   dy = d act(gate),  dgate = d y act'(gate),  dweight = sum dy n,  dbias = sum dy  (sums over rows)
//   dn = dy weight,  dz = rho (dn - n mean(dn n) - [layer] mean(dn))
//   norm_add: dx = dz, dchannel_scale = scale sum dout act(gate) y
//   add_norm: dz += dstream (the gradient of the written z), dresidual = dz, dx = s dz, dchannel_scale = scale sum dz x
//
// Bound by HBM traffic: every operand is read once and every result written once.  A row lives in the registers of the
// WAVES waves that share it (CHUNKS 16-byte chunks per lane), so the statistics take no second read; the variance is that of
// the centred values (two sums one after the other), which a difference of sums would lose the digits of.  The gradients
// of the vectors are sums over rows: a block walks many rows with its columns' sums in registers, writes them once as
// partial sums, and a second launch adds the partial sums of each column in a fixed order (no atomics: the same input
// gives the same bits).  16384 x 4096 bf16 with residual 89 us (537 MB, 6.0 TB/s, part of it served by the last-level cache), the
// gradient of the gated layer form with 8192 x 4096 79 us + 4.7 for the partial sums (336 MB, 4.1 TB/s: every row passes through
// two reductions over its 8 waves), 12 x 2048 fp16 3.8 us.
#pragma once

#include "elements.hpp"

namespace tcu {

constexpr int kNormRms = 0, kNormLayer = 1;      // tcu_norm
constexpr int kOrderAddNorm = 0, kOrderNormAdd = 1;  // tcu_norm_order

struct FusedNormParams {
  const void *x, *residual, *gate, *weight, *bias, *channel_scale;  // all but x may be null
  void *out, *z_out;                                                // z_out may be null
  size_t x_stride, residual_stride, gate_stride, out_stride, z_out_stride;
  size_t rows;
  unsigned dim;
  float eps, scale;
  int norm, order, act;
};

// sums over the WAVES waves that share a row, in every lane; `lds` has 4 * WAVES floats per parity, and consecutive
// calls alternate the parity, so one barrier a call is enough
template <int WAVES, int N>
TCU_DEVICE void row_sums(float (&v)[N], float *lds, int wave, int parity) {
#pragma unroll
  for (int i = 0; i < N; i++) v[i] = wave_sum(v[i]);
  if constexpr (WAVES > 1) {
    float *slot = lds + parity * (4 * WAVES);
    if (lane_id() == 0) {
#pragma unroll
      for (int i = 0; i < N; i++) slot[i * WAVES + wave] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; w++) s += slot[i * WAVES + w];
      v[i] = s;
    }
  }
}

// V values of a vector operand of the row (null: `missing` everywhere)
template <int DT, bool ALIGNED>
TCU_DEVICE void load_vector(const void *p, unsigned at, int count, float missing, float (&v)[Elem<DT>::V]) {
  if (p) {
    unpack_chunk<DT>(load_chunk_of<DT, ALIGNED, false>(p, at, count), v);
  } else {
#pragma unroll
    for (int e = 0; e < Elem<DT>::V; e++) v[e] = missing;
  }
}

// WAVES waves share a row; a block has BLOCK_WAVES waves, i.e. BLOCK_WAVES / WAVES rows.
template <int DT, bool ALIGNED, int WAVES, int CHUNKS, int BLOCK_WAVES>
__global__ __launch_bounds__(64 * BLOCK_WAVES) void fused_norm_kernel(FusedNormParams p) {
  constexpr int V = Elem<DT>::V;
  constexpr bool EXACT = DT == kF32;
  __shared__ float lds[WAVES > 1 ? 8 * WAVES : 1];
  static_assert(WAVES == 1 || WAVES == BLOCK_WAVES, "rows that share a block share no sums");
  const int wave = wave_in_block();
  const size_t row = WAVES == 1 ? (size_t)blockIdx.x * BLOCK_WAVES + wave : blockIdx.x;
  if (row >= p.rows) return;  // a whole wave, of rows that need no barrier
  const int lane = WAVES == 1 ? lane_id() : (int)threadIdx.x;
  auto column = [&](int k) { return (unsigned)(k * 64 * WAVES + lane) * V; };
  auto exists = [&](int k) { return (int)p.dim - (int)column(k); };

  const bool add_first = p.order == kOrderAddNorm && p.residual != nullptr;
  float z[CHUNKS][V];
  uint4_t cr[CHUNKS], cg[CHUNKS];
#pragma unroll
  for (int k = 0; k < CHUNKS; k++) {
    unpack_chunk<DT>(load_chunk_of<DT, ALIGNED>(p.x, row * p.x_stride + column(k), exists(k)), z[k]);
    if (p.residual) cr[k] = load_chunk_of<DT, ALIGNED>(p.residual, row * p.residual_stride + column(k), exists(k));
    if (p.gate) cg[k] = load_chunk_of<DT, ALIGNED>(p.gate, row * p.gate_stride + column(k), exists(k));
  }
  if (add_first) {
#pragma unroll
    for (int k = 0; k < CHUNKS; k++) {
      float s[V], r[V];
      load_vector<DT, ALIGNED>(p.channel_scale, column(k), exists(k), 1.0f, s);
      unpack_chunk<DT>(cr[k], r);
#pragma unroll
      for (int e = 0; e < V; e++) z[k][e] = __builtin_fmaf(p.scale * s[e], z[k][e], r[e]);
      if (p.z_out) store_chunk_of<DT, ALIGNED>(p.z_out, row * p.z_out_stride + column(k), exists(k), z[k]);
    }
  }
  const float inv = 1.0f / (float)p.dim;
  float mean = 0.0f, sum[1];
  if (p.norm == kNormLayer) {
    sum[0] = 0.0f;
#pragma unroll
    for (int k = 0; k < CHUNKS; k++)
#pragma unroll
      for (int e = 0; e < V; e++) sum[0] += z[k][e];  // columns beyond the row hold 0
    row_sums<WAVES>(sum, lds, wave, 0);
    mean = sum[0] * inv;
  }
  sum[0] = 0.0f;
#pragma unroll
  for (int k = 0; k < CHUNKS; k++)
#pragma unroll
    for (int e = 0; e < V; e++) {
      z[k][e] -= mean;
      if (e < exists(k)) sum[0] = __builtin_fmaf(z[k][e], z[k][e], sum[0]);
    }
  row_sums<WAVES>(sum, lds, wave, 1);
  const float rho = hw_rsqrt(__builtin_fmaf(sum[0], inv, p.eps));
#pragma unroll
  for (int k = 0; k < CHUNKS; k++) {
    float w[V], b[V], y[V];
    load_vector<DT, ALIGNED>(p.weight, column(k), exists(k), 1.0f, w);
    load_vector<DT, ALIGNED>(p.bias, column(k), exists(k), 0.0f, b);
#pragma unroll
    for (int e = 0; e < V; e++) y[e] = __builtin_fmaf(z[k][e] * rho, w[e], b[e]);
    if (p.gate) {
      float g[V];
      unpack_chunk<DT>(cg[k], g);
      activate<EXACT>(p.act, g);
#pragma unroll
      for (int e = 0; e < V; e++) y[e] *= g[e];
    }
    if (p.order == kOrderNormAdd) {
      float s[V], r[V];
      load_vector<DT, ALIGNED>(p.channel_scale, column(k), exists(k), 1.0f, s);
#pragma unroll
      for (int e = 0; e < V; e++) r[e] = 0.0f;
      if (p.residual) unpack_chunk<DT>(cr[k], r);
#pragma unroll
      for (int e = 0; e < V; e++) y[e] = __builtin_fmaf(p.scale * s[e], y[e], r[e]);
    }
    store_chunk_of<DT, ALIGNED>(p.out, row * p.out_stride + column(k), exists(k), y);
  }
}

struct FusedNormBackParams {
  const void *dout, *z, *gate, *weight, *bias, *channel_scale, *x, *dstream;  // all but dout and z may be null
  void *dx, *dgate, *dresidual;                                              // all but dx may be null
  size_t dout_stride, z_stride, gate_stride, x_stride, dstream_stride, dx_stride, dgate_stride, dresidual_stride;
  float *partial;  // [part][vector][dim]: dweight, dbias, dchannel_scale, those that are asked for
  size_t rows;
  unsigned dim;
  float eps, scale;
  int norm, order, act;
  bool want_weight, want_bias, want_scale;
};

// GATE, STREAM: there is a gate; there is a dstream or x is read (each costs registers; not ALIGNED: there may be).
// LEAN: for rows so long that the rest would not fit the registers (a spill here costs several times the kernel): the next row
// is not fetched ahead, only z stays in registers between the statistics and the gradients, and the other operands are read a
// second time, from the cache.
template <int DT, bool ALIGNED, bool GATE, bool STREAM, bool LEAN, int WAVES, int CHUNKS, int BLOCK_WAVES>
__global__ __launch_bounds__(64 * BLOCK_WAVES) void fused_norm_backward_kernel(FusedNormBackParams p) {
  constexpr int V = Elem<DT>::V;
  constexpr bool EXACT = DT == kF32;
  __shared__ float lds[WAVES > 1 ? 8 * WAVES : 1];
  static_assert(WAVES == 1 || WAVES == BLOCK_WAVES, "rows that share a block share no sums");
  const int wave = wave_in_block();
  const size_t part = WAVES == 1 ? (size_t)blockIdx.x * BLOCK_WAVES + wave : blockIdx.x;
  const size_t parts = WAVES == 1 ? (size_t)gridDim.x * BLOCK_WAVES : gridDim.x;
  const int lane = WAVES == 1 ? lane_id() : (int)threadIdx.x;
  auto column = [&](int k) { return (unsigned)(k * 64 * WAVES + lane) * V; };
  auto exists = [&](int k) { return (int)p.dim - (int)column(k); };
  const bool add_norm = p.order == kOrderAddNorm;
  const float inv = 1.0f / (float)p.dim;

  float sw[CHUNKS][V], sb[CHUNKS][V], ss[CHUNKS][V];  // column sums of dweight, dbias, dchannel_scale
#pragma unroll
  for (int k = 0; k < CHUNKS; k++)
#pragma unroll
    for (int e = 0; e < V; e++) sw[k][e] = sb[k][e] = ss[k][e] = 0.0f;

  // the vectors stay in registers as they are stored (LEAN: in the cache)
  constexpr int HELD = LEAN ? 1 : CHUNKS;
  uint4_t vw[HELD], vb[HELD], vc[HELD];
  if constexpr (!LEAN) {
#pragma unroll
    for (int k = 0; k < CHUNKS; k++) {
      vw[k] = vb[k] = vc[k] = uint4_t{0u, 0u, 0u, 0u};
      if (p.weight) vw[k] = load_chunk_of<DT, ALIGNED, false>(p.weight, column(k), exists(k));
      if (p.bias) vb[k] = load_chunk_of<DT, ALIGNED, false>(p.bias, column(k), exists(k));
      if (p.channel_scale) vc[k] = load_chunk_of<DT, ALIGNED, false>(p.channel_scale, column(k), exists(k));
    }
  }
  auto held = [&](const void *there, const uint4_t &kept, int k) {
    if constexpr (LEAN) return there ? load_chunk_of<DT, ALIGNED, false>(there, column(k), exists(k)) : uint4_t{0u, 0u, 0u, 0u};
    return kept;
  };
  auto four_of = [](const void *there, const uint4_t &c, int q, float missing, float(&v)[4]) {
    if (there) {
      unpack_four<DT>(c, q, v);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = missing;
    }
  };
  uint4_t nz[CHUNKS], nd[HELD], ng[HELD], ns[HELD], nx[HELD];
  const bool read_x = p.want_scale && add_norm, gated = GATE && (ALIGNED || p.gate);
  auto load_z = [&](size_t row, int k) { return load_chunk_of<DT, ALIGNED>(p.z, row * p.z_stride + column(k), exists(k)); };
  auto load_d = [&](size_t row, int k) { return load_chunk_of<DT, ALIGNED, !LEAN>(p.dout, row * p.dout_stride + column(k), exists(k)); };
  auto load_g = [&](size_t row, int k) { return load_chunk_of<DT, ALIGNED, !LEAN>(p.gate, row * p.gate_stride + column(k), exists(k)); };
  auto load_rest = [&](size_t row, int k, int at) {
    if (STREAM && p.dstream) ns[at] = load_chunk_of<DT, ALIGNED>(p.dstream, row * p.dstream_stride + column(k), exists(k));
    if (STREAM && read_x) nx[at] = load_chunk_of<DT, ALIGNED>(p.x, row * p.x_stride + column(k), exists(k));
  };
  auto load_row = [&](size_t row) {
#pragma unroll
    for (int k = 0; k < CHUNKS; k++) {
      nz[k] = load_z(row, k);
      if constexpr (!LEAN) {
        nd[k] = load_d(row, k);
        if (gated) ng[k] = load_g(row, k);
        load_rest(row, k, k);
      }
    }
  };
  // the next row's operands are on their way while a row is worked on
  if (!LEAN && part < p.rows) load_row(part);

  int parity = 0;
  for (size_t row = part; row < p.rows; row += parts) {
    float z[CHUNKS][V];  // centred
    float f[HELD][V], slope[HELD][V];  // act(gate) and act'(gate)
    uint4_t cd[HELD], cs[HELD], cx[HELD];
    auto gate_factors = [&](const uint4_t &gate, int q, float(&value)[4], float(&slopes)[4]) {
      if (gated) {
        float g[4];
        unpack_four<DT>(gate, q, g);
        activate_slope<EXACT>(p.act, g, value, slopes);
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          value[e] = 1.0f;
          slopes[e] = 0.0f;
        }
      }
    };
    if constexpr (LEAN) load_row(row);
#pragma unroll
    for (int k = 0; k < CHUNKS; k++) {
      unpack_chunk<DT>(nz[k], z[k]);
      if constexpr (!LEAN) {
        cd[k] = nd[k];
#pragma unroll
        for (int q = 0; q < V / 4; q++) {
          float v[4], t[4];
          gate_factors(ng[k], q, v, t);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            f[k][4 * q + e] = v[e];
            slope[k][4 * q + e] = t[e];
          }
        }
        if (STREAM && p.dstream) cs[k] = ns[k];
        if (STREAM && read_x) cx[k] = nx[k];
      }
    }
    if constexpr (!LEAN) {
      if (row + parts < p.rows) load_row(row + parts);
#pragma unroll
      for (int k = 0; k < CHUNKS; k++) {
        keep_packed(vw[k]);
        keep_packed(vb[k]);
        keep_packed(vc[k]);
      }
    }
    float mean = 0.0f;
    if (p.norm == kNormLayer) {
      float s[1] = {0.0f};
#pragma unroll
      for (int k = 0; k < CHUNKS; k++)
#pragma unroll
        for (int e = 0; e < V; e++) s[0] += z[k][e];
      row_sums<WAVES>(s, lds, wave, parity);
      parity ^= 1;
      mean = s[0] * inv;
    }
    // the factors of values 4 q ... of chunk k, and the gradient with respect to act(gate) y there
    constexpr int H = LEAN ? 0 : 1;
    auto upstream = [&](int k, int q, const uint4_t &scale, float(&v)[4], float(&t)[4], float(&d)[4], float(&up)[4], float(&c)[4]) {
      if constexpr (LEAN) {
        gate_factors(ng[0], q, v, t);
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          v[e] = f[H * k][4 * q + e];
          t[e] = slope[H * k][4 * q + e];
        }
      }
      unpack_four<DT>(cd[H * k], q, d);
      four_of(p.channel_scale, scale, q, 1.0f, c);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        c[e] *= p.scale;
        up[e] = add_norm ? d[e] : c[e] * d[e];
      }
    };
    // sums of z^2, dn z and dn over the row (z centred)
    float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < CHUNKS; k++) {
      if constexpr (LEAN) {
        cd[0] = load_d(row, k);
        if (gated) ng[0] = load_g(row, k);
      }
      const uint4_t cw = held(p.weight, vw[H * k], k), cc = held(p.channel_scale, vc[H * k], k);
#pragma unroll
      for (int q = 0; q < V / 4; q++) {
        float w[4], v[4], t[4], d[4], up[4], c[4];
        four_of(p.weight, cw, q, 1.0f, w);
        upstream(k, q, cc, v, t, d, up, c);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          float &zc = z[k][4 * q + e];
          zc -= mean;
          if (4 * q + e < exists(k)) {
            const float dn = up[e] * v[e] * w[e];
            s[0] = __builtin_fmaf(zc, zc, s[0]);
            s[1] = __builtin_fmaf(dn, zc, s[1]);
            s[2] += dn;
          }
        }
      }
    }
    row_sums<WAVES>(s, lds, wave, parity);
    parity ^= 1;
    const float rho = hw_rsqrt(__builtin_fmaf(s[0], inv, p.eps));
    const float mean_dnn = s[1] * rho * inv, mean_dn = p.norm == kNormLayer ? s[2] * inv : 0.0f;
#pragma unroll
    for (int k = 0; k < CHUNKS; k++) {
      if constexpr (LEAN) {
        cd[0] = load_d(row, k);
        if (gated) ng[0] = load_g(row, k);
        load_rest(row, k, 0);
        if (STREAM && p.dstream) cs[0] = ns[0];
        if (STREAM && read_x) cx[0] = nx[0];
      }
      const uint4_t cw = held(p.weight, vw[H * k], k), cb = held(p.bias, vb[H * k], k), cc = held(p.channel_scale, vc[H * k], k);
      uint4_t odx, odg, odr;
#pragma unroll
      for (int q = 0; q < V / 4; q++) {
        float w[4], b[4], v[4], t[4], d[4], up[4], c[4], extra[4], x[4], dx[4], dg[4];
        four_of(p.weight, cw, q, 1.0f, w);
        four_of(p.bias, cb, q, 0.0f, b);
        upstream(k, q, cc, v, t, d, up, c);
        four_of(STREAM ? p.dstream : nullptr, cs[H * k], q, 0.0f, extra);
        four_of(STREAM && read_x ? p.x : nullptr, cx[H * k], q, 0.0f, x);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int i = 4 * q + e;
          const float n = z[k][i] * rho, y = __builtin_fmaf(n, w[e], b[e]), dy = up[e] * v[e];
          dg[e] = up[e] * y * t[e];
          sw[k][i] = __builtin_fmaf(dy, n, sw[k][i]);
          sb[k][i] += dy;
          if (!add_norm) ss[k][i] = __builtin_fmaf(d[e], v[e] * y, ss[k][i]);
          dx[e] = rho * (__builtin_fmaf(-n, mean_dnn, dy * w[e]) - mean_dn);
          if (add_norm) {
            dx[e] += extra[e];
            if constexpr (STREAM) ss[k][i] = __builtin_fmaf(dx[e], x[e], ss[k][i]);
          }
        }
        pack_four<DT>(odr, q, dx);
        if (add_norm) {
#pragma unroll
          for (int e = 0; e < 4; e++) dx[e] *= c[e];
        }
        pack_four<DT>(odx, q, dx);
        if constexpr (GATE) pack_four<DT>(odg, q, dg);
      }
      if (p.dresidual) store_packed<DT, ALIGNED>(p.dresidual, row * p.dresidual_stride + column(k), exists(k), odr);
      store_packed<DT, ALIGNED>(p.dx, row * p.dx_stride + column(k), exists(k), odx);
      if (GATE && p.dgate) store_packed<DT, ALIGNED>(p.dgate, row * p.dgate_stride + column(k), exists(k), odg);
    }
  }
  const int vectors = (int)p.want_weight + (int)p.want_bias + (int)p.want_scale;
  float *to = p.partial + part * vectors * p.dim;
#pragma unroll
  for (int k = 0; k < CHUNKS; k++) {
    float *q = to;
#pragma unroll
    for (int e = 0; e < V; e++) ss[k][e] *= p.scale;
    if (p.want_weight) {
      store_floats<V, ALIGNED>(q, column(k), exists(k), sw[k]);
      q += p.dim;
    }
    if (p.want_bias) {
      store_floats<V, ALIGNED>(q, column(k), exists(k), sb[k]);
      q += p.dim;
    }
    if (p.want_scale) store_floats<V, ALIGNED>(q, column(k), exists(k), ss[k]);
  }
}

}  // namespace tcu

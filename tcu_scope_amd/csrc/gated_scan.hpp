// Gated linear recurrence along the tokens of each sequence, every channel by itself:
//
//   h[t] = a[t] h[t-1] + b[t],  h[-1] = h0 of the sequence (0 without one), from a gate g and an input x:
//     decay    a = g            b = x
//     log      a = exp(g)       b = x
//     sigmoid  a = sigmoid(g)   b = (1 - a) x
//
// and its gradient: with delta[t] the gradient with respect to h[t], all paths into the future included,
//
//   u[t] = a[t] delta[t],  delta[t] = dh[t] + u[t+1],  u[behind the last token] = dh_last of the sequence,
//   i.e. u[t] = a[t] u[t+1] + a[t] dh[t]: the same recurrence down the tokens in reverse;
//   dx = delta (sigmoid: (1 - a) delta);  dg = delta h[t-1] (log: * a;  sigmoid: delta (h[t-1] - x) a (1 - a));
//   dh0 = u[first token].
//
// The step is a scan under (A, B) then (A', B') = (A' A, A' B + B'), as the prefix sums of this library are under +.
// Tokens are the rows of row-major matrices, sequences follow each other down the rows (equal lengths, or an offsets
// array), channels are contiguous.  Both directions run in one order of "places" 0, 1, ...: place p is row p forwards and
// row rows-1-p backwards.
//
// One pass over the data: a block takes a tile of TILE_ROWS places x TILE_CHANNELS channels into registers (a thread has
// RPT consecutive places of one 16-byte chunk of channels), works out the (A, B) of each thread's places, the carry into
// each thread from those in LDS, and finishes from registers.  The bound is HBM traffic (2 streams in, 1 out; backwards
// 3 or 4 in, 2 out); exponential and reciprocal are quarter-rate instructions, so a and b are worked out once and kept.
//
// Tiles that follow each other along the sequences hand the state on through descriptors in the workspace, two 64-bit
// words per channel, each a tag with a value, so that a word is whole whenever it is seen and needs no fence.  A tile
// publishes either its aggregate (A, B), as soon as it has read its input, or the state behind it; which of the two is
// settled by its place alone: the state where a sequence begins inside the tile (nothing from in front is needed) and at
// every kGroupTiles-th tile; so a tile waits for its group's aggregates, which wait for nothing, and for one state, and
// combines them in one fixed order: the same input gives the same bits every time, and the chain of waits is a
// kGroupTiles-th of the tiles.  Tiles are handed out by a ticket, so the one that is waited for has always been started;
// a wait is bounded and leaves NaN in what depended on it.
#pragma once

#include "elements.hpp"

namespace tcu {

constexpr int kGateDecay = 0, kGateLog = 1, kGateSigmoid = 2;  // tcu_gate
constexpr unsigned kScanGroupTiles = 8;

struct GatedScanParams {
  const void *x, *g, *h, *dh;  // x: also the input of the sigmoid gate's gradient; h: backwards only
  void *out, *out_g;           // h forwards; dx and dg backwards
  const float *seed;           // state in front of a sequence in place order: h0 / dh_last (may be null)
  const float *h0;             // backwards: h[-1] of the gradient's formulas (may be null)
  float *last;                 // state behind it: h_last / dh0 (may be null)
  const int *row_sequence;     // sequence of each row, -1 outside all; null: sequence_rows rows each
  size_t x_stride, g_stride, h_stride, dh_stride, out_stride, out_g_stride;  // elements from row to row
  unsigned rows, sequence_rows, channels, strips, chunks;
  bool zero_outside;               // rows of no sequence: their outputs become 0, or are left as they are
  unsigned *ticket;                // null: one chunk of places, the block index is the tile
  unsigned long long *descriptors; // [chunk][strip][channel of the tile][2]
  unsigned poll_limit, mute_tile;  // mute_tile: tests only, tile mute_tile - 1 publishes nothing
  unsigned *expired;
};

constexpr unsigned kDescAggregate = 1, kDescState = 2;
TCU_DEVICE unsigned long long tagged(unsigned tag, float v) { return ((unsigned long long)tag << 32) | __float_as_uint(v); }
TCU_DEVICE unsigned tag_of(unsigned long long w) { return (unsigned)(w >> 32); }
TCU_DEVICE float value_of(unsigned long long w) { return __uint_as_float((unsigned)w); }

template <int DT, int GATE>
TCU_DEVICE void gate_of(float g, float *a, float *keep) {  // keep = 1 - a (sigmoid only)
  *keep = 1.0f;
  if constexpr (GATE == kGateDecay) *a = g;
  if constexpr (GATE == kGateLog) *a = exp_of<DT == kF32>(g);
  if constexpr (GATE == kGateSigmoid) sigmoid_pair<DT == kF32>(g, a, keep);
}

// The carry into this tile for channel `c` of it; the tile's own aggregate is (A, B).  One thread per channel.
//   own_state: a sequence begins in the tile, so B is the state behind it whatever came in front
//   needs: the tile's first place continues a sequence
TCU_DEVICE float exchange_carry(const GatedScanParams &p, unsigned chunk, unsigned strip, int tile_channels, int c, float A, float B, bool own_state, bool needs) {
  const size_t stride = (size_t)p.strips * tile_channels * 2;  // words from chunk to chunk
  unsigned long long *mine = p.descriptors + ((size_t)chunk * p.strips + strip) * tile_channels * 2 + 2 * c;
  const bool muted = p.mute_tile != 0 && chunk * p.strips + strip == p.mute_tile - 1;
  const bool closes_group = chunk % kScanGroupTiles == kScanGroupTiles - 1;
  if (own_state && !muted) {
    atomic_store_u64(mine, tagged(kDescState, B));
  } else if (!closes_group && !muted) {
    atomic_store_u64(mine, tagged(kDescAggregate, A));
    atomic_store_u64(mine + 1, tagged(kDescAggregate, B));
  }
  float carry = 0.0f;
  if (needs) {
    // the group's tiles in front of this one, and the one that closed the group before
    const unsigned in_group = chunk % kScanGroupTiles;
    const unsigned count = in_group + (chunk >= kScanGroupTiles ? 1u : 0u);  // >= 1: the first tile of all begins a sequence
    const unsigned long long *first = mine - (size_t)count * stride;
    unsigned long long w0[kScanGroupTiles], w1[kScanGroupTiles];
#pragma unroll
    for (unsigned j = 0; j < kScanGroupTiles; j++) w0[j] = w1[j] = 0;
    unsigned polls = 0;
    bool waiting = true, gave_up = false;
    while (waiting) {
      waiting = false;
#pragma unroll
      for (unsigned j = 0; j < kScanGroupTiles; j++) {
        if (j < count) {
          if (tag_of(w0[j]) == 0) w0[j] = atomic_load_u64(first + j * stride);
          if (tag_of(w1[j]) == 0 && tag_of(w0[j]) != kDescState) w1[j] = atomic_load_u64(first + j * stride + 1);
        }
      }
#pragma unroll
      for (unsigned j = 0; j < kScanGroupTiles; j++)
        if (j < count && (tag_of(w0[j]) == 0 || (tag_of(w0[j]) == kDescAggregate && tag_of(w1[j]) == 0))) waiting = true;
      if (waiting && polls++ >= p.poll_limit) {
        gave_up = true;
        break;
      }
      if (waiting) spin_pause();
    }
#pragma unroll
    for (unsigned j = 0; j < kScanGroupTiles; j++)
      if (j < count) carry = tag_of(w0[j]) == kDescState ? value_of(w0[j]) : __builtin_fmaf(value_of(w0[j]), carry, value_of(w1[j]));
    if (gave_up) {
      carry = __builtin_nanf("");
      if (c == 0 && p.expired) atomic_add_u32(p.expired, 1u);
    }
  }
  if (!own_state && closes_group && !muted) atomic_store_u64(mine, tagged(kDescState, __builtin_fmaf(A, carry, B)));
  return carry;
}

// TCL lanes share a row of the tile (TCL * V channels); blocks of THREADS threads, RPT places per thread.
template <int DT, int GATE, bool BACK, bool ALIGNED, int TCL, int RPT, int THREADS>
__global__ __launch_bounds__(THREADS) void gated_scan_kernel(GatedScanParams p) {
  constexpr int V = Elem<DT>::V, TC = TCL * V, GROUPS = THREADS / TCL, TILE_ROWS = GROUPS * RPT;
  static_assert(TC <= THREADS, "one thread per channel carries the state through the tile");
  __shared__ __attribute__((aligned(16))) float lds_a[GROUPS * TC];
  __shared__ __attribute__((aligned(16))) float lds_b[GROUPS * TC];
  __shared__ unsigned lds_reset[GROUPS];  // bit 0: a sequence begins in the group, bit 1: it does so at the group's first place
  __shared__ unsigned lds_tile;
  const int tid = (int)threadIdx.x, lane = tid % TCL, group = tid / TCL;
  unsigned tile = blockIdx.x;
  if (p.ticket) {  // the same for every block of the launch
    if (tid == 0) lds_tile = atomic_add_u32(p.ticket, 1u);
    __syncthreads();
    tile = lds_tile;
  }
  const unsigned chunk = tile / p.strips, strip = tile % p.strips;
  const unsigned place0 = chunk * TILE_ROWS + group * RPT;
  const unsigned channel = strip * TC + lane * V;
  const int count = (int)p.channels - (int)channel;  // channels of this chunk that exist (<= 0: none)

  // what each of the thread's places is: inside a sequence, the first or the last one of it in place order
  unsigned inside = 0, begins = 0, ends = 0;
  auto row_of = [&](unsigned place) { return BACK ? p.rows - 1 - place : place; };
  if (p.row_sequence) {
    int before = -1;
    if (place0 > 0 && place0 <= p.rows) before = p.row_sequence[row_of(place0 - 1)];
    int now = place0 < p.rows ? p.row_sequence[row_of(place0)] : -1;
#pragma unroll
    for (int i = 0; i < RPT; i++) {
      const unsigned next_place = place0 + i + 1;
      const int next = next_place < p.rows ? p.row_sequence[row_of(next_place)] : -1;
      if (now >= 0) {
        inside |= 1u << i;
        if (now != before) begins |= 1u << i;
        if (now != next) ends |= 1u << i;
      }
      before = now;
      now = next;
    }
  } else {
    unsigned at = place0 % p.sequence_rows;  // the rows are whole sequences, so this holds in either direction
#pragma unroll
    for (int i = 0; i < RPT; i++) {
      if (place0 + i < p.rows) {
        inside |= 1u << i;
        if (at == 0) begins |= 1u << i;
        if (at == p.sequence_rows - 1) ends |= 1u << i;
      }
      at = at == p.sequence_rows - 1 ? 0 : at + 1;
    }
  }
  auto sequence_at = [&](int i) {
    const unsigned row = row_of(place0 + i);
    return p.row_sequence ? (unsigned)p.row_sequence[row] : row / p.sequence_rows;
  };

  // all loads first
  uint4_t cx[RPT], cg[RPT], ch[BACK ? RPT : 1], cd[BACK ? RPT : 1];
#pragma unroll
  for (int i = 0; i < RPT; i++) {
    const int n = (inside >> i) & 1u ? count : 0;
    const size_t row = n > 0 ? row_of(place0 + i) : 0;
    cg[i] = load_chunk_of<DT, ALIGNED>(p.g, row * p.g_stride + channel, n);
    if constexpr (!BACK || GATE == kGateSigmoid) cx[i] = load_chunk_of<DT, ALIGNED>(p.x, row * p.x_stride + channel, n);
    if constexpr (BACK) {
      cd[i] = load_chunk_of<DT, ALIGNED>(p.dh, row * p.dh_stride + channel, n);
      const int nh = (ends >> i) & 1u ? 0 : n;  // the row in front of a sequence's first one is another sequence's
      ch[i] = load_chunk_of<DT, ALIGNED>(p.h, (nh > 0 ? row - 1 : 0) * p.h_stride + channel, nh);
    }
  }
  // a, b of every place (b: what the place adds to the state; where a sequence begins, with its seed) and the aggregate
  float a[RPT][V], b[RPT][V], A[V], B[V];
#pragma unroll
  for (int e = 0; e < V; e++) {
    A[e] = 1.0f;
    B[e] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < RPT; i++) {
    const bool in = (inside >> i) & 1u, first = (begins >> i) & 1u;
    float g[V], x[V], seed[V];
    unpack_chunk<DT>(cg[i], g);
    unpack_chunk<DT>(BACK ? cd[BACK ? i : 0] : cx[i], x);
    if (first && p.seed) {
      load_floats<V, ALIGNED>(p.seed, (size_t)sequence_at(i) * p.channels + channel, count, seed);
    } else {
#pragma unroll
      for (int e = 0; e < V; e++) seed[e] = 0.0f;
    }
#pragma unroll
    for (int e = 0; e < V; e++) {
      float keep;
      gate_of<DT, GATE>(g[e], &a[i][e], &keep);
      if constexpr (BACK) {
        b[i][e] = first ? x[e] + seed[e] : x[e];  // delta without the carry; the state is u = a delta
        if (in) {
          B[e] = a[i][e] * (first ? b[i][e] : b[i][e] + B[e]);
          A[e] = first ? 0.0f : a[i][e] * A[e];
        }
      } else {
        b[i][e] = GATE == kGateSigmoid ? keep * x[e] : x[e];
        if (first) b[i][e] = __builtin_fmaf(a[i][e], seed[e], b[i][e]);
        if (in) {
          B[e] = first ? b[i][e] : __builtin_fmaf(a[i][e], B[e], b[i][e]);
          A[e] = first ? 0.0f : a[i][e] * A[e];
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V / 4; i++) {
    *reinterpret_cast<float4_t *>(&lds_a[group * TC + lane * V + 4 * i]) = float4_t{A[4 * i], A[4 * i + 1], A[4 * i + 2], A[4 * i + 3]};
    *reinterpret_cast<float4_t *>(&lds_b[group * TC + lane * V + 4 * i]) = float4_t{B[4 * i], B[4 * i + 1], B[4 * i + 2], B[4 * i + 3]};
  }
  // a place outside every sequence ends what came before it, too: what follows it begins a sequence
  const unsigned outside = ~inside & ((1u << RPT) - 1u);
  if (lane == 0) lds_reset[group] = (begins ? 1u : 0u) | ((begins & 1u) || (outside & 1u) ? 2u : 0u);
  __syncthreads();
  if (tid < TC) {
    const bool exists = strip * TC + tid < p.channels;
    float TA = 1.0f, TB = 0.0f;
    bool own_state = false;
#pragma unroll
    for (int j = 0; j < GROUPS; j++) {
      const bool reset = lds_reset[j] & 1u;
      const float ga = lds_a[j * TC + tid], gb = lds_b[j * TC + tid];
      TB = reset ? gb : __builtin_fmaf(ga, TB, gb);
      TA = reset ? 0.0f : ga * TA;
      own_state = own_state || reset;
    }
    float state = 0.0f;
    if (p.ticket && exists) state = exchange_carry(p, chunk, strip, TC, tid, TA, TB, own_state, (lds_reset[0] & 2u) == 0);
#pragma unroll
    for (int j = 0; j < GROUPS; j++) {
      const bool reset = lds_reset[j] & 1u;
      const float ga = lds_a[j * TC + tid], gb = lds_b[j * TC + tid];
      lds_a[j * TC + tid] = state;  // from here on: the state in front of the group
      state = reset ? gb : __builtin_fmaf(ga, state, gb);
    }
  }
  __syncthreads();
  float state[V];
#pragma unroll
  for (int i = 0; i < V / 4; i++) {
    const float4_t s = *reinterpret_cast<const float4_t *>(&lds_a[group * TC + lane * V + 4 * i]);
#pragma unroll
    for (int e = 0; e < 4; e++) state[4 * i + e] = s[e];
  }
#pragma unroll
  for (int i = 0; i < RPT; i++) {
    const bool in = (inside >> i) & 1u, first = (begins >> i) & 1u, end = (ends >> i) & 1u;
    const int n = in || (p.zero_outside && place0 + i < p.rows) ? count : 0;
    const size_t row = n > 0 ? row_of(place0 + i) : 0;
    if constexpr (BACK) {
      float h[V], x[V], dx[V], dg[V];
      unpack_chunk<DT>(ch[i], h);
      if (end && p.h0) load_floats<V, ALIGNED>(p.h0, (size_t)sequence_at(i) * p.channels + channel, count, h);
      if constexpr (GATE == kGateSigmoid) unpack_chunk<DT>(cx[i], x);
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float delta = first ? b[i][e] : b[i][e] + state[e];
        if (in) state[e] = a[i][e] * delta;
        dx[e] = delta;
        dg[e] = delta * h[e];
        if constexpr (GATE == kGateLog) dg[e] *= a[i][e];
        if constexpr (GATE == kGateSigmoid) {
          float g[V];
          unpack_chunk<DT>(cg[i], g);
          float s, keep;
          sigmoid_pair<DT == kF32>(g[e], &s, &keep);
          dx[e] = keep * delta;
          dg[e] = delta * (h[e] - x[e]) * (s * keep);
        }
      }
      if (!in) {
#pragma unroll
        for (int e = 0; e < V; e++) dx[e] = dg[e] = 0.0f;
      }
      store_chunk_of<DT, ALIGNED>(p.out, row * p.out_stride + channel, n, dx);
      store_chunk_of<DT, ALIGNED>(p.out_g, row * p.out_g_stride + channel, n, dg);
    } else {
#pragma unroll
      for (int e = 0; e < V; e++) state[e] = !in ? 0.0f : first ? b[i][e] : __builtin_fmaf(a[i][e], state[e], b[i][e]);  // behind a row of no sequence another one begins
      store_chunk_of<DT, ALIGNED>(p.out, row * p.out_stride + channel, n, state);
    }
    if (end && p.last) store_floats<V, ALIGNED>(p.last, (size_t)sequence_at(i) * p.channels + channel, count, state);
  }
}

// Ahead of the scan: clears the ticket and the descriptors, finds every row's sequence from the offsets (rows of no
// sequence get -1), and hands the seed of each empty sequence on as the state behind it.
struct GatedScanSetup {
  unsigned *head;          // 64 words: ticket, expired waits
  uint4_t *clear;          // descriptors
  size_t clear_chunks;     // 16-byte chunks of them
  const void *offsets;     // sequences + 1 of them, or null (then all sequences are empty, or none is)
  int offset_bits;
  unsigned sequences, rows, channels;
  int *row_sequence;
  const float *seed;
  float *last;
};
TCU_DEVICE long long offset_at(const GatedScanSetup &s, unsigned j) { return s.offset_bits == 32 ? (long long)static_cast<const int *>(s.offsets)[j] : static_cast<const long long *>(s.offsets)[j]; }

__global__ __launch_bounds__(256) inline void gated_scan_setup_kernel(GatedScanSetup s) {
  const size_t me = (size_t)blockIdx.x * blockDim.x + threadIdx.x, all = (size_t)gridDim.x * blockDim.x;
  if (me < 64) s.head[me] = 0u;
  for (size_t i = me; i < s.clear_chunks; i += all) s.clear[i] = uint4_t{0u, 0u, 0u, 0u};
  for (size_t r = me; s.offsets && r < s.rows; r += all) {
    unsigned lo = 0, hi = s.sequences;  // the last sequence that begins at or in front of the row is in [lo - 1, hi - 1]
    while (lo < hi) {
      const unsigned mid = lo + (hi - lo) / 2;
      if (offset_at(s, mid) <= (long long)r)
        lo = mid + 1;
      else
        hi = mid;
    }
    s.row_sequence[r] = lo > 0 && (long long)r < offset_at(s, lo) ? (int)lo - 1 : -1;
  }
  if (s.last && (s.offsets || s.rows == 0)) {
    // one block per sequence and round: most have tokens and are passed over after two reads
    for (unsigned j = blockIdx.x; j < s.sequences; j += gridDim.x) {
      if (s.rows != 0 && offset_at(s, j + 1) > offset_at(s, j)) continue;
      for (unsigned c = threadIdx.x; c < s.channels; c += blockDim.x) s.last[(size_t)j * s.channels + c] = s.seed ? s.seed[(size_t)j * s.channels + c] : 0.0f;
    }
  }
}

// One token for each of `rows` running sequences.  A block takes one row (and kStepThreads chunks of channels); rows that
// name the same slot are advanced one after the other, in row order, by the block of the first of them.
struct GatedStepParams {
  const void *x, *g;
  void *out;
  const float *state;
  float *new_state;
  const int *slots;  // null: row i uses slot i
  size_t x_stride, g_stride, out_stride;
  unsigned rows, num_slots, channels, chunks;  // chunks: blocks per row
  bool zero_padding;
};
constexpr int kStepThreads = 64;
template <int DT, int GATE, bool ALIGNED>
__global__ __launch_bounds__(kStepThreads) void gated_scan_step_kernel(GatedStepParams p) {
  constexpr int V = Elem<DT>::V;
  const unsigned row = blockIdx.x / p.chunks;
  const unsigned channel = ((blockIdx.x % p.chunks) * kStepThreads + threadIdx.x) * V;
  const int count = (int)p.channels - (int)channel;
  int slot = (int)row;
  uint4_t cg = load_chunk_of<DT, ALIGNED>(p.g, row * p.g_stride + channel, count);
  uint4_t cx = load_chunk_of<DT, ALIGNED>(p.x, row * p.x_stride + channel, count);
  bool again = false;
  if (p.slots) {
    slot = p.slots[row];
    if (slot < 0 || (unsigned)slot >= p.num_slots) {  // a row of padding: the whole block
      const float zero[V] = {};
      if (p.zero_padding) store_chunk_of<DT, ALIGNED, false>(p.out, row * p.out_stride + channel, count, zero);
      return;
    }
    bool earlier = false;
    for (unsigned base = 0; base < p.rows; base += kStepThreads) {
      const unsigned j = base + threadIdx.x;
      const bool same = j < p.rows && j != row && p.slots[j] == slot;
      earlier = earlier || ballot(same && j < row) != 0;
      again = again || ballot(same && j > row) != 0;
    }
    if (earlier) return;
  }
  float h[V];
  load_floats<V, ALIGNED>(p.state, (size_t)slot * p.channels + channel, count, h);
  unsigned at = row;
  while (true) {
    float g[V], x[V];
    unpack_chunk<DT>(cg, g);
    unpack_chunk<DT>(cx, x);
#pragma unroll
    for (int e = 0; e < V; e++) {
      float a, keep;
      gate_of<DT, GATE>(g[e], &a, &keep);
      h[e] = __builtin_fmaf(a, h[e], GATE == kGateSigmoid ? keep * x[e] : x[e]);
    }
    store_chunk_of<DT, ALIGNED, false>(p.out, at * p.out_stride + channel, count, h);
    if (!again) break;
    do at++;
    while (at < p.rows && p.slots[at] != slot);
    if (at >= p.rows) break;
    cg = load_chunk_of<DT, ALIGNED>(p.g, at * p.g_stride + channel, count);
    cx = load_chunk_of<DT, ALIGNED>(p.x, at * p.x_stride + channel, count);
  }
  store_floats<V, ALIGNED>(p.new_state, (size_t)slot * p.channels + channel, count, h);
}

}  // namespace tcu

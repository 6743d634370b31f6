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
// One pass over the data: a block takes a tile of TILE_ROWS places x TILE_CHANNELS channels into registers.  A thread has
// RPT consecutive places of one 16-byte chunk of channels and works out their (a, b) once (exponential and reciprocal are
// quarter-rate instructions) and the (A, B) of all of them; the groups of a wave combine theirs by lane exchanges, the waves
// in LDS; from the state in front of the tile every thread finishes from registers.  The bound is HBM traffic (2 streams in,
// 1 out; backwards 3 or 4 in, 2 out).
//
// Tiles that follow each other along the sequences hand the state on through entries in the workspace, one 64-bit word per
// channel, whole whenever it is seen, so that no fence is needed: an aggregate (A, B), or a state.  Every tile publishes its
// own aggregate, or, where a sequence begins inside it, the state behind it; every 8th tile the same for the 8 tiles it closes,
// which wait for nothing but each other; every 64th tile the state behind it, which waits for the state 64 tiles before.  A
// tile's carry is that state with at most 7 entries of 8 tiles and 7 entries of one tile applied in their order.  What is
// published and in which order it is combined depends on places alone, never on timing: the same input gives the same bits
// every time.  The chain of waits is a 64th of the tiles long (with every 8th tile handing a state on, 512 tiles along a
// sequence waited for a third of their time: 65536 x 2048 fp16, 390 us against 264 with the waits left out).
// Gates may be above 1, so a product of them may pass the range of fp32 where the states do not.  What is zero stays zero then
// (carried_over, joined_gates): a state of zero adds nothing however far the product has grown, and a product that has come down to
// zero is not raised again.  Everything else is left to the arithmetic: a state that is not zero under a product that has overflowed becomes an
// infinity or a NaN, never a finite number that is not the recurrence's.
// Tiles are handed out by a ticket, so the one that is waited for has always been started; a wait is bounded and leaves NaN
// in what depended on it.
//
// Calls in a row, set-up launch included: 65536 x 2048 fp16 178 us (805 MB, 4.5 TB/s; a copy reaches 5.1), 8 x 4096 x 2048 bf16 97
// (403 MB, 4.1 TB/s), its gradient 165 (805 MB, 4.9 TB/s), 8191 x 1000 packed bf16 24 (49 MB; this kernel 19: 256 tiles, a block for
// each compute unit, bound by its own chain of load, combine, wait and store), 4099 x 769 packed fp32 backwards 27 (63 MB; this kernel 24:
// likewise, its rows beginning anywhere).
#pragma once

#include "elements.hpp"

namespace tcu {

constexpr int kGateDecay = 0, kGateLog = 1, kGateSigmoid = 2;  // tcu_gate
constexpr float kTameGates = 2147483648.0f;  // 2^31: the product of the four groups of a wave stays below 2^128
constexpr unsigned kScanGroup = 8;  // tiles that share an entry, and entries under one state

struct GatedScanParams {
  const void *x, *g, *h, *dh;  // x: also the input of the sigmoid gate's gradient; h: backwards only
  void *out, *out_g;           // h forwards; dx and dg backwards
  const float *seed;           // state in front of a sequence in place order: h0 / dh_last (may be null)
  const float *h0;             // backwards: h[-1] of the gradient's formulas (may be null)
  float *last;                 // state behind it: h_last / dh0 (may be null)
  const int *row_sequence;     // sequence of each row, -1 outside all; null: sequence_rows rows each
  size_t x_stride, g_stride, h_stride, dh_stride, out_stride, out_g_stride;  // elements from row to row
  unsigned rows, sequence_rows, channels, strips, chunks;
  bool near_rows;                  // 64 rows of any matrix lie within 4 GiB
  bool zero_outside;               // rows of no sequence: their outputs become 0, or are left as they are
  unsigned *ticket;                // null: one chunk of places, the block index is the tile
  unsigned long long *entries;     // [chunks + chunks / 8 + chunks / 64][strip][channel of the tile]
  unsigned poll_limit, mute_tile;  // mute_tile: tests only, tile mute_tile - 1 publishes nothing
  unsigned *expired;
};

// An entry: (A, B) as two fp32 words, or a state with kIsState in the place of A; kNoEntry before it is published.  Both marks
// are NaNs that no A carries: a NaN is published as the one the hardware makes.
constexpr unsigned kIsState = 0xfffffffeu, kQuietNaN = 0x7fc00000u;
constexpr unsigned long long kNoEntry = ~0ull;
TCU_DEVICE unsigned published_bits(float v) { return v != v ? kQuietNaN : __float_as_uint(v); }
TCU_DEVICE unsigned long long entry_of(bool is_state, float A, float B) { return ((unsigned long long)published_bits(B) << 32) | (is_state ? kIsState : published_bits(A)); }

// A h + B for a state h in front of the step (A, B), and the product of the gates of two steps: zero times an overflowed product is zero.
// Where no product has overflowed the plain forms say the same, and an overflow shows in all that is computed from it: so the plain
// ones are taken first, the others where something is not finite (65536 x 2048 fp16 1.7 us of 177; selects in the chain of waits 2.5).
template <bool CAREFUL>
TCU_DEVICE float carried_over(float A, float h, float B) { return CAREFUL && h == 0.0f ? B : __builtin_fmaf(A, h, B); }
template <bool CAREFUL>
TCU_DEVICE float joined_gates(float behind, float front) { return CAREFUL && front == 0.0f ? front : behind * front; }
TCU_DEVICE bool finite(float v) { return __builtin_fabsf(v) < __builtin_inff(); }
struct Plainly { static constexpr bool careful = false; };
struct Carefully { static constexpr bool careful = true; };

// (A, B), then an entry's step: a state replaces what came before it
struct ScanStep {
  float A, B;
  bool is_state;
};
TCU_DEVICE bool finite(const ScanStep &s) { return finite(s.A) && finite(s.B); }
// what `f` makes of its inputs, plainly if that is finite
template <typename F>
TCU_DEVICE auto settled(F &&f) {
  auto got = f(Plainly{});
  if (!finite(got)) got = f(Carefully{});
  return got;
}
template <bool CAREFUL>
TCU_DEVICE void apply_entry(ScanStep &s, unsigned long long w) {
  const bool state = (unsigned)w == kIsState;
  const float A = __uint_as_float((unsigned)w), B = __uint_as_float((unsigned)(w >> 32));
  s.B = state ? B : carried_over<CAREFUL>(A, s.B, B);
  s.A = state ? 0.0f : joined_gates<CAREFUL>(A, s.A);
  s.is_state = s.is_state || state;
}

template <int DT, int GATE>
TCU_DEVICE void gate_of(float g, float *a, float *keep) {  // keep = 1 - a (sigmoid only)
  *keep = 1.0f;
  if constexpr (GATE == kGateDecay) *a = g;
  if constexpr (GATE == kGateLog) *a = exp_of<DT == kF32>(g);
  if constexpr (GATE == kGateSigmoid) sigmoid_pair<DT == kF32>(g, a, keep);
}

// Reads those of the first `count` entries that have not been seen published yet; true if all have.
TCU_DEVICE bool read_entries(const unsigned long long *first, size_t stride, unsigned count, unsigned long long (&w)[kScanGroup]) {
#pragma unroll
  for (unsigned j = 0; j < kScanGroup; j++)
    if (j < count && w[j] == kNoEntry) w[j] = atomic_load_u64(first + j * stride);
  bool all = true;
#pragma unroll
  for (unsigned j = 0; j < kScanGroup; j++) all = all && !(j < count && w[j] == kNoEntry);
  return all;
}

// The carry into this tile for channel `c` of it; the tile's own step is `own`.  One thread per channel.
//   needs: the tile's first place continues a sequence
TCU_DEVICE float exchange_carry(const GatedScanParams &p, unsigned chunk, unsigned strip, int tile_channels, int c, const ScanStep &own, bool needs) {
  constexpr unsigned G = kScanGroup;
  const size_t stride = (size_t)p.strips * tile_channels;  // from chunk to chunk
  unsigned long long *tiles = p.entries + (size_t)strip * tile_channels + c;
  unsigned long long *groups = tiles + (size_t)p.chunks * stride, *states = groups + (size_t)(p.chunks / G) * stride;
  const unsigned group = chunk / G, in_group = chunk % G, super = group / G, in_super = group % G;
  const bool closes_group = in_group == G - 1, closes_super = closes_group && in_super == G - 1;
  const bool muted = p.mute_tile != 0 && chunk * p.strips + strip == p.mute_tile - 1;
  if (!closes_group && !muted) atomic_store_u64(tiles + chunk * stride, entry_of(own.is_state, own.A, own.B));
  if (!needs && !closes_group) return 0.0f;
  // everything this tile may have to know is asked for at once (one wait on memory instead of three)
  const unsigned long long *tile0 = tiles + (size_t)group * G * stride, *group0 = groups + (size_t)super * G * stride, *state0 = states + (size_t)(super > 0 ? super - 1 : 0) * stride;
  const unsigned tile_count = !own.is_state || needs ? in_group : 0u, group_count = needs ? in_super : 0u, state_count = needs && super > 0 ? 1u : 0u;
  unsigned long long w[G], v[G], u[G];
#pragma unroll
  for (unsigned j = 0; j < G; j++) w[j] = v[j] = u[j] = kNoEntry;
  bool have_tiles = read_entries(tile0, stride, tile_count, w), have_states = read_entries(state0, stride, state_count, u), have_groups = read_entries(group0, stride, group_count, v);
  unsigned polls = 0;
  for (; !have_tiles && polls < p.poll_limit; polls++) {
    spin_pause();
    have_tiles = read_entries(tile0, stride, tile_count, w);
  }
  const ScanStep front = settled([&](auto way) {  // the group's tiles in front of this one
    ScanStep s{1.0f, 0.0f, false};
#pragma unroll
    for (unsigned j = 0; j < G; j++)
      if (j < tile_count) apply_entry<decltype(way)::careful>(s, w[j]);
    return s;
  });
  const float bad = __builtin_nanf("");
  if (closes_group && !closes_super && !muted) {
    const ScanStep both = settled([&](auto way) {
      constexpr bool C = decltype(way)::careful;
      return ScanStep{joined_gates<C>(own.A, front.A), own.is_state ? own.B : carried_over<C>(own.A, front.B, own.B), own.is_state || front.is_state};
    });
    const bool known = have_tiles || own.is_state;
    atomic_store_u64(groups + (size_t)group * stride, entry_of(!known || both.is_state, both.A, known ? both.B : bad));
  }
  float carry = 0.0f;
  if (needs) {
    const bool behind = have_tiles && !front.is_state;  // what lies in front of the group matters
    for (; behind && !(have_states && have_groups) && polls < p.poll_limit; polls++) {
      spin_pause();
      have_states = read_entries(state0, stride, state_count, u);
      have_groups = read_entries(group0, stride, group_count, v);
    }
    carry = settled([&](auto way) {
      constexpr bool C = decltype(way)::careful;
      ScanStep s{0.0f, state_count ? __uint_as_float((unsigned)(u[0] >> 32)) : 0.0f, true};
#pragma unroll
      for (unsigned j = 0; j < G; j++)
        if (j < group_count) apply_entry<C>(s, v[j]);
      return front.is_state ? front.B : carried_over<C>(front.A, s.B, front.B);
    });
    if (!have_tiles || (behind && !(have_states && have_groups))) {
      carry = bad;
      if (c == 0 && p.expired) atomic_add_u32(p.expired, 1u);
    }
  }
  if (closes_super && !muted) {
    const float behind = settled([&](auto way) { return own.is_state ? own.B : carried_over<decltype(way)::careful>(own.A, carry, own.B); });
    atomic_store_u64(states + (size_t)super * stride, entry_of(true, 0.0f, behind));
  }
  return carry;
}

// Combines the steps of the wave's groups of TCL lanes: on return (A, B, reset) is the step of all of them, and
// (FA, FB, front_reset) that of the groups in front of the lane's own.  A lane exchange leaves the half in front in one
// register and the half behind in the other, in every lane.  PLAIN: no sequence begins in any of them, and no product of their A overflows.
template <int TCL, int V, bool PLAIN>
TCU_DEVICE void combine_groups(float (&A)[V], float (&B)[V], unsigned &reset, float (&FA)[V], float (&FB)[V], unsigned &front_reset) {
#pragma unroll
  for (int e = 0; e < V; e++) {
    FA[e] = 1.0f;
    FB[e] = 0.0f;
  }
  front_reset = 0;
  static_for<2>([&](auto step) {
    constexpr int D = TCL << decltype(step)::value;
    static_assert(D == 16 || D == 32, "groups of 16 lanes");
    const bool upper = (lane_id() & D) != 0;
    unsigned lo_reset = reset, hi_reset = reset;
    if constexpr (!PLAIN) swap_halves<D>(lo_reset, hi_reset);
#pragma unroll
    for (int e = 0; e < V; e++) {
      unsigned la = __float_as_uint(A[e]), ha = la, lb = __float_as_uint(B[e]), hb = lb;
      swap_halves<D>(la, ha);
      swap_halves<D>(lb, hb);
      const float lA = __uint_as_float(la), hA = __uint_as_float(ha), lB = __uint_as_float(lb), hB = __uint_as_float(hb);
      float nB, nA;
      if constexpr (PLAIN) {
        nB = __builtin_fmaf(FA[e], lB, FB[e]);
        nA = FA[e] * lA;
        B[e] = __builtin_fmaf(hA, lB, hB);
        A[e] = hA * lA;
      } else {
        nB = front_reset ? FB[e] : carried_over<true>(FA[e], lB, FB[e]);
        nA = front_reset ? 0.0f : joined_gates<true>(FA[e], lA);
        B[e] = hi_reset ? hB : carried_over<true>(hA, lB, hB);
        A[e] = hi_reset ? 0.0f : joined_gates<true>(hA, lA);
      }
      FB[e] = upper ? nB : FB[e];  // what lies in front of the group now begins with the other half
      FA[e] = upper ? nA : FA[e];
    }
    if constexpr (!PLAIN) {
      if (upper) front_reset |= lo_reset;
      reset = lo_reset | hi_reset;
    }
  });
}

// TCL lanes share a row of the tile (TCL * V channels); blocks of THREADS threads, RPT places per thread.
template <int DT, int GATE, bool BACK, bool ALIGNED, int TCL, int RPT, int THREADS>
__global__ __launch_bounds__(THREADS) void gated_scan_kernel(GatedScanParams p) {
  constexpr int V = Elem<DT>::V, TC = TCL * V, GROUPS = THREADS / TCL, TILE_ROWS = GROUPS * RPT, WAVES = THREADS / 64;
  static_assert(TC <= THREADS, "one thread per channel carries the state through the tile");
  __shared__ __attribute__((aligned(16))) float lds_a[WAVES * TC];  // a wave's step, then the state in front of the wave
  __shared__ __attribute__((aligned(16))) float lds_b[WAVES * TC];
  __shared__ unsigned lds_reset[WAVES];  // bit 0: a sequence begins in the wave's places, bit 1: the first of them continues none
  __shared__ unsigned lds_tile;
  const int tid = (int)threadIdx.x, lane = tid % TCL, group = tid / TCL;
  unsigned tile = blockIdx.x;
  if (p.ticket) {  // the same for every block of the launch
    if (tid == 0) lds_tile = atomic_add_u32(p.ticket, 1u);
    __syncthreads();
    tile = wave_uniform(lds_tile);
  }
  const unsigned chunk = tile / p.strips, strip = tile % p.strips;
  const unsigned place0 = chunk * TILE_ROWS + group * RPT;
  const unsigned channel = strip * TC + lane * V;
  const int count = (int)p.channels - (int)channel;  // channels of this chunk that exist (<= 0: none)

  // Where the wave's places are all there, a lane's addresses are one 32-bit offset from a base that the wave's rows share.
  const int wave = wave_in_block();
  constexpr int WAVE_GROUPS = 64 / TCL;
  const unsigned wave_place = wave_uniform(chunk * TILE_ROWS + wave * (WAVE_GROUPS * RPT));
  const unsigned wave_row = BACK ? p.rows - wave_place - WAVE_GROUPS * RPT : wave_place;  // the lowest of them
  const unsigned lane_row = (unsigned)(BACK ? WAVE_GROUPS - 1 - group % WAVE_GROUPS : group % WAVE_GROUPS) * RPT;
  const unsigned strip_at = wave_uniform(strip * TC);
  const unsigned lane_channel = count > 0 ? (unsigned)(lane * V) : 0u;  // a lane without channels reads the strip's first ones
  constexpr size_t E = sizeof(typename Elem<DT>::word_t);
  const bool fits = p.near_rows && (ALIGNED || strip * TC + TC <= p.channels) && wave_place + WAVE_GROUPS * RPT <= p.rows && (!BACK || wave_row > 0);  // the same for the whole wave
  // place i of the thread lies in row wave_row + lane_row + step_row(i)
  auto step_row = [](int i) { return BACK ? RPT - 1 - i : i; };
  auto plain_load = [&](const void *q, size_t stride, int row) {
    const char *base = static_cast<const char *>(q) + (((ptrdiff_t)wave_row + row) * (ptrdiff_t)stride + strip_at) * (ptrdiff_t)E;
    return load_at<ALIGNED>(base, (lane_row * (unsigned)stride + lane_channel) * (unsigned)E);
  };
  auto plain_store = [&](void *q, size_t stride, int row, const float (&v)[V]) {
    char *base = static_cast<char *>(q) + (((ptrdiff_t)wave_row + row) * (ptrdiff_t)stride + strip_at) * (ptrdiff_t)E;
    if (count > 0) store_at<ALIGNED>(base, (lane_row * (unsigned)stride + lane_channel) * (unsigned)E, pack_chunk<DT>(v));
  };

  constexpr bool KEEP = GATE == kGateSigmoid;
  uint4_t cg[BACK ? 1 : RPT], cin[BACK ? 1 : RPT];          // gate, input (backwards: within the branches below)
  uint4_t cx[BACK && KEEP ? RPT : 1], ch[BACK ? RPT : 1];  // what the gradient needs at the end
  auto load_all = [&](auto &gates, auto &inputs) {  // inputs: x, or dh
#pragma unroll
    for (int i = 0; i < RPT; i++) {
      gates[i] = plain_load(p.g, p.g_stride, step_row(i));
      inputs[i] = BACK ? plain_load(p.dh, p.dh_stride, step_row(i)) : plain_load(p.x, p.x_stride, step_row(i));
    }
    if constexpr (BACK) {
#pragma unroll
      for (int i = 0; i < RPT; i++) {
        ch[i] = plain_load(p.h, p.h_stride, step_row(i) - 1);
        if constexpr (KEEP) cx[i] = plain_load(p.x, p.x_stride, step_row(i));
      }
    }
  };
  // Forwards the loads go out before it is known which sequences the places belong to, which takes a load or two (65536 x 2048 fp16
  // 187 -> 173 us; backwards the registers do not suffice for that: 164 -> 233).
  if constexpr (!BACK) {
    if (fits) load_all(cg, cin);
  }

  // what each of the thread's places is: inside a sequence, the first or the last one of it in place order
  constexpr unsigned kAll = (1u << RPT) - 1u;
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
    if (at > 0 && at + RPT < p.sequence_rows) {
      inside = place0 < p.rows ? kAll : 0u;
    } else {
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
  }
  auto sequence_at = [&](int i) {
    const unsigned row = row_of(place0 + i);
    return p.row_sequence ? (unsigned)p.row_sequence[row] : row / p.sequence_rows;
  };

  // Most waves have places in the middle of one sequence only.  For them nothing has to be looked at place by place: the general
  // form takes 53 instruction slots per element, this one 26, and the kernel is bound by them as soon as it is not by memory.
  const bool plain = fits && ballot(inside != kAll || (begins | ends) != 0) == 0;
  float a[RPT][V], b[RPT][V], A[V], B[V];                  // b: what the place adds to the state; where a sequence begins, with its seed
  float keep[BACK && KEEP ? RPT : 1][V];
#pragma unroll
  for (int e = 0; e < V; e++) {
    A[e] = 1.0f;
    B[e] = 0.0f;
  }
  auto element = [&](int i, int e, float g, float x) {  // x: the input, or dh
    float k;
    gate_of<DT, GATE>(g, &a[i][e], &k);
    if constexpr (BACK) {
      b[i][e] = x;  // delta without the carry; the state is u = a delta
      if constexpr (KEEP) keep[i][e] = k;
    } else {
      b[i][e] = KEEP ? k * x : x;
    }
  };
  auto plain_steps = [&](auto &gates, auto &inputs) {
#pragma unroll
    for (int i = 0; i < RPT; i++) {
      float g[V], x[V];
      unpack_chunk<DT>(gates[i], g);
      unpack_chunk<DT>(inputs[i], x);
#pragma unroll
      for (int e = 0; e < V; e++) {
        element(i, e, g[e], x[e]);
        B[e] = BACK ? a[i][e] * (b[i][e] + B[e]) : __builtin_fmaf(a[i][e], B[e], b[i][e]);
        A[e] *= a[i][e];
      }
    }
  };
  auto load_some = [&](auto &gates, auto &inputs) {
#pragma unroll
    for (int i = 0; i < RPT; i++) {
      const int n = (inside >> i) & 1u ? count : 0;
      const size_t row = n > 0 ? row_of(place0 + i) : 0;
      gates[i] = load_chunk_of<DT, ALIGNED>(p.g, row * p.g_stride + channel, n);
      if constexpr (!BACK) inputs[i] = load_chunk_of<DT, ALIGNED>(p.x, row * p.x_stride + channel, n);
      if constexpr (BACK) {
        inputs[i] = load_chunk_of<DT, ALIGNED>(p.dh, row * p.dh_stride + channel, n);
        if constexpr (KEEP) cx[i] = load_chunk_of<DT, ALIGNED>(p.x, row * p.x_stride + channel, n);
        const int nh = (ends >> i) & 1u ? 0 : n;  // the row in front of a sequence's first one is another sequence's
        ch[i] = load_chunk_of<DT, ALIGNED>(p.h, (nh > 0 ? row - 1 : 0) * p.h_stride + channel, nh);
      }
    }
  };
  auto general_steps = [&](auto &gates, auto &inputs) {
#pragma unroll
    for (int i = 0; i < RPT; i++) {
      const bool in = (inside >> i) & 1u, first = (begins >> i) & 1u;
      float g[V], x[V], seed[V];
      unpack_chunk<DT>(gates[i], g);
      unpack_chunk<DT>(inputs[i], x);
      if (first && p.seed) {
        load_floats<V, ALIGNED>(p.seed, (size_t)sequence_at(i) * p.channels + channel, count, seed);
      } else {
#pragma unroll
        for (int e = 0; e < V; e++) seed[e] = 0.0f;
      }
#pragma unroll
      for (int e = 0; e < V; e++) {
        element(i, e, g[e], x[e]);
        if constexpr (BACK) {
          if (first) b[i][e] += seed[e];
          if (in) B[e] = a[i][e] * (first ? b[i][e] : b[i][e] + B[e]);
        } else {
          if (first) b[i][e] = __builtin_fmaf(a[i][e], seed[e], b[i][e]);
          if (in) B[e] = first ? b[i][e] : __builtin_fmaf(a[i][e], B[e], b[i][e]);
        }
        if (in) A[e] = first ? 0.0f : a[i][e] * A[e];
      }
    }
  };
  if constexpr (BACK) {
    uint4_t gates[RPT], inputs[RPT];
    if (plain) {
      load_all(gates, inputs);
      plain_steps(gates, inputs);
    } else {
      load_some(gates, inputs);
      general_steps(gates, inputs);
    }
  } else {
    if (!fits) load_some(cg, cin);
    if (plain) plain_steps(cg, cin);
    else general_steps(cg, cin);
  }
  unsigned reset = begins ? 1u : 0u, front_reset;
  float FA[V], FB[V];
  float largest = 0.0f;
#pragma unroll
  for (int e = 0; e < V; e++) largest = __builtin_fmaxf(largest, __builtin_fabsf(A[e]));  // (a NaN is in B as well, and passes either way)
  const bool tame = plain && ballot(largest > kTameGates) == 0;
  if (tame) combine_groups<TCL, V, true>(A, B, reset, FA, FB, front_reset);
  else combine_groups<TCL, V, false>(A, B, reset, FA, FB, front_reset);
  if (lane_id() < TCL) {
#pragma unroll
    for (int i = 0; i < V / 4; i++) {
      *reinterpret_cast<float4_t *>(&lds_a[wave * TC + lane * V + 4 * i]) = float4_t{A[4 * i], A[4 * i + 1], A[4 * i + 2], A[4 * i + 3]};
      *reinterpret_cast<float4_t *>(&lds_b[wave * TC + lane * V + 4 * i]) = float4_t{B[4 * i], B[4 * i + 1], B[4 * i + 2], B[4 * i + 3]};
    }
    // behind a place outside every sequence another one begins: nothing is carried over it
    if (lane == 0) lds_reset[wave] = reset | ((begins & 1u) || !(inside & 1u) ? 2u : 0u);
  }
  __syncthreads();
  if (tid < TC) {
    float ga[WAVES], gb[WAVES];
    unsigned gr[WAVES];
#pragma unroll
    for (int j = 0; j < WAVES; j++) {
      ga[j] = lds_a[j * TC + tid];
      gb[j] = lds_b[j * TC + tid];
      gr[j] = lds_reset[j];
    }
    const ScanStep own = settled([&](auto way) {
      constexpr bool C = decltype(way)::careful;
      ScanStep s{1.0f, 0.0f, false};
#pragma unroll
      for (int j = 0; j < WAVES; j++) {
        s.B = gr[j] & 1u ? gb[j] : carried_over<C>(ga[j], s.B, gb[j]);
        s.A = gr[j] & 1u ? 0.0f : joined_gates<C>(ga[j], s.A);
        s.is_state = s.is_state || (gr[j] & 1u);
      }
      return s;
    });
    float carry = 0.0f;
    if (p.ticket && strip * TC + tid < p.channels) carry = exchange_carry(p, chunk, strip, TC, tid, own, (gr[0] & 2u) == 0);
    auto hand_on = [&](auto way) {  // the sum is finite if all of the states are, a reset behind one that is not notwithstanding
      float s = carry, sum = 0.0f;
#pragma unroll
      for (int j = 0; j < WAVES; j++) {
        lds_a[j * TC + tid] = s;
        sum = __builtin_fmaf(s, 0.0f, sum);
        s = gr[j] & 1u ? gb[j] : carried_over<decltype(way)::careful>(ga[j], s, gb[j]);
      }
      return sum;
    };
    (void)settled(hand_on);
  }
  __syncthreads();
  float state[V];
#pragma unroll
  for (int i = 0; i < V / 4; i++) {
    const float4_t s = *reinterpret_cast<const float4_t *>(&lds_a[wave * TC + lane * V + 4 * i]);
#pragma unroll
    for (int e = 0; e < 4; e++) state[4 * i + e] = s[e];
  }
  if (tame) {
#pragma unroll
    for (int e = 0; e < V; e++) state[e] = __builtin_fmaf(FA[e], state[e], FB[e]);
  } else {
#pragma unroll
    for (int e = 0; e < V; e++) state[e] = front_reset ? FB[e] : carried_over<true>(FA[e], state[e], FB[e]);
  }
  auto gradients = [&](int i, int e, float delta, float h, float x, float *dx, float *dg) {
    if constexpr (KEEP) {
      *dx = keep[i][e] * delta;
      *dg = *dx * ((h - x) * a[i][e]);
    } else {
      *dx = delta;
      *dg = delta * h;
      if constexpr (GATE == kGateLog) *dg *= a[i][e];
    }
  };
  if (plain) {
#pragma unroll
    for (int i = 0; i < RPT; i++) {
      if constexpr (BACK) {
        float h[V], x[V], dx[V], dg[V];
        unpack_chunk<DT>(ch[i], h);
        if constexpr (KEEP) unpack_chunk<DT>(cx[i], x);
#pragma unroll
        for (int e = 0; e < V; e++) {
          const float delta = b[i][e] + state[e];
          state[e] = a[i][e] * delta;
          gradients(i, e, delta, h[e], KEEP ? x[e] : 0.0f, &dx[e], &dg[e]);
        }
        plain_store(p.out, p.out_stride, step_row(i), dx);
        plain_store(p.out_g, p.out_g_stride, step_row(i), dg);
      } else {
#pragma unroll
        for (int e = 0; e < V; e++) state[e] = __builtin_fmaf(a[i][e], state[e], b[i][e]);
        plain_store(p.out, p.out_stride, step_row(i), state);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < RPT; i++) {
    const bool in = (inside >> i) & 1u, first = (begins >> i) & 1u, end = (ends >> i) & 1u;
    const int n = in || (p.zero_outside && place0 + i < p.rows) ? count : 0;
    const size_t row = n > 0 ? row_of(place0 + i) : 0;
    if constexpr (BACK) {
      float h[V], x[V], dx[V], dg[V];
      unpack_chunk<DT>(ch[i], h);
      if (end) {  // the row in front is another sequence's
#pragma unroll
        for (int e = 0; e < V; e++) h[e] = 0.0f;
        if (p.h0) load_floats<V, ALIGNED>(p.h0, (size_t)sequence_at(i) * p.channels + channel, count, h);
      }
      if constexpr (KEEP) unpack_chunk<DT>(cx[i], x);
#pragma unroll
      for (int e = 0; e < V; e++) {
        const float delta = first ? b[i][e] : b[i][e] + state[e];
        if (in) state[e] = a[i][e] * delta;
        gradients(i, e, delta, h[e], KEEP ? x[e] : 0.0f, &dx[e], &dg[e]);
        if (!in) dx[e] = dg[e] = 0.0f;
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

// Ahead of the scan: clears the ticket and the entries, finds every row's sequence from the offsets (rows of no
// sequence get -1), and hands the seed of each sequence without rows on as the state behind it.
struct GatedScanSetup {
  unsigned *head;          // 64 words: ticket, expired waits
  uint4_t *clear;          // entries
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
  for (size_t i = me; i < s.clear_chunks; i += all) s.clear[i] = uint4_t{~0u, ~0u, ~0u, ~0u};  // kNoEntry
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
      if (s.rows != 0) {
        const long long from = offset_at(s, j), to = offset_at(s, j + 1);
        if ((from > 0 ? from : 0) < (to < (long long)s.rows ? to : (long long)s.rows)) continue;  // it has rows that exist
      }
      for (unsigned c = threadIdx.x; c < s.channels; c += blockDim.x) s.last[(size_t)j * s.channels + c] = s.seed ? s.seed[(size_t)j * s.channels + c] : 0.0f;
    }
  }
}

// One token for each of `rows` running sequences.  A block takes one row (and kStepThreads chunks of channels); rows that
// name the same slot are advanced one after the other, in row order, by the block of the first of them.  Every block looks through all
// slots for that, so the time grows with the square of the rows from some thousand on: 48 ... 512 rows of 2048 bf16 9 us a call (the
// host's), 2048 rows 21, 8192 rows 189, 32768 rows 2570 (without slots 10, 39 and 159).
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

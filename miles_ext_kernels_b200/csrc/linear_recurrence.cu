// Gated linear recurrence per channel over long or packed sequences, forward and backward, and its single-token step:
//     h[t] = a[t] h[t-1] + x[t],  a = exp(g),  y = h                    (h[-1] = h0 of the sequence, or zero)
//     dh[t] = dy[t] + a[t+1] dh[t+1],  dx = dh,  dg[t] = dh[t] a[t] h[t-1],  dh0 = a[0] dh[0]
// States in FP32, one rounding per output.
//
// One step is affine in the state, so a run of tokens is (A, B) with h_out = A h_in + B.  A block owns 128 tokens of 64
// channels: a warp takes 16 tokens (a lane two channels), folds them to (A, B) in registers, and the warps' pairs
// chain through shared memory.  A state is always folded left to right, tile by tile, h <- A h + B: whoever does it
// gets the same bits.  A sequence's first token makes the run independent of what came before; its pair is marked
// (A < 0) and the fold then takes B alone, so nothing of a sequence -- not even an infinity -- reaches the next one.
#include "common.cuh"
#include "rowio.cuh"

namespace mek {

constexpr int kGlrTokens = 16;                       // tokens a warp folds
constexpr int kGlrWarps = 8;
constexpr int kGlrTile = kGlrTokens * kGlrWarps;     // tokens a block owns
constexpr int kGlrChannels = 64;                     // channels a block owns
constexpr float kGlrReset = -1.0f;                   // A of a run that holds a sequence's first token

// exp(g) from its Taylor series about zero after a reduction by multiples of log 2: the last operation rounds 1 + p once,
// so a decay next to one carries no bias.  (CUDA's expf is off by up to an ulp to one side there, and a thousand tokens'
// memory adds that up: relative error of a state 7e-6 with expf, 4e-7 with this.)  The remainder of degree 7 at
// |r| <= log(2) / 2 is below 6e-9.  Below -87 the result is zero, above log(FLT_MAX) infinity; NaN stays NaN.
__device__ __forceinline__ float decay_of(float g) {
  const float n = __fadd_rn(fmaf(g, 1.44269504f, 12582912.f), -12582912.f);  // nearest integer
  float r = fmaf(n, -0.693359375f, g);                                       // log 2 in two parts, the first exact
  r = fmaf(n, 2.12194440e-4f, r);
  float q = fmaf(r, 1.f / 5040.f, 1.f / 720.f);
  q = fmaf(q, r, 1.f / 120.f);
  q = fmaf(q, r, 1.f / 24.f);
  q = fmaf(q, r, 1.f / 6.f);
  q = fmaf(q, r, 0.5f);
  const float p = fmaf(r * r, q, r);
  const float e = __int_as_float(__float_as_int(1.f + p) + (int(n) << 23));
  return g < -87.f ? 0.f : g > 88.7228f ? __int_as_float(0x7f800000) : e;
}

__device__ __forceinline__ float fold(float A, float B, float h) { return A < 0.f ? B : fmaf(A, h, B); }

// Where sequences lie: dense batches (cu = NULL: row b is sequence b, all T tokens) or one packed row.
struct Sequences {
  const int32_t* cu;  // [count + 1] or NULL
  int count, tokens;
};

// How many of cu's entries are below t; every lane of the warp gets it.  Whatever cu holds, 0 <= result <= entries.
__device__ __forceinline__ int entries_below(const int32_t* __restrict__ cu, int entries, int t) {
  const int lane = threadIdx.x & 31;
  int base = 0, end = entries;
  while (base < end) {
    const int step = (end - base + 31) / 32;
    const int at = base + (lane + 1) * step - 1;
    const int blocks = __popc(__ballot_sync(0xffffffffu, at < end && cu[at] < t));
    base += blocks * step;
    if (step == 1) break;
    end = min(end, base + step - 1);  // the entry at base + step - 1 is not below t
  }
  return min(base, entries);
}
// The sequence of token t of batch row b.
__device__ __forceinline__ int sequence_of(const Sequences& s, int b, int t) {
  if (s.cu == nullptr) return b;
  return min(max(entries_below(s.cu, s.count + 1, t + 1) - 1, 0), s.count - 1);
}

// The boundaries among tokens t0 .. t0 + 16 (bit j: a sequence starts, or the last one has ended, at t0 + j) and the
// tokens [lo, hi) that belong to a sequence.
struct Span {
  uint32_t bounds;
  int lo, hi;
  __device__ __forceinline__ bool starts(int j) const { return (bounds >> j) & 1; }
  __device__ __forceinline__ bool ends(int j) const { return (bounds >> (j + 1)) & 1; }
};
__device__ __forceinline__ Span span_of(const Sequences& s, int t0) {
  Span span{0u, 0, s.tokens};
  if (s.cu == nullptr) {
    if (t0 == 0) span.bounds = 1u;
    const int last = s.tokens - t0;
    if (last >= 0 && last <= kGlrTokens) span.bounds |= 1u << last;
    return span;
  }
  const int lane = threadIdx.x & 31;
  span.lo = max(s.cu[0], 0), span.hi = min(s.cu[s.count], s.tokens);
  for (int i = entries_below(s.cu, s.count + 1, t0); i <= s.count; i += 32) {
    const int at = i + lane <= s.count ? min(s.cu[i + lane], s.tokens) : 0x7fffffff;
    const bool in = at >= t0 && at <= t0 + kGlrTokens;
    span.bounds |= __reduce_or_sync(0xffffffffu, in ? 1u << (at - t0) : 0u);
    if (__ballot_sync(0xffffffffu, in) != 0xffffffffu) break;
  }
  return span;
}

// Two channels of a lane: neighbours (one access) when the rows allow it, else 32 apart.
template <bool kPair>
__device__ __forceinline__ int channel_of(int c0, int i) {
  const int lane = threadIdx.x & 31;
  return kPair ? c0 + 2 * lane + i : c0 + lane + 32 * i;
}
template <typename T, bool kPair>
__device__ __forceinline__ void load2(const T* __restrict__ row, int c0, int channels, float (&v)[2]) {
  if constexpr (kPair) {
    const int c = channel_of<true>(c0, 0);
    v[0] = v[1] = 0.f;
    if (c < channels) unpack(*reinterpret_cast<const Vec<T, 2>*>(row + c), v);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = channel_of<false>(c0, i);
      v[i] = c < channels ? to_float(row[c]) : 0.f;
    }
  }
}
template <typename T, bool kPair>
__device__ __forceinline__ void store2(T* __restrict__ row, int c0, int channels, const float (&v)[2]) {
  if constexpr (kPair) {
    const int c = channel_of<true>(c0, 0);
    if (c < channels) *reinterpret_cast<Vec<T, 2>*>(row + c) = pack<T, 2>(v);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = channel_of<false>(c0, i);
      if (c < channels) row[c] = from_float<T>(v[i]);
    }
  }
}

template <typename T>
struct Rows {  // [batch, tokens, channels] with strides between batches and tokens
  T* base;
  int64_t batch_stride, token_stride;
  __device__ __forceinline__ T* row(int b, int t) const { return base + b * batch_stride + t * token_stride; }
};

struct GlrShape {
  Sequences seq;
  int batch, tokens, channels, tiles, channel_blocks;
};
struct GlrTileAt {
  int b, tile, c0;
};
// Block -> (tile, channel block, batch): tiles vary slowest, so the first tiles of all chains run first.
__device__ __forceinline__ GlrTileAt tile_at(const GlrShape& s, int64_t index) {
  const int chains = s.channel_blocks * s.batch;
  const int chain = int(index % chains);
  return {chain / s.channel_blocks, int(index / chains), (chain % s.channel_blocks) * kGlrChannels};
}
__device__ __forceinline__ int64_t state_at(const GlrShape& s, const GlrTileAt& at, int tile, int c) {
  return (int64_t(at.b) * s.tiles + tile) * s.channels + c;
}

// This warp's 16 tokens: decays and inputs in registers.
template <typename X, typename G, bool kPair>
__device__ __forceinline__ void load_tokens(const Rows<const X>& x, const Rows<const G>& g, const GlrShape& s,
                                            const GlrTileAt& at, int t0, float (&xv)[kGlrTokens][2],
                                            float (&a)[kGlrTokens][2]) {
#pragma unroll
  for (int j = 0; j < kGlrTokens; ++j) {
    if (t0 + j < s.tokens) {
      load2<X, kPair>(x.row(at.b, t0 + j), at.c0, s.channels, xv[j]);
      load2<G, kPair>(g.row(at.b, t0 + j), at.c0, s.channels, a[j]);
    } else {
      xv[j][0] = xv[j][1] = a[j][0] = a[j][1] = 0.f;  // a token past the end changes nothing
    }
  }
#pragma unroll
  for (int j = 0; j < kGlrTokens; ++j) a[j][0] = decay_of(a[j][0]), a[j][1] = decay_of(a[j][1]);
}
template <bool kPair>
__device__ __forceinline__ void load_state(const float* __restrict__ state, const GlrShape& s, const GlrTileAt& at,
                                           int seq, float (&h)[2]) {
  if (state != nullptr) load2<float, kPair>(state + int64_t(seq) * s.channels, at.c0, s.channels, h);
  else h[0] = h[1] = 0.f;
}

// (A, B) of the warp's tokens.
template <bool kPair>
__device__ __forceinline__ void fold_tokens(const float (&xv)[kGlrTokens][2], const float (&a)[kGlrTokens][2],
                                            const Span& span, const float* __restrict__ h0, const GlrShape& s,
                                            const GlrTileAt& at, int t0, float (&A)[2], float (&B)[2]) {
  A[0] = A[1] = 1.f, B[0] = B[1] = 0.f;
  const uint32_t starts = span.bounds & ((1u << kGlrTokens) - 1);
#pragma unroll
  for (int j = 0; j < kGlrTokens; ++j) {
    if ((starts >> j) & 1) {  // uniform over the warp
      load_state<kPair>(h0, s, at, sequence_of(s.seq, at.b, t0 + j), B);
      A[0] = A[1] = kGlrReset;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      B[i] = fmaf(a[j][i], B[i], xv[j][i]);
      A[i] = A[i] < 0.f ? A[i] : A[i] * a[j][i];
    }
  }
}

// mode 0: the tiles' pairs to agg [2, batch, tiles, channels]; mode 1: y (and final states) from the tiles' entering
// states (ends of the tiles before).
template <typename X, typename G, bool kPair, int kMode>
__global__ void __launch_bounds__(kGlrWarps * 32) glr_fwd_kernel(Rows<const X> x, Rows<const G> g, Rows<X> y,
                                                                 GlrShape s, const float* __restrict__ h0,
                                                                 float* __restrict__ agg,
                                                                 const float* __restrict__ ends,
                                                                 float* __restrict__ final_state) {
  __shared__ float2 s_A[kGlrWarps][32], s_B[kGlrWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const GlrTileAt at = tile_at(s, blockIdx.x);
  const int t0 = at.tile * kGlrTile + warp * kGlrTokens;
  float xv[kGlrTokens][2], a[kGlrTokens][2], A[2], B[2];
  load_tokens<X, G, kPair>(x, g, s, at, t0, xv, a);
  const Span span = span_of(s.seq, t0);
  fold_tokens<kPair>(xv, a, span, h0, s, at, t0, A, B);
  s_A[warp][lane] = make_float2(A[0], A[1]), s_B[warp][lane] = make_float2(B[0], B[1]);
  __syncthreads();
  if constexpr (kMode == 0) {
    if (warp != 0) return;
    for (int w = 1; w < kGlrWarps; ++w) {
      const float2 A2 = s_A[w][lane], B2 = s_B[w][lane];
      B[0] = fold(A2.x, B2.x, B[0]), B[1] = fold(A2.y, B2.y, B[1]);
      A[0] = A[0] < 0.f || A2.x < 0.f ? kGlrReset : A[0] * A2.x;
      A[1] = A[1] < 0.f || A2.y < 0.f ? kGlrReset : A[1] * A2.y;
    }
    float* row = agg + state_at(s, at, at.tile, 0);
    store2<float, kPair>(row, at.c0, s.channels, A);
    store2<float, kPair>(row + int64_t(s.batch) * s.tiles * s.channels, at.c0, s.channels, B);
    return;
  } else {
    float h[2] = {0.f, 0.f};
    if (at.tile > 0) load2<float, kPair>(ends + state_at(s, at, at.tile - 1, 0), at.c0, s.channels, h);
    for (int w = 0; w < warp; ++w) {
      const float2 A2 = s_A[w][lane], B2 = s_B[w][lane];
      h[0] = fold(A2.x, B2.x, h[0]), h[1] = fold(A2.y, B2.y, h[1]);
    }
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) {
      const int t = t0 + j;
      if (t >= s.tokens) break;
      if (span.starts(j)) load_state<kPair>(h0, s, at, sequence_of(s.seq, at.b, t), h);
#pragma unroll
      for (int i = 0; i < 2; ++i) h[i] = fmaf(a[j][i], h[i], xv[j][i]);
      const bool in = t >= span.lo && t < span.hi;
      const float out[2] = {in ? h[0] : 0.f, in ? h[1] : 0.f};
      store2<X, kPair>(y.row(at.b, t), at.c0, s.channels, out);
      if (final_state != nullptr && in && span.ends(j))
        store2<float, kPair>(final_state + int64_t(sequence_of(s.seq, at.b, t)) * s.channels, at.c0, s.channels, h);
    }
  }
}

// ends[b, tile] = the state after the tile (forward) or the adjoint that leaves it to the left (reverse).
__global__ void __launch_bounds__(256) glr_carry_kernel(const float* __restrict__ agg, float* __restrict__ ends,
                                                        GlrShape s, int reverse) {
  const int64_t at = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (at >= int64_t(s.batch) * s.channels) return;
  const int64_t first = at / s.channels * s.tiles * s.channels + at % s.channels;
  const float* B = agg + int64_t(s.batch) * s.tiles * s.channels;
  float h = 0.f;
  for (int k = 0; k < s.tiles; ++k) {
    const int64_t i = first + int64_t(reverse ? s.tiles - 1 - k : k) * s.channels;
    h = fold(agg[i], B[i], h);
    ends[i] = h;
  }
}

// Sequences without tokens pass their state through: out[seq] = in[seq] (or zero).
__global__ void __launch_bounds__(256) glr_empty_kernel(const int32_t* __restrict__ cu, int tokens, int channels,
                                                        const float* __restrict__ in, float* __restrict__ out) {
  const int seq = blockIdx.x;
  if (cu[seq] < min(cu[seq + 1], tokens)) return;
  for (int c = threadIdx.x; c < channels; c += 256)
    out[int64_t(seq) * channels + c] = in ? in[int64_t(seq) * channels + c] : 0.f;
}

template <typename X, typename G, bool kPair, int kMode>
__global__ void __launch_bounds__(kGlrWarps * 32) glr_bwd_kernel(Rows<const X> dy, Rows<const X> x, Rows<const G> g,
                                                                 Rows<X> dx, Rows<G> dg, GlrShape s,
                                                                 const float* __restrict__ h0,
                                                                 const float* __restrict__ d_final,
                                                                 const float* __restrict__ ends,
                                                                 float* __restrict__ agg,
                                                                 const float* __restrict__ adjoints,
                                                                 float* __restrict__ dh0) {
  __shared__ float2 s_A[kGlrWarps][32], s_B[kGlrWarps][32], s_D[kGlrWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const GlrTileAt at = tile_at(s, blockIdx.x);
  const int t0 = at.tile * kGlrTile + warp * kGlrTokens;
  float xv[kGlrTokens][2], a[kGlrTokens][2], dyv[kGlrTokens][2];
  load_tokens<X, G, kPair>(x, g, s, at, t0, xv, a);
#pragma unroll
  for (int j = 0; j < kGlrTokens; ++j) {
    dyv[j][0] = dyv[j][1] = 0.f;
    if (t0 + j < s.tokens) load2<X, kPair>(dy.row(at.b, t0 + j), at.c0, s.channels, dyv[j]);
  }
  const Span span = span_of(s.seq, t0);
  // the adjoint that leaves the warp's first token to the left: D + A c for the c that enters at its last
  float R[2] = {1.f, 1.f}, D[2] = {0.f, 0.f};
#pragma unroll
  for (int j = kGlrTokens - 1; j >= 0; --j) {
    if (span.ends(j) && t0 + j < s.tokens) {
      load_state<kPair>(d_final, s, at, sequence_of(s.seq, at.b, t0 + j), D);
      R[0] = R[1] = kGlrReset;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      D[i] = a[j][i] * (dyv[j][i] + D[i]);
      R[i] = R[i] < 0.f ? R[i] : R[i] * a[j][i];
    }
  }
  if constexpr (kMode == 0) {
    s_A[warp][lane] = make_float2(R[0], R[1]), s_D[warp][lane] = make_float2(D[0], D[1]);
    __syncthreads();
    if (warp != kGlrWarps - 1) return;
    for (int w = kGlrWarps - 2; w >= 0; --w) {
      const float2 A2 = s_A[w][lane], D2 = s_D[w][lane];
      D[0] = fold(A2.x, D2.x, D[0]), D[1] = fold(A2.y, D2.y, D[1]);
      R[0] = R[0] < 0.f || A2.x < 0.f ? kGlrReset : R[0] * A2.x;
      R[1] = R[1] < 0.f || A2.y < 0.f ? kGlrReset : R[1] * A2.y;
    }
    float* row = agg + state_at(s, at, at.tile, 0);
    store2<float, kPair>(row, at.c0, s.channels, R);
    store2<float, kPair>(row + int64_t(s.batch) * s.tiles * s.channels, at.c0, s.channels, D);
  } else {
    __shared__ float2 s_R[kGlrWarps][32];
    float A[2], B[2];
    fold_tokens<kPair>(xv, a, span, h0, s, at, t0, A, B);
    s_R[warp][lane] = make_float2(R[0], R[1]), s_D[warp][lane] = make_float2(D[0], D[1]);
    s_A[warp][lane] = make_float2(A[0], A[1]), s_B[warp][lane] = make_float2(B[0], B[1]);
    __syncthreads();
    float h[2] = {0.f, 0.f}, c[2] = {0.f, 0.f};
    if (at.tile > 0) load2<float, kPair>(ends + state_at(s, at, at.tile - 1, 0), at.c0, s.channels, h);
    if (at.tile + 1 < s.tiles) load2<float, kPair>(adjoints + state_at(s, at, at.tile + 1, 0), at.c0, s.channels, c);
    for (int w = 0; w < warp; ++w) {
      const float2 A2 = s_A[w][lane], B2 = s_B[w][lane];
      h[0] = fold(A2.x, B2.x, h[0]), h[1] = fold(A2.y, B2.y, h[1]);
    }
    for (int w = kGlrWarps - 1; w > warp; --w) {
      const float2 A2 = s_R[w][lane], D2 = s_D[w][lane];
      c[0] = fold(A2.x, D2.x, c[0]), c[1] = fold(A2.y, D2.y, c[1]);
    }
    // xv[j] becomes the state before token j
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) {
      if (span.starts(j) && t0 + j < s.tokens) load_state<kPair>(h0, s, at, sequence_of(s.seq, at.b, t0 + j), h);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float next = fmaf(a[j][i], h[i], xv[j][i]);
        xv[j][i] = h[i];
        h[i] = next;
      }
    }
#pragma unroll
    for (int j = kGlrTokens - 1; j >= 0; --j) {
      const int t = t0 + j;
      if (t >= s.tokens) continue;
      if (span.ends(j)) load_state<kPair>(d_final, s, at, sequence_of(s.seq, at.b, t), c);
      const bool in = t >= span.lo && t < span.hi;
      float dxv[2], dgv[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float dh = dyv[j][i] + c[i];
        c[i] = a[j][i] * dh;
        dxv[i] = in ? dh : 0.f;
        dgv[i] = in ? c[i] * xv[j][i] : 0.f;
      }
      store2<X, kPair>(dx.row(at.b, t), at.c0, s.channels, dxv);
      store2<G, kPair>(dg.row(at.b, t), at.c0, s.channels, dgv);
      if (dh0 != nullptr && in && span.starts(j))
        store2<float, kPair>(dh0 + int64_t(sequence_of(s.seq, at.b, t)) * s.channels, at.c0, s.channels, c);
    }
  }
}

// One token of every row: state[slot[r]] = a state[slot[r]] + x, y = the new state.  A row whose slot is outside the pool
// leaves every state alone and gets zeros.  Rows that name one slot take their turns in row order: the first of them
// does the work of all.
template <typename X, typename G, typename I, int V>
__global__ void __launch_bounds__(256) glr_step_kernel(const X* __restrict__ x, int64_t x_stride,
                                                       const G* __restrict__ g, int64_t g_stride,
                                                       float* __restrict__ state, int64_t state_stride,
                                                       const I* __restrict__ slots, X* __restrict__ y, int rows,
                                                       int pool, int channels) {
  const int r = blockIdx.x, c = (blockIdx.y * 256 + threadIdx.x) * V;
  const int64_t slot = slots ? int64_t(slots[r]) : r;
  const bool mine = c < channels, in = slot >= 0 && slot < pool;
  float h[V];
  if (!in) {
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = 0.f;
    if (mine) *reinterpret_cast<Vec<X, V>*>(y + int64_t(r) * channels + c) = pack<X, V>(h);
    return;
  }
  Vec<X, V> xr;
  Vec<G, V> gr;
  Vec<float, V> hr;
  if (mine) {
    xr = *reinterpret_cast<const Vec<X, V>*>(x + r * x_stride + c);
    gr = *reinterpret_cast<const Vec<G, V>*>(g + r * g_stride + c);
    hr = *reinterpret_cast<const Vec<float, V>*>(state + slot * state_stride + c);
  }
  bool again = false;
  if (slots) {
    bool before = false;
    for (int k = threadIdx.x; k < rows; k += 256) {
      const bool same = int64_t(slots[k]) == slot;
      before |= same && k < r, again |= same && k > r;
    }
    if (__syncthreads_or(before)) return;
    again = __syncthreads_or(again);
  }
  if (!mine) return;
  unpack(hr, h);
  for (int k = r;;) {
    float xv[V], gv[V];
    unpack(xr, xv), unpack(gr, gv);
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = fmaf(decay_of(gv[i]), h[i], xv[i]);
    *reinterpret_cast<Vec<X, V>*>(y + int64_t(k) * channels + c) = pack<X, V>(h);
    if (!again) break;
    do ++k; while (k < rows && int64_t(slots[k]) != slot);
    if (k >= rows) break;
    xr = *reinterpret_cast<const Vec<X, V>*>(x + k * x_stride + c);
    gr = *reinterpret_cast<const Vec<G, V>*>(g + k * g_stride + c);
  }
  *reinterpret_cast<Vec<float, V>*>(state + slot * state_stride + c) = pack<float, V>(h);
}

}  // namespace mek

namespace {

using namespace mek;

int check_glr(const char* what, int x_type, int g_type, int64_t batch, int64_t tokens, int64_t channels, int64_t seqs,
              const void* cu) {
  if (x_type < 0 || x_type > 2 || g_type < 0 || g_type > 2)
    return fail(MEK_ERR_UNSUPPORTED, "%s: an element type is 0 (bf16), 1 (fp16) or 2 (fp32)", what);
  if (batch <= 0 || tokens <= 0 || channels <= 0 || tokens > (1ll << 30) || channels > (1 << 24) || batch > (1 << 24))
    return fail(MEK_ERR_INVALID, "%s: batch, tokens and channels must be positive and tokens at most 2^30", what);
  if (cu != nullptr && (batch != 1 || seqs <= 0 || seqs > (1 << 30)))
    return fail(MEK_ERR_INVALID, "%s: packed sequences lie in one batch row", what);
  const int64_t tiles = (tokens + kGlrTile - 1) / kGlrTile, blocks = (channels + kGlrChannels - 1) / kGlrChannels;
  if (tiles * blocks * batch > 0x7fffffff) return fail(MEK_ERR_INVALID, "%s: more than 2^31 tiles", what);
  return MEK_OK;
}
GlrShape glr_shape(int64_t batch, int64_t tokens, int64_t channels, int64_t seqs, const int32_t* cu) {
  return {{cu, int(cu ? seqs : batch), int(tokens)}, int(batch), int(tokens), int(channels),
          int((tokens + kGlrTile - 1) / kGlrTile), int((channels + kGlrChannels - 1) / kGlrChannels)};
}
int size_of(int type) { return type == kTypeFp32 ? 4 : 2; }
bool pairs(const void* p, int type, int64_t a, int64_t b) {
  return reinterpret_cast<uintptr_t>(p) % (2 * size_of(type)) == 0 && a % 2 == 0 && b % 2 == 0;
}

// CALL(X, G) for the element types x_type, g_type.
#define MEK_GLR_TYPES(CALL)                                                      \
  do {                                                                           \
    switch (x_type * 3 + g_type) {                                               \
      case 0: return CALL(__nv_bfloat16, __nv_bfloat16);                         \
      case 1: return CALL(__nv_bfloat16, __half);                                \
      case 2: return CALL(__nv_bfloat16, float);                                 \
      case 3: return CALL(__half, __nv_bfloat16);                                \
      case 4: return CALL(__half, __half);                                       \
      case 5: return CALL(__half, float);                                        \
      case 6: return CALL(float, __nv_bfloat16);                                 \
      case 7: return CALL(float, __half);                                        \
      default: return CALL(float, float);                                        \
    }                                                                            \
  } while (0)

struct GlrFwd {
  const void *x, *g;
  void* y;
  int64_t xb, xt, gb, gt;
  const float* h0;
  float *agg, *ends, *final_state;
};
template <typename X, typename G, bool kPair>
int glr_fwd(const GlrFwd& p, const GlrShape& s, cudaStream_t stream) {
  const Rows<const X> x{static_cast<const X*>(p.x), p.xb, p.xt};
  const Rows<const G> g{static_cast<const G*>(p.g), p.gb, p.gt};
  const Rows<X> y{static_cast<X*>(p.y), int64_t(s.tokens) * s.channels, s.channels};
  const unsigned grid = unsigned(s.tiles) * s.channel_blocks * s.batch;
  if (s.tiles > 1) {
    glr_fwd_kernel<X, G, kPair, 0><<<grid, kGlrWarps * 32, 0, stream>>>(x, g, y, s, p.h0, p.agg, nullptr, nullptr);
    glr_carry_kernel<<<unsigned((int64_t(s.batch) * s.channels + 255) / 256), 256, 0, stream>>>(p.agg, p.ends, s, 0);
  }
  glr_fwd_kernel<X, G, kPair, 1><<<grid, kGlrWarps * 32, 0, stream>>>(x, g, y, s, p.h0, nullptr, p.ends, p.final_state);
  return launched("linear_recurrence_fwd");
}
struct GlrBwd {
  const void *dy, *x, *g;
  void *dx, *dg;
  int64_t xb, xt, gb, gt;
  const float *h0, *d_final, *ends;
  float *agg, *adjoints, *dh0;
};
template <typename X, typename G, bool kPair>
int glr_bwd(const GlrBwd& p, const GlrShape& s, cudaStream_t stream) {
  const int64_t dense = int64_t(s.tokens) * s.channels;
  const Rows<const X> dy{static_cast<const X*>(p.dy), dense, s.channels}, x{static_cast<const X*>(p.x), p.xb, p.xt};
  const Rows<const G> g{static_cast<const G*>(p.g), p.gb, p.gt};
  const Rows<X> dx{static_cast<X*>(p.dx), dense, s.channels};
  const Rows<G> dg{static_cast<G*>(p.dg), dense, s.channels};
  const unsigned grid = unsigned(s.tiles) * s.channel_blocks * s.batch;
  if (s.tiles > 1) {
    glr_bwd_kernel<X, G, kPair, 0><<<grid, kGlrWarps * 32, 0, stream>>>(dy, x, g, dx, dg, s, p.h0, p.d_final, p.ends,
                                                                        p.agg, nullptr, nullptr);
    glr_carry_kernel<<<unsigned((int64_t(s.batch) * s.channels + 255) / 256), 256, 0, stream>>>(p.agg, p.adjoints, s, 1);
  }
  glr_bwd_kernel<X, G, kPair, 1><<<grid, kGlrWarps * 32, 0, stream>>>(dy, x, g, dx, dg, s, p.h0, p.d_final, p.ends,
                                                                      nullptr, p.adjoints, p.dh0);
  return launched("linear_recurrence_bwd");
}

int glr_empty(const GlrShape& s, const float* in, float* out, cudaStream_t stream) {
  if (s.seq.cu == nullptr || out == nullptr) return MEK_OK;
  glr_empty_kernel<<<unsigned(s.seq.count), 256, 0, stream>>>(s.seq.cu, s.tokens, s.channels, in, out);
  return launched("linear_recurrence (sequences without tokens)");
}

struct GlrStep {
  const void *x, *g, *slots;
  void* y;
  float* state;
  int64_t xs, gs, ss;
  int rows, pool, channels, wide;
  bool slots64;
};
template <typename X, typename G, typename I, int V>
int glr_step_of(const GlrStep& p, cudaStream_t stream) {
  const dim3 grid(unsigned(p.rows), unsigned((p.channels + 256 * V - 1) / (256 * V)));
  glr_step_kernel<X, G, I, V><<<grid, 256, 0, stream>>>(static_cast<const X*>(p.x), p.xs, static_cast<const G*>(p.g),
                                                        p.gs, p.state, p.ss, static_cast<const I*>(p.slots),
                                                        static_cast<X*>(p.y), p.rows, p.pool, p.channels);
  return launched("linear_recurrence_step");
}
template <typename X, typename G>
int glr_step(const GlrStep& p, cudaStream_t stream) {
  if (p.slots64) return p.wide ? glr_step_of<X, G, int64_t, 4>(p, stream) : glr_step_of<X, G, int64_t, 1>(p, stream);
  return p.wide ? glr_step_of<X, G, int32_t, 4>(p, stream) : glr_step_of<X, G, int32_t, 1>(p, stream);
}

}  // namespace

extern "C" {

int mek_linear_recurrence_tile(void) { return kGlrTile; }

int mek_linear_recurrence_fwd(const void* x, int x_type, const void* g, int g_type, void* y, int64_t batch,
                              int64_t tokens, int64_t channels, int64_t x_batch_stride, int64_t x_token_stride,
                              int64_t g_batch_stride, int64_t g_token_stride, const int32_t* cu_seqlens, int64_t num_seqs,
                              const float* initial_state, float* final_state, float* scratch, float* ends,
                              void* stream) {
  if (!x || !g || !y) return fail(MEK_ERR_INVALID, "linear_recurrence_fwd: a null pointer");
  if (int rc = check_glr("linear_recurrence_fwd", x_type, g_type, batch, tokens, channels, num_seqs, cu_seqlens)) return rc;
  if (tokens > kGlrTile && (!scratch || !ends)) return fail(MEK_ERR_INVALID, "linear_recurrence_fwd: no scratch");
  const GlrShape s = glr_shape(batch, tokens, channels, num_seqs, cu_seqlens);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const GlrFwd p{x, g, y, x_batch_stride, x_token_stride, g_batch_stride, g_token_stride, initial_state, scratch, ends, final_state};
  if (int rc = glr_empty(s, initial_state, final_state, st)) return rc;
  const bool pair = channels % 2 == 0 && pairs(x, x_type, x_batch_stride, x_token_stride) &&
                    pairs(g, g_type, g_batch_stride, g_token_stride) && pairs(y, x_type, 0, 0) &&
                    pairs(initial_state, kTypeFp32, 0, 0) && pairs(final_state, kTypeFp32, 0, 0) &&
                    pairs(scratch, kTypeFp32, 0, 0) && pairs(ends, kTypeFp32, 0, 0);
#define MEK_GLR_FWD(X, G) (pair ? glr_fwd<X, G, true>(p, s, st) : glr_fwd<X, G, false>(p, s, st))
  MEK_GLR_TYPES(MEK_GLR_FWD);
}

int mek_linear_recurrence_bwd(const void* dy, const void* x, int x_type, const void* g, int g_type, void* dx, void* dg,
                              int64_t batch, int64_t tokens, int64_t channels, int64_t x_batch_stride,
                              int64_t x_token_stride, int64_t g_batch_stride, int64_t g_token_stride,
                              const int32_t* cu_seqlens, int64_t num_seqs, const float* initial_state,
                              const float* d_final_state, const float* ends, float* dh0, float* scratch, void* stream) {
  if (!dy || !x || !g || !dx || !dg) return fail(MEK_ERR_INVALID, "linear_recurrence_bwd: a null pointer");
  if (int rc = check_glr("linear_recurrence_bwd", x_type, g_type, batch, tokens, channels, num_seqs, cu_seqlens)) return rc;
  if (tokens > kGlrTile && (!scratch || !ends)) return fail(MEK_ERR_INVALID, "linear_recurrence_bwd: no scratch");
  const GlrShape s = glr_shape(batch, tokens, channels, num_seqs, cu_seqlens);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  float* adjoints = scratch ? scratch + 2 * int64_t(s.batch) * s.tiles * s.channels : nullptr;
  const GlrBwd p{dy, x, g, dx, dg, x_batch_stride, x_token_stride, g_batch_stride, g_token_stride, initial_state, d_final_state, ends,
                 scratch, adjoints, dh0};
  if (int rc = glr_empty(s, d_final_state, dh0, st)) return rc;
  const bool pair = channels % 2 == 0 && pairs(x, x_type, x_batch_stride, x_token_stride) &&
                    pairs(g, g_type, g_batch_stride, g_token_stride) && pairs(dy, x_type, 0, 0) &&
                    pairs(dx, x_type, 0, 0) && pairs(dg, g_type, 0, 0) && pairs(initial_state, kTypeFp32, 0, 0) &&
                    pairs(d_final_state, kTypeFp32, 0, 0) && pairs(dh0, kTypeFp32, 0, 0) &&
                    pairs(scratch, kTypeFp32, 0, 0) && pairs(ends, kTypeFp32, 0, 0);
#define MEK_GLR_BWD(X, G) (pair ? glr_bwd<X, G, true>(p, s, st) : glr_bwd<X, G, false>(p, s, st))
  MEK_GLR_TYPES(MEK_GLR_BWD);
}

int mek_linear_recurrence_step(const void* x, int x_type, const void* g, int g_type, float* state, const void* slots,
                               int slots_are_int64, void* y, int64_t rows, int64_t pool, int64_t channels,
                               int64_t x_row_stride, int64_t g_row_stride, int64_t state_row_stride, void* stream) {
  if (!x || !g || !state || !y) return fail(MEK_ERR_INVALID, "linear_recurrence_step: a null pointer");
  if (x_type < 0 || x_type > 2 || g_type < 0 || g_type > 2)
    return fail(MEK_ERR_UNSUPPORTED, "linear_recurrence_step: an element type is 0 (bf16), 1 (fp16) or 2 (fp32)");
  if (rows <= 0 || rows > 0x7fffffff || channels <= 0 || channels > (1 << 23) || pool <= 0 || pool > 0x7fffffff)
    return fail(MEK_ERR_INVALID, "linear_recurrence_step: rows, channels and the pool's slots must be positive");
  if (!slots && rows > pool)
    return fail(MEK_ERR_INVALID, "linear_recurrence_step: %lld rows and %lld states without slots", (long long)rows, (long long)pool);
  auto wide = [](const void* p, int type, int64_t stride) {
    return reinterpret_cast<uintptr_t>(p) % (4 * size_of(type)) == 0 && stride % 4 == 0;
  };
  const GlrStep p{x, g, slots, y, state, x_row_stride, g_row_stride, state_row_stride, int(rows), int(pool), int(channels),
                  wide(x, x_type, x_row_stride) && wide(g, g_type, g_row_stride) &&
                      wide(state, kTypeFp32, state_row_stride) && wide(y, x_type, channels),
                  slots_are_int64 != 0};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define MEK_GLR_STEP(X, G) glr_step<X, G>(p, st)
  MEK_GLR_TYPES(MEK_GLR_STEP);
}

}  // extern "C"

// Gated linear recurrence per channel over long or packed sequences, forward and backward, and its single-token step:
//     h[t] = a[t] h[t-1] + x[t],  a = exp(g),  y = h                    (h[-1] = h0 of the sequence, or zero)
//     dh[t] = dy[t] + a[t+1] dh[t+1],  dx = dh,  dg[t] = dh[t] a[t] h[t-1],  dh0 = a[0] dh[0]
// States in FP32, one rounding per output.
//
// HBM-bound, so each direction is ONE pass over the tokens.  One step is affine in the state, so a run of tokens is
// (A, B) with h_out = A h_in + B.  A block owns a tile of 128 tokens x 64 channels: a warp takes 16 tokens (a lane two
// channels) into registers, folds them to (A, B), and the warps' pairs chain through shared memory.  Between tiles the
// state travels through a word (A, B) per tile and channel in global memory: a block publishes its tile's pair, looks
// back over its predecessors' words for the nearest one that already stands for a state, folds forward from it,
// publishes its own state and only then goes over its tokens (still in registers) a second time.
//
// A state is a pair that does not depend on what came before, marked A < 0 (a decay never is): the fold then takes B
// alone.  The same mark is set by a sequence's first token, so nothing of a sequence -- not even an infinity -- reaches
// the next one, and a tile that holds a boundary makes nobody behind it wait.  Whoever folds, from whichever
// published state, does the same operations h <- A h + B in tile order: the bits do not depend on the timing.
//
// Tiles are taken from a counter in the order of time (all channels' first tiles, then all second ones, ...), so a
// tile's predecessors have always been taken before it by a block that is running or done: no wait can be for good.
// Every wait is bounded all the same (one second); the carried state is then NaN.
#include "common.cuh"
#include "rowio.cuh"
#include "umma.cuh"

namespace mek {

constexpr int kGlrTokens = 16;                       // tokens a warp folds
constexpr int kGlrWarps = 8;
constexpr int kGlrTile = kGlrTokens * kGlrWarps;     // tokens a block owns
constexpr int kGlrChannels = 64;                     // channels a block owns
constexpr float kGlrReset = -1.0f;                   // A of a run that holds a sequence's first token

// Two FP32 numbers in one register pair: the packed operations halve the instructions of a lane's two channels.
typedef unsigned long long Two;
__device__ __forceinline__ Two two(float x, float y) {
  Two v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
  return v;
}
__device__ __forceinline__ Two two(float x) { return two(x, x); }
__device__ __forceinline__ float2 split(Two v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// exp(g) from its Taylor series about zero after a reduction by multiples of log 2: the last operation rounds 1 + p once,
// so a decay next to one carries no bias.  (CUDA's expf is off by up to an ulp to one side there, and a thousand tokens'
// memory adds that up: relative error of a state 7e-6 with expf, 4e-7 with this.)  The remainder of degree 7 at
// |r| <= log(2) / 2 is below 6e-9.  For |g| <= 87; the nearest integer n sits in the low bits of the shifted product, so
// 2^n is added to the exponent with one multiply-add.
constexpr float kDecayRange = 87.f;
__device__ __forceinline__ Two decays_in_range(Two g) {
  const Two shifted = fma2(g, two(1.44269504f), two(12582912.f));
  const Two n = add2(shifted, two(-12582912.f));
  Two r = fma2(n, two(-0.693359375f), g);  // log 2 in two parts, the first exact
  r = fma2(n, two(2.12194440e-4f), r);
  Two q = fma2(r, two(1.f / 5040.f), two(1.f / 720.f));
  q = fma2(q, r, two(1.f / 120.f));
  q = fma2(q, r, two(1.f / 24.f));
  q = fma2(q, r, two(1.f / 6.f));
  q = fma2(q, r, two(0.5f));
  const float2 e = split(add2(fma2(mul2(r, r), q, r), two(1.f))), k = split(shifted);
  return two(__int_as_float(__float_as_int(k.x) * (1 << 23) + __float_as_int(e.x)),
             __int_as_float(__float_as_int(k.y) * (1 << 23) + __float_as_int(e.y)));
}
// Any g: below -87 the result is zero, above log(FLT_MAX) infinity; NaN stays NaN.
__device__ __forceinline__ float decay_fixed(float g, float e) {
  return g < -kDecayRange ? 0.f : g <= 88.7228f ? e : g + __int_as_float(0x7f800000);
}
__device__ __forceinline__ Two decays(Two g) {
  const float2 v = split(g), e = split(decays_in_range(g));
  return two(decay_fixed(v.x, e.x), decay_fixed(v.y, e.y));
}

__device__ __forceinline__ float fold(float A, float B, float h) { return A < 0.f ? B : fmaf(A, h, B); }
// (A, B), then (A2, B2)
__device__ __forceinline__ void chain(float& A, float& B, float A2, float B2) {
  B = fold(A2, B2, B);
  A = A < 0.f || A2 < 0.f ? kGlrReset : A * A2;
}

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
__device__ __forceinline__ Vec<T, 2> load2(const T* __restrict__ row, int c0, int channels) {
  Vec<T, 2> v;
  v.e[0] = v.e[1] = from_float<T>(0.f);
  if constexpr (kPair) {
    const int c = channel_of<true>(c0, 0);
    if (c < channels) v = *reinterpret_cast<const Vec<T, 2>*>(row + c);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = channel_of<false>(c0, i);
      if (c < channels) v.e[i] = row[c];
    }
  }
  return v;
}
template <typename T>
__device__ __forceinline__ Two widened(const Vec<T, 2>& v) { return two(to_float(v.e[0]), to_float(v.e[1])); }
template <typename T, bool kPair>
__device__ __forceinline__ void store2(T* __restrict__ row, int c0, int channels, Two value) {
  const float2 f = split(value);
  const float v[2] = {f.x, f.y};
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
  int window;        // words a warp looks back over at once
  int* counter;      // the last tile taken (-1 before the launch); NULL where there is one tile a chain
};
struct GlrTileAt {
  int b, tile, c0;
};
// The index-th tile in the order of time (from the end when reversed).
template <bool kReverse>
__device__ __forceinline__ GlrTileAt tile_at(const GlrShape& s, int index) {
  const int chains = s.channel_blocks * s.batch;
  const int chain = index % chains, step = index / chains;
  return {chain / s.channel_blocks, kReverse ? s.tiles - 1 - step : step, (chain % s.channel_blocks) * kGlrChannels};
}

// ---- the words between tiles: (A, B) per tile and channel, all ones before the launch -------------------------------
struct Words {  // of a lane's two channels
  float A0, B0, A1, B1;
  __device__ __forceinline__ bool set() const {
    return __float_as_uint(A0) != 0xffffffffu && __float_as_uint(A1) != 0xffffffffu;  // no operation makes this NaN
  }
  __device__ __forceinline__ bool state() const { return A0 < 0.f && A1 < 0.f; }
};
__device__ __forceinline__ float* words_at(float* words, const GlrShape& s, const GlrTileAt& at, int tile) {
  return words + (int64_t(at.b) * s.tiles + tile) * s.channels * 2;
}
// A word is read and written as one 64-bit access, so A and B always belong together.
template <bool kPair>
__device__ __forceinline__ Words load_words(const float* row, const GlrShape& s, int c0) {
  Two w[2] = {two(kGlrReset, 0.f), two(kGlrReset, 0.f)};
  if constexpr (kPair) {
    const int c = channel_of<true>(c0, 0);
    if (c < s.channels)
      asm volatile("ld.relaxed.gpu.global.v2.b64 {%0, %1}, [%2];" : "=l"(w[0]), "=l"(w[1]) : "l"(row + 2 * c) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = channel_of<false>(c0, i);
      if (c < s.channels) asm volatile("ld.relaxed.gpu.global.b64 %0, [%1];" : "=l"(w[i]) : "l"(row + 2 * c) : "memory");
    }
  }
  const float2 a = split(w[0]), b = split(w[1]);
  return {a.x, a.y, b.x, b.y};
}
template <bool kPair>
__device__ __forceinline__ void publish(float* row, const GlrShape& s, int c0, const Words& v) {
  const Two w[2] = {two(v.A0, v.B0), two(v.A1, v.B1)};
  if constexpr (kPair) {
    const int c = channel_of<true>(c0, 0);
    if (c < s.channels)
      asm volatile("st.relaxed.gpu.global.v2.b64 [%0], {%1, %2};" ::"l"(row + 2 * c), "l"(w[0]), "l"(w[1]) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = channel_of<false>(c0, i);
      if (c < s.channels) asm volatile("st.relaxed.gpu.global.b64 [%0], %1;" ::"l"(row + 2 * c), "l"(w[i]) : "memory");
    }
  }
}

struct GlrShared {
  float4 pairs[2][kGlrWarps][32];  // the warps' (A0, B0, A1, B1), forward and reverse
  int2 marks[kGlrWarps];           // nearest word not set, nearest state, among the words a warp looked at
  int ticket, late;
};
extern __shared__ float4 s_look[];  // [warps x window][32] words looked at

// The block's tile: the next in order, or its own index where tiles do not wait for one another.
template <bool kReverse>
__device__ __forceinline__ GlrTileAt take_tile(const GlrShape& s, GlrShared& sh) {
  if (s.counter == nullptr) return tile_at<kReverse>(s, blockIdx.x);
  if (threadIdx.x == 0) {
    sh.ticket = atomicAdd(s.counter, 1) + 1;
    sh.late = 0;
  }
  __syncthreads();
  return tile_at<kReverse>(s, sh.ticket);
}

// The state that enters the tile (from the left; reversed: the adjoint from the right), in every warp.  Called by the
// whole block after warp 0 has published the tile's own pair.
template <bool kPair, bool kReverse>
__device__ __forceinline__ void carry_in(float* words, const GlrShape& s, const GlrTileAt& at, GlrShared& sh, float (&h)[2]) {
  h[0] = h[1] = 0.f;
  const int before = kReverse ? s.tiles - 1 - at.tile : at.tile;  // tiles that come before this one
  if (before == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kFar = 0x7fffffff;
  const uint64_t began = global_timer_ns();
  int from;
  for (;;) {
    int unset = kFar, state = kFar;
    for (int k = warp * s.window; k < (warp + 1) * s.window; ++k) {
      Words v{kGlrReset, 0.f, kGlrReset, 0.f};  // before the first tile: a state of zero
      if (k < before) v = load_words<kPair>(words_at(words, s, at, kReverse ? at.tile + 1 + k : at.tile - 1 - k), s, at.c0);
      s_look[k * 32 + lane] = make_float4(v.A0, v.B0, v.A1, v.B1);
      if (!__all_sync(0xffffffffu, v.set())) unset = min(unset, k);
      else if (__all_sync(0xffffffffu, v.state())) state = min(state, k);
    }
    if (lane == 0) sh.marks[warp] = make_int2(unset, state);
    if (threadIdx.x == 0 && global_timer_ns() - began > kWaitLimitNs) sh.late = 1;
    __syncthreads();
    unset = from = kFar;
#pragma unroll
    for (int w = 0; w < kGlrWarps; ++w) unset = min(unset, sh.marks[w].x), from = min(from, sh.marks[w].y);
    const bool late = sh.late != 0;
    if (from < unset) break;
    if (late) {
      h[0] = h[1] = __int_as_float(0x7fffffff);
      return;
    }
    __syncthreads();  // before the words are looked at again
  }
  for (int k = from; k >= 0; --k) {
    const float4 v = s_look[k * 32 + lane];
    h[0] = fold(v.x, v.y, h[0]), h[1] = fold(v.z, v.w, h[1]);
  }
}

template <bool kPair>
__device__ __forceinline__ Two load_state(const float* __restrict__ state, const GlrShape& s, const GlrTileAt& at, int seq) {
  return state == nullptr ? two(0.f) : widened(load2<float, kPair>(state + int64_t(seq) * s.channels, at.c0, s.channels));
}

// The decays of the warp's tokens from their gates.
template <typename G>
__device__ __forceinline__ void to_decays(const Vec<G, 2> (&gv)[kGlrTokens], Two (&a)[kGlrTokens]) {
  bool plain = true;
#pragma unroll
  for (int j = 0; j < kGlrTokens; ++j) {
    const float2 v = split(widened(gv[j]));
    plain &= fabsf(v.x) <= kDecayRange && fabsf(v.y) <= kDecayRange;  // false for NaN
  }
  if (__all_sync(0xffffffffu, plain)) {
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) a[j] = decays_in_range(widened(gv[j]));
  } else {
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) a[j] = decays(widened(gv[j]));
  }
}

// (A, B) of the warp's tokens.
template <typename X, bool kPair>
__device__ __forceinline__ Words fold_tokens(const Vec<X, 2> (&xv)[kGlrTokens], const Two (&a)[kGlrTokens], const Span& span,
                                             const float* __restrict__ h0, const GlrShape& s, const GlrTileAt& at, int t0) {
  Two A = two(1.f), B = two(0.f);
  const int n = min(kGlrTokens, s.tokens - t0);
  const uint32_t starts = n > 0 ? span.bounds & ((1u << n) - 1) : 0u;
  if (starts == 0) {
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) A = mul2(A, a[j]), B = fma2(a[j], B, widened(xv[j]));
  } else {
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) {
      if ((starts >> j) & 1) B = load_state<kPair>(h0, s, at, sequence_of(s.seq, at.b, t0 + j));
      B = fma2(a[j], B, widened(xv[j]));
    }
    A = two(kGlrReset);
  }
  const float2 p = split(A), q = split(B);
  return {p.x, q.x, p.y, q.y};
}

__device__ __forceinline__ void chain(Words& v, const float4& w) {
  chain(v.A0, v.B0, w.x, w.y);
  chain(v.A1, v.B1, w.z, w.w);
}

template <typename X, typename G, bool kPair>
__global__ void __launch_bounds__(kGlrWarps * 32) glr_fwd_kernel(Rows<const X> x, Rows<const G> g, Rows<X> y, GlrShape s,
                                                                 const float* __restrict__ h0, float* words,
                                                                 float* __restrict__ final_state) {
  __shared__ GlrShared sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const GlrTileAt at = take_tile<false>(s, sh);
  const int t0 = at.tile * kGlrTile + warp * kGlrTokens;
  Vec<X, 2> xv[kGlrTokens];
  Two a[kGlrTokens];
  {
    Vec<G, 2> gv[kGlrTokens];
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) {
      const int t = min(t0 + j, s.tokens - 1);  // a token past the end changes nothing: nobody reads what it gives
      xv[j] = load2<X, kPair>(x.row(at.b, t), at.c0, s.channels);
      gv[j] = load2<G, kPair>(g.row(at.b, t), at.c0, s.channels);
    }
    to_decays(gv, a);
  }
  const Span span = span_of(s.seq, t0);
  const Words mine = fold_tokens<X, kPair>(xv, a, span, h0, s, at, t0);
  sh.pairs[0][warp][lane] = make_float4(mine.A0, mine.B0, mine.A1, mine.B1);
  __syncthreads();
  Words tile = mine;
  if (s.tiles > 1 && warp == 0) {
#pragma unroll
    for (int w = 1; w < kGlrWarps; ++w) chain(tile, sh.pairs[0][w][lane]);
    publish<kPair>(words_at(words, s, at, at.tile), s, at.c0, tile);
  }
  float in[2];
  carry_in<kPair, false>(words, s, at, sh, in);
  if (s.tiles > 1 && warp == 0 && !tile.state()) {
    publish<kPair>(words_at(words, s, at, at.tile), s, at.c0,
                   Words{kGlrReset, fold(tile.A0, tile.B0, in[0]), kGlrReset, fold(tile.A1, tile.B1, in[1])});
  }
  for (int w = 0; w < warp; ++w) {
    const float4 v = sh.pairs[0][w][lane];
    in[0] = fold(v.x, v.y, in[0]), in[1] = fold(v.z, v.w, in[1]);
  }
  Two h = two(in[0], in[1]);
  if (span.bounds == 0 && t0 >= span.lo && t0 + kGlrTokens <= span.hi) {  // all of one sequence, which goes on
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) {
      h = fma2(a[j], h, widened(xv[j]));
      store2<X, kPair>(y.row(at.b, t0 + j), at.c0, s.channels, h);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < kGlrTokens; ++j) {
    const int t = t0 + j;
    if (t < s.tokens) {
      if (span.starts(j)) h = load_state<kPair>(h0, s, at, sequence_of(s.seq, at.b, t));
      h = fma2(a[j], h, widened(xv[j]));
      const bool in_one = t >= span.lo && t < span.hi;
      store2<X, kPair>(y.row(at.b, t), at.c0, s.channels, in_one ? h : two(0.f));
      if (final_state != nullptr && in_one && span.ends(j))
        store2<float, kPair>(final_state + int64_t(sequence_of(s.seq, at.b, t)) * s.channels, at.c0, s.channels, h);
    }
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

// Tiles from the last to the first.  The states inside a tile are recomputed from the state that entered it, which the
// forward's words hold; the adjoint travels through words of its own.
template <typename X, typename G, bool kPair>
__global__ void __launch_bounds__(kGlrWarps * 32) glr_bwd_kernel(Rows<const X> dy, Rows<const X> x, Rows<const G> g,
                                                                 Rows<X> dx, Rows<G> dg, GlrShape s,
                                                                 const float* __restrict__ h0,
                                                                 const float* __restrict__ d_final,
                                                                 const float* __restrict__ states, float* words,
                                                                 float* __restrict__ dh0) {
  __shared__ GlrShared sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const GlrTileAt at = take_tile<true>(s, sh);
  const int t0 = at.tile * kGlrTile + warp * kGlrTokens;
  Vec<X, 2> xv[kGlrTokens], dyv[kGlrTokens];
  Two a[kGlrTokens];
  {
    Vec<G, 2> gv[kGlrTokens];
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) {
      const int t = min(t0 + j, s.tokens - 1);
      gv[j] = load2<G, kPair>(g.row(at.b, t), at.c0, s.channels);
      dyv[j] = load2<X, kPair>(dy.row(at.b, t), at.c0, s.channels);
      xv[j] = load2<X, kPair>(x.row(at.b, t), at.c0, s.channels);
    }
    to_decays(gv, a);
  }
  float h_in[2] = {0.f, 0.f};
  if (at.tile > 0) {
    const float* row = words_at(const_cast<float*>(states), s, at, at.tile - 1);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = channel_of<kPair>(at.c0, i);
      if (c < s.channels) h_in[i] = row[2 * c + 1];
    }
  }
  const Span span = span_of(s.seq, t0);
  const int n = min(max(s.tokens - t0, 0), kGlrTokens);
  // the adjoint that leaves the warp's first token to the left: D + R c for the c that enters at its last
  Words back;
  {
    Two R = two(1.f), D = two(0.f);
    const uint32_t ends = (span.bounds >> 1) & ((1u << n) - 1);
    if (ends == 0 && n == kGlrTokens) {
#pragma unroll
      for (int j = kGlrTokens - 1; j >= 0; --j) R = mul2(R, a[j]), D = mul2(a[j], add2(widened(dyv[j]), D));
    } else {
#pragma unroll
      for (int j = kGlrTokens - 1; j >= 0; --j) {
        if (j < n) {
          if (span.ends(j)) D = load_state<kPair>(d_final, s, at, sequence_of(s.seq, at.b, t0 + j));
          D = mul2(a[j], add2(widened(dyv[j]), D));
          R = mul2(R, a[j]);
        }
      }
      if (ends) R = two(kGlrReset);
    }
    const float2 p = split(R), q = split(D);
    back = {p.x, q.x, p.y, q.y};
  }
  sh.pairs[1][warp][lane] = make_float4(back.A0, back.B0, back.A1, back.B1);
  {
    const Words mine = fold_tokens<X, kPair>(xv, a, span, h0, s, at, t0);
    sh.pairs[0][warp][lane] = make_float4(mine.A0, mine.B0, mine.A1, mine.B1);
  }
  __syncthreads();
  if (s.tiles > 1 && warp == kGlrWarps - 1) {
#pragma unroll
    for (int w = kGlrWarps - 2; w >= 0; --w) chain(back, sh.pairs[1][w][lane]);
    publish<kPair>(words_at(words, s, at, at.tile), s, at.c0, back);
  }
  float c_in[2];
  carry_in<kPair, true>(words, s, at, sh, c_in);
  if (s.tiles > 1 && warp == kGlrWarps - 1 && !back.state()) {
    publish<kPair>(words_at(words, s, at, at.tile), s, at.c0,
                   Words{kGlrReset, fold(back.A0, back.B0, c_in[0]), kGlrReset, fold(back.A1, back.B1, c_in[1])});
  }
  for (int w = 0; w < warp; ++w) {
    const float4 v = sh.pairs[0][w][lane];
    h_in[0] = fold(v.x, v.y, h_in[0]), h_in[1] = fold(v.z, v.w, h_in[1]);
  }
  for (int w = kGlrWarps - 1; w > warp; --w) {
    const float4 v = sh.pairs[1][w][lane];
    c_in[0] = fold(v.x, v.y, c_in[0]), c_in[1] = fold(v.z, v.w, c_in[1]);
  }
  Two h = two(h_in[0], h_in[1]), c = two(c_in[0], c_in[1]);
  Two before[kGlrTokens];  // the state before every token
  if (span.bounds == 0 && t0 >= span.lo && t0 + kGlrTokens <= span.hi) {
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) before[j] = h, h = fma2(a[j], h, widened(xv[j]));
#pragma unroll
    for (int j = kGlrTokens - 1; j >= 0; --j) {
      const Two dh = add2(widened(dyv[j]), c);
      c = mul2(a[j], dh);
      store2<X, kPair>(dx.row(at.b, t0 + j), at.c0, s.channels, dh);
      store2<G, kPair>(dg.row(at.b, t0 + j), at.c0, s.channels, mul2(c, before[j]));
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < kGlrTokens; ++j) {
    if (j < n) {
      if (span.starts(j)) h = load_state<kPair>(h0, s, at, sequence_of(s.seq, at.b, t0 + j));
      before[j] = h, h = fma2(a[j], h, widened(xv[j]));
    }
  }
#pragma unroll
  for (int j = kGlrTokens - 1; j >= 0; --j) {
    const int t = t0 + j;
    if (j < n) {
      if (span.ends(j)) c = load_state<kPair>(d_final, s, at, sequence_of(s.seq, at.b, t));
      const bool in_one = t >= span.lo && t < span.hi;
      const Two dh = add2(widened(dyv[j]), c);
      c = mul2(a[j], dh);
      store2<X, kPair>(dx.row(at.b, t), at.c0, s.channels, in_one ? dh : two(0.f));
      store2<G, kPair>(dg.row(at.b, t), at.c0, s.channels, in_one ? mul2(c, before[j]) : two(0.f));
      if (dh0 != nullptr && in_one && span.starts(j))
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
    for (int i = 0; i < V; ++i) h[i] = fmaf(split(decays(two(gv[i]))).x, h[i], xv[i]);
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
// The window: words a warp looks back over, eight warps together.  With few chains (channel blocks x batch rows) the tiles
// in flight lie one behind the other, so the nearest state may be as many tiles back as there are blocks on the GPU
// per chain (3 x 148); with many chains it is near, and wide windows would only read more.
GlrShape glr_shape(int64_t batch, int64_t tokens, int64_t channels, int64_t seqs, const int32_t* cu) {
  GlrShape s{{cu, int(cu ? seqs : batch), int(tokens)}, int(batch), int(tokens), int(channels),
             int((tokens + kGlrTile - 1) / kGlrTile), int((channels + kGlrChannels - 1) / kGlrChannels), 1, nullptr};
  const int64_t chains = int64_t(s.batch) * s.channel_blocks, depth = (3 * 148 + chains - 1) / chains;
  s.window = int(depth <= kGlrWarps ? 1 : depth >= 8 * kGlrWarps ? 8 : (depth + kGlrWarps - 1) / kGlrWarps);
  return s;
}
size_t glr_look_bytes(const GlrShape& s) { return s.tiles > 1 ? size_t(s.window) * kGlrWarps * 32 * sizeof(float4) : 0; }
int64_t glr_words(const GlrShape& s) { return int64_t(s.batch) * s.tiles * s.channels * 2; }

// Words unset and the counter behind them at -1: one asynchronous fill with ones (nothing where a chain is one tile).
int glr_clear(const char* what, GlrShape& s, float* words, cudaStream_t stream) {
  if (s.tiles <= 1) return MEK_OK;
  s.counter = reinterpret_cast<int*>(words + glr_words(s));
  const cudaError_t err = cudaMemsetAsync(words, 0xff, size_t(glr_words(s) + 1) * sizeof(float), stream);
  return err == cudaSuccess ? MEK_OK : fail(MEK_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
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
  float *words, *final_state;
};
template <typename X, typename G, bool kPair>
int glr_fwd(const GlrFwd& p, const GlrShape& s, cudaStream_t stream) {
  const Rows<const X> x{static_cast<const X*>(p.x), p.xb, p.xt};
  const Rows<const G> g{static_cast<const G*>(p.g), p.gb, p.gt};
  const Rows<X> y{static_cast<X*>(p.y), int64_t(s.tokens) * s.channels, s.channels};
  const unsigned grid = unsigned(s.tiles) * s.channel_blocks * s.batch;
  glr_fwd_kernel<X, G, kPair><<<grid, kGlrWarps * 32, glr_look_bytes(s), stream>>>(x, g, y, s, p.h0, p.words, p.final_state);
  return launched("linear_recurrence_fwd");
}
struct GlrBwd {
  const void *dy, *x, *g;
  void *dx, *dg;
  int64_t xb, xt, gb, gt;
  const float *h0, *d_final, *states;
  float *words, *dh0;
};
template <typename X, typename G, bool kPair>
int glr_bwd(const GlrBwd& p, const GlrShape& s, cudaStream_t stream) {
  const int64_t dense = int64_t(s.tokens) * s.channels;
  const Rows<const X> dy{static_cast<const X*>(p.dy), dense, s.channels}, x{static_cast<const X*>(p.x), p.xb, p.xt};
  const Rows<const G> g{static_cast<const G*>(p.g), p.gb, p.gt};
  const Rows<X> dx{static_cast<X*>(p.dx), dense, s.channels};
  const Rows<G> dg{static_cast<G*>(p.dg), dense, s.channels};
  const unsigned grid = unsigned(s.tiles) * s.channel_blocks * s.batch;
  glr_bwd_kernel<X, G, kPair><<<grid, kGlrWarps * 32, glr_look_bytes(s), stream>>>(dy, x, g, dx, dg, s, p.h0, p.d_final,
                                                                                   p.states, p.words, p.dh0);
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
                              const float* initial_state, float* final_state, float* states, void* stream) {
  const char* what = "linear_recurrence_fwd";
  if (!x || !g || !y) return fail(MEK_ERR_INVALID, "%s: a null pointer", what);
  if (int rc = check_glr(what, x_type, g_type, batch, tokens, channels, num_seqs, cu_seqlens)) return rc;
  if (tokens > kGlrTile && !states) return fail(MEK_ERR_INVALID, "%s: no room for the tiles' states", what);
  GlrShape s = glr_shape(batch, tokens, channels, num_seqs, cu_seqlens);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const GlrFwd p{x, g, y, x_batch_stride, x_token_stride, g_batch_stride, g_token_stride, initial_state, states, final_state};
  const bool pair = channels % 2 == 0 && pairs(x, x_type, x_batch_stride, x_token_stride) &&
                    pairs(g, g_type, g_batch_stride, g_token_stride) && pairs(y, x_type, 0, 0) &&
                    pairs(initial_state, kTypeFp32, 0, 0) && pairs(final_state, kTypeFp32, 0, 0) &&
                    reinterpret_cast<uintptr_t>(states) % 16 == 0;
  if (reinterpret_cast<uintptr_t>(states) % 8 != 0) return fail(MEK_ERR_INVALID, "%s: states must be 8-byte aligned", what);
  if (int rc = glr_clear(what, s, states, st)) return rc;
  if (int rc = glr_empty(s, initial_state, final_state, st)) return rc;
#define MEK_GLR_FWD(X, G) (pair ? glr_fwd<X, G, true>(p, s, st) : glr_fwd<X, G, false>(p, s, st))
  MEK_GLR_TYPES(MEK_GLR_FWD);
}

int mek_linear_recurrence_bwd(const void* dy, const void* x, int x_type, const void* g, int g_type, void* dx, void* dg,
                              int64_t batch, int64_t tokens, int64_t channels, int64_t x_batch_stride,
                              int64_t x_token_stride, int64_t g_batch_stride, int64_t g_token_stride,
                              const int32_t* cu_seqlens, int64_t num_seqs, const float* initial_state,
                              const float* d_final_state, const float* states, float* dh0, float* scratch, void* stream) {
  const char* what = "linear_recurrence_bwd";
  if (!dy || !x || !g || !dx || !dg) return fail(MEK_ERR_INVALID, "%s: a null pointer", what);
  if (int rc = check_glr(what, x_type, g_type, batch, tokens, channels, num_seqs, cu_seqlens)) return rc;
  if (tokens > kGlrTile && (!scratch || !states)) return fail(MEK_ERR_INVALID, "%s: no scratch", what);
  GlrShape s = glr_shape(batch, tokens, channels, num_seqs, cu_seqlens);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const GlrBwd p{dy, x, g, dx, dg, x_batch_stride, x_token_stride, g_batch_stride, g_token_stride, initial_state,
                 d_final_state, states, scratch, dh0};
  const bool pair = channels % 2 == 0 && pairs(x, x_type, x_batch_stride, x_token_stride) &&
                    pairs(g, g_type, g_batch_stride, g_token_stride) && pairs(dy, x_type, 0, 0) &&
                    pairs(dx, x_type, 0, 0) && pairs(dg, g_type, 0, 0) && pairs(initial_state, kTypeFp32, 0, 0) &&
                    pairs(d_final_state, kTypeFp32, 0, 0) && pairs(dh0, kTypeFp32, 0, 0) &&
                    reinterpret_cast<uintptr_t>(scratch) % 16 == 0;
  if (reinterpret_cast<uintptr_t>(scratch) % 8 != 0) return fail(MEK_ERR_INVALID, "%s: scratch must be 8-byte aligned", what);
  if (int rc = glr_clear(what, s, scratch, st)) return rc;
  if (int rc = glr_empty(s, d_final_state, dh0, st)) return rc;
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

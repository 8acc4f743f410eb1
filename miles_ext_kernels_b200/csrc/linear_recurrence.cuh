// Gated linear recurrence per channel over long or packed sequences, forward and backward, and its single-token step:
//     h[t] = a[t] h[t-1] + x[t],  a = exp(g),  y = h                    (h[-1] = h0 of the sequence, or zero)
//     dh[t] = dy[t] + a[t+1] dh[t+1],  dx = dh,  dg[t] = dh[t] a[t] h[t-1],  dh0 = a[0] dh[0]
// States in FP32, one rounding per output.
//
// HBM-bound, so each direction is ONE pass over the tokens.  One step is affine in the state, so a run of tokens is
// (A, B) with h_out = A h_in + B.  A block owns a tile of 128 tokens x 64 channels: a warp takes 16 tokens (a lane two
// neighbouring channels), folds them to (A, B), and the warps' pairs chain through shared memory.  Between tiles the
// state travels through a word (A, B) per tile and channel in global memory: a block publishes its tile's pair, looks
// back over its predecessors' words for the nearest one that already stands for a state, folds forward from it,
// publishes its own state and only then goes over its tokens (still on chip) a second time.
//
// The tokens come by TMA, a box of 16 tokens x 64 channels per warp and tensor, and the outputs leave the same way from
// the place of the inputs: no thread computes an address per token (which took more instructions than the recurrence
// did), nothing is predicated, and what lies past the last token or channel arrives as zeros, a gate of zero and an
// input of zero, which change nothing.  Rows that TMA cannot address (16-byte strides) are moved by plain loads and
// stores into and out of the same shared tiles.
//
// A state is a pair that does not depend on what came before, marked A < 0 (a decay never is): the fold then takes B
// alone.  The same mark is set by a sequence's first token, so nothing of a sequence -- not even an infinity -- reaches
// the next one, and a tile that holds a boundary makes nobody behind it wait.  Whoever folds, from whichever
// published state, does the same operations h <- A h + B in tile order: the bits do not depend on the timing.
//
// Tiles are taken from a counter in the order of time (all channels' first tiles, then all second ones, ...), so a
// tile's predecessors have always been taken before it by a block that is running or done: no wait can be for good.
// Every wait is bounded all the same (one second); the carried state is then NaN.
#pragma once

#include "common.cuh"
#include "rowio.cuh"
#include "tma.cuh"
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

template <typename T>
__device__ __forceinline__ Two widened(const Vec<T, 2>& v) { return two(to_float(v.e[0]), to_float(v.e[1])); }
template <typename T>
__device__ __forceinline__ Vec<T, 2> narrowed(Two v) {
  const float2 f = split(v);
  const float a[2] = {f.x, f.y};
  return pack<T, 2>(a);
}

// One tensor [batch, tokens, channels] of a call: its map (kTma) or its base and strides (elements).
struct GlrTensor {
  void* base;
  int64_t batch_stride, token_stride;
};

struct GlrShape {
  Sequences seq;
  int batch, tokens, channels, tiles, channel_blocks;
  int window;        // words a warp looks back over at once
  int slice;         // bytes of a warp's part of the exchange area
  int exchange;      // where that area starts in dynamic shared memory
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

struct GlrShared {
  uint64_t arrived[kGlrWarps];  // a warp's boxes
  int2 marks[kGlrWarps];        // nearest word not set, nearest state, among the words a warp looked at
  int ticket, late;
};

// The block's tile -- the next in order, or its own index where tiles do not wait for one another -- and the barriers.
template <bool kReverse>
__device__ __forceinline__ GlrTileAt take_tile(const GlrShape& s, GlrShared& sh) {
  if (threadIdx.x == 0) {
    sh.ticket = s.counter ? atomicAdd(s.counter, 1) + 1 : int(blockIdx.x);
    sh.late = 0;
#pragma unroll
    for (int w = 0; w < kGlrWarps; ++w) mbar_init(&sh.arrived[w], 1);
    fence_mbar_init();
  }
  __syncthreads();
  return tile_at<kReverse>(s, sh.ticket);
}

// ---- tokens between global memory and a warp's shared tile [16][64] -------------------------------------------------
__device__ __forceinline__ void box_load(void* tile, const CUtensorMap* map, int c, int t, int b, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(tile)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c), "r"(t), "r"(b)
      : "memory");
}
__device__ __forceinline__ void box_store(const CUtensorMap* map, int c, int t, int b, const void* tile) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(tile)), "r"(c), "r"(t), "r"(b)
               : "memory");
}
template <typename T>
constexpr uint32_t kGlrBox = kGlrTokens * kGlrChannels * sizeof(T);

template <typename T>
__device__ __forceinline__ void plain_load(T* tile, const GlrTensor& g, const GlrShape& s, const GlrTileAt& at, int t0) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < kGlrChannels / 32; ++i) {
    const int c = at.c0 + 32 * i + lane;
    const T* from = static_cast<const T*>(g.base) + at.b * g.batch_stride + t0 * g.token_stride + c;
    T v[kGlrTokens];
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) {
      v[j] = from_float<T>(0.f);
      if (c < s.channels && t0 + j < s.tokens) v[j] = *from;
      from += g.token_stride;
    }
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) tile[j * kGlrChannels + 32 * i + lane] = v[j];
  }
}
template <typename T>
__device__ __forceinline__ void plain_store(const T* tile, const GlrTensor& g, const GlrShape& s, const GlrTileAt& at, int t0) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < kGlrChannels / 32; ++i) {
    const int c = at.c0 + 32 * i + lane;
    T* to = static_cast<T*>(g.base) + at.b * g.batch_stride + t0 * g.token_stride + c;
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) {
      if (c < s.channels && t0 + j < s.tokens) *to = tile[j * kGlrChannels + 32 * i + lane];
      to += g.token_stride;
    }
  }
}
// A lane's two channels of token j.
template <typename T>
__device__ __forceinline__ Vec<T, 2>& token(T* tile, int j) {
  return *reinterpret_cast<Vec<T, 2>*>(tile + j * kGlrChannels + 2 * (threadIdx.x & 31));
}

// ---- state vectors [rows, channels]: a lane's two channels -----------------------------------------------------------
template <bool kPair>
__device__ __forceinline__ Two load_state(const float* __restrict__ state, const GlrShape& s, const GlrTileAt& at, int row) {
  const int c = at.c0 + 2 * (threadIdx.x & 31);
  if (state == nullptr || c >= s.channels) return two(0.f);
  const float* p = state + int64_t(row) * s.channels + c;
  if constexpr (kPair) return widened(*reinterpret_cast<const Vec<float, 2>*>(p));
  return two(p[0], c + 1 < s.channels ? p[1] : 0.f);
}
template <bool kPair>
__device__ __forceinline__ void store_state(float* __restrict__ state, const GlrShape& s, const GlrTileAt& at, int row, Two v) {
  const int c = at.c0 + 2 * (threadIdx.x & 31);
  if (c >= s.channels) return;
  float* p = state + int64_t(row) * s.channels + c;
  if constexpr (kPair) {
    *reinterpret_cast<Vec<float, 2>*>(p) = narrowed<float>(v);
  } else {
    p[0] = split(v).x;
    if (c + 1 < s.channels) p[1] = split(v).y;
  }
}

// ---- the words between tiles: (A, B) per tile and channel, all ones before the launch --------------------------------
struct Words {  // of a lane's two channels
  float A0, B0, A1, B1;
  __device__ __forceinline__ bool set() const {
    return __float_as_uint(A0) != 0xffffffffu && __float_as_uint(A1) != 0xffffffffu;  // no operation makes this NaN
  }
  __device__ __forceinline__ bool state() const { return A0 < 0.f && A1 < 0.f; }
};
__device__ __forceinline__ float* words_at(float* words, const GlrShape& s, const GlrTileAt& at, int tile) {
  return words + ((int64_t(at.b) * s.tiles + tile) * s.channels + at.c0 + 2 * (threadIdx.x & 31)) * 2;
}
// A word is read and written as one 64-bit access, so A and B always belong together.
template <bool kPair>
__device__ __forceinline__ Words load_words(const float* row, const GlrShape& s, const GlrTileAt& at) {
  const int left = s.channels - at.c0 - 2 * int(threadIdx.x & 31);
  Two w[2] = {two(kGlrReset, 0.f), two(kGlrReset, 0.f)};
  if constexpr (kPair) {
    if (left > 0)
      asm volatile("ld.relaxed.gpu.global.v2.b64 {%0, %1}, [%2];" : "=l"(w[0]), "=l"(w[1]) : "l"(row) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (i < left) asm volatile("ld.relaxed.gpu.global.b64 %0, [%1];" : "=l"(w[i]) : "l"(row + 2 * i) : "memory");
  }
  const float2 a = split(w[0]), b = split(w[1]);
  return {a.x, a.y, b.x, b.y};
}
template <bool kPair>
__device__ __forceinline__ void publish(float* row, const GlrShape& s, const GlrTileAt& at, const Words& v) {
  const int left = s.channels - at.c0 - 2 * int(threadIdx.x & 31);
  const Two w[2] = {two(v.A0, v.B0), two(v.A1, v.B1)};
  if constexpr (kPair) {
    if (left > 0) asm volatile("st.relaxed.gpu.global.v2.b64 [%0], {%1, %2};" ::"l"(row), "l"(w[0]), "l"(w[1]) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (i < left) asm volatile("st.relaxed.gpu.global.b64 [%0], %1;" ::"l"(row + 2 * i), "l"(w[i]) : "memory");
  }
}

// The exchange area: per warp kDirections pairs (A0, B0, A1, B1) of 32 lanes, then the words the warp looked at.  It lies
// in the shared tiles of the gates where it fits: they are in registers by then.
template <int kDirections>
struct Exchange {
  uint8_t* base;
  int slice;
  __device__ __forceinline__ float4& pair(int direction, int warp) const {
    return reinterpret_cast<float4*>(base + warp * slice)[direction * 32 + (threadIdx.x & 31)];
  }
  __device__ __forceinline__ float4& look(int warp, int k) const {
    return reinterpret_cast<float4*>(base + warp * slice)[(kDirections + k) * 32 + (threadIdx.x & 31)];
  }
};

// The state that enters the tile (from the left; reversed: the adjoint from the right), in every warp.  Called by the
// whole block after one warp has published the tile's own pair.
template <bool kPair, bool kReverse, int kDirections>
__device__ __forceinline__ Two carry_in(float* words, const GlrShape& s, const GlrTileAt& at, GlrShared& sh,
                                        const Exchange<kDirections>& ex) {
  const int before = kReverse ? s.tiles - 1 - at.tile : at.tile;  // tiles that come before this one
  if (before == 0) return two(0.f);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kFar = 0x7fffffff;
  uint64_t began = 0;
  int from;
  for (;;) {
    int unset = kFar, state = kFar;
    for (int k = 0; k < s.window; ++k) {
      const int back = warp * s.window + k;
      Words v{kGlrReset, 0.f, kGlrReset, 0.f};  // before the first tile: a state of zero
      if (back < before)
        v = load_words<kPair>(words_at(words, s, at, kReverse ? at.tile + 1 + back : at.tile - 1 - back), s, at);
      ex.look(warp, k) = make_float4(v.A0, v.B0, v.A1, v.B1);
      if (!__all_sync(0xffffffffu, v.set())) unset = min(unset, back);
      else if (__all_sync(0xffffffffu, v.state())) state = min(state, back);
    }
    if (lane == 0) sh.marks[warp] = make_int2(unset, state);
    if (threadIdx.x == 0) {
      const uint64_t now = global_timer_ns();
      if (began == 0) began = now;
      if (now - began > kWaitLimitNs) sh.late = 1;
    }
    __syncthreads();
    const int2 mark = sh.marks[lane & (kGlrWarps - 1)];
    unset = __reduce_min_sync(0xffffffffu, mark.x), from = __reduce_min_sync(0xffffffffu, mark.y);
    const bool late = sh.late != 0;
    if (from < unset) break;
    if (late) return two(__int_as_float(0x7fffffff));
    __syncthreads();  // before the words are looked at again
  }
  float h[2] = {0.f, 0.f};
  for (int w = from / s.window, k = from % s.window; w >= 0; --w, k = s.window - 1)
    for (; k >= 0; --k) {
      const float4 v = ex.look(w, k);
      h[0] = fold(v.x, v.y, h[0]), h[1] = fold(v.z, v.w, h[1]);
    }
  return two(h[0], h[1]);
}
__device__ __forceinline__ Two folded(const float4& v, Two h) {
  const float2 f = split(h);
  return two(fold(v.x, v.y, f.x), fold(v.z, v.w, f.y));
}
__device__ __forceinline__ void chain(Words& v, const float4& w) {
  chain(v.A0, v.B0, w.x, w.y);
  chain(v.A1, v.B1, w.z, w.w);
}

// The decays of the warp's tokens from their gates.
template <typename G>
__device__ __forceinline__ void to_decays(G* gates, Two (&a)[kGlrTokens]) {
  bool plain = true;
#pragma unroll
  for (int j = 0; j < kGlrTokens; ++j) {
    const Two g = widened(token(gates, j));
    const float2 v = split(g);
    plain &= fabsf(v.x) <= kDecayRange && fabsf(v.y) <= kDecayRange;  // false for NaN
    a[j] = decays_in_range(g);
  }
  if (!__all_sync(0xffffffffu, plain)) {
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) a[j] = decays(widened(token(gates, j)));
  }
}

// (A, B) of the warp's tokens; starts: its tokens that begin a sequence.
template <typename X, bool kPair>
__device__ __forceinline__ Words fold_tokens(X* xs, const Two (&a)[kGlrTokens], uint32_t starts, const float* __restrict__ h0,
                                             const GlrShape& s, const GlrTileAt& at, int t0) {
  Two A = two(1.f), B = two(0.f);
  if (starts == 0) {
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) A = mul2(A, a[j]), B = fma2(a[j], B, widened(token(xs, j)));
  } else {
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) {
      if ((starts >> j) & 1) B = load_state<kPair>(h0, s, at, sequence_of(s.seq, at.b, t0 + j));
      B = fma2(a[j], B, widened(token(xs, j)));
    }
    A = two(kGlrReset);
  }
  const float2 p = split(A), q = split(B);
  return {p.x, q.x, p.y, q.y};
}

// After a wait that ran out: copies that are still in flight may write to this block's shared memory.
__device__ __forceinline__ void let_copies_land() {
  const uint64_t t0 = global_timer_ns();
  while (global_timer_ns() - t0 < 100000) __nanosleep(1000);
}

// ---- host ------------------------------------------------------------------------------------------------------------
inline int check_glr(const char* what, int x_type, int g_type, int64_t batch, int64_t tokens, int64_t channels, int64_t seqs,
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

inline int size_of(int type) { return type == kTypeFp32 ? 4 : 2; }

inline GlrShape glr_shape(int64_t batch, int64_t tokens, int64_t channels, int64_t seqs, const int32_t* cu) {
  return {{cu, int(cu ? seqs : batch), int(tokens)}, int(batch), int(tokens), int(channels),
          int((tokens + kGlrTile - 1) / kGlrTile), int((channels + kGlrChannels - 1) / kGlrChannels), 1, 0, 0, nullptr};
}

// Shared memory of a launch: the tiles of `tensors` bytes a token and channel (the gates' last), then the exchange area
// unless it fits into the gates' tiles.  The window: words a warp looks back over, eight warps together.  With few
// chains (channel blocks x batch rows) the tiles in flight lie one behind the other, so the nearest state may be as
// many tiles back as there are blocks on the GPU per chain; with many chains it is near, and a wide window would only
// read more.
template <int kDirections>
size_t glr_layout(GlrShape& s, int tensors, int gate_size, int blocks_per_sm) {
  const int64_t chains = int64_t(s.batch) * s.channel_blocks, depth = (blocks_per_sm * 148 + chains - 1) / chains;
  s.window = int(depth >= 6 * kGlrWarps ? 6 : depth <= kGlrWarps ? 1 : (depth + kGlrWarps - 1) / kGlrWarps);
  const int need = 32 * int(sizeof(float4)) * (kDirections + s.window);
  const int tiles = kGlrTile * kGlrChannels * tensors, gates = kGlrTokens * kGlrChannels * gate_size;
  const bool inside = need <= gates;
  s.slice = inside ? gates : need;
  s.exchange = inside ? tiles - kGlrTile * kGlrChannels * gate_size : tiles;
  return inside ? tiles : tiles + need * kGlrWarps;
}

// Words unset and the counter behind them at -1: one asynchronous fill with ones (nothing where a chain is one tile).
inline int glr_clear(const char* what, GlrShape& s, float* words, cudaStream_t stream) {
  if (s.tiles <= 1) return MEK_OK;
  const int64_t count = int64_t(s.batch) * s.tiles * s.channels * 2;
  s.counter = reinterpret_cast<int*>(words + count);
  const cudaError_t err = cudaMemsetAsync(words, 0xff, size_t(count + 1) * sizeof(float), stream);
  return err == cudaSuccess ? MEK_OK : fail(MEK_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
}

// Sequences without tokens pass their state through: out[seq] = in[seq] (or zero).
static __global__ void __launch_bounds__(256) glr_empty_kernel(const int32_t* __restrict__ cu, int tokens, int channels,
                                                               const float* __restrict__ in, float* __restrict__ out) {
  const int seq = blockIdx.x;
  if (cu[seq] < min(cu[seq + 1], tokens)) return;
  for (int c = threadIdx.x; c < channels; c += 256)
    out[int64_t(seq) * channels + c] = in ? in[int64_t(seq) * channels + c] : 0.f;
}
inline int glr_empty(const GlrShape& s, const float* in, float* out, cudaStream_t stream) {
  if (s.seq.cu == nullptr || out == nullptr) return MEK_OK;
  glr_empty_kernel<<<unsigned(s.seq.count), 256, 0, stream>>>(s.seq.cu, s.tokens, s.channels, in, out);
  return launched("linear_recurrence (sequences without tokens)");
}

// Whether TMA can address a tensor: 16-byte aligned base and strides (of extents that have more than one element).
inline bool glr_mappable(const GlrTensor& t, int type, const GlrShape& s) {
  const int size = size_of(type);
  auto fits = [&](int64_t stride) { return stride > 0 && stride * size % 16 == 0 && stride * size < (1ll << 40); };
  return reinterpret_cast<uintptr_t>(t.base) % 16 == 0 && (s.tokens == 1 || fits(t.token_stride)) &&
         (s.batch == 1 || fits(t.batch_stride));
}
inline int glr_map(CUtensorMap* map, const GlrTensor& t, int type, const GlrShape& s, const char* what) {
  EncodeTiledFn encode = encode_tiled_fn();
  if (encode == nullptr) return fail(MEK_ERR_CUDA, "%s: the driver does not export cuTensorMapEncodeTiled", what);
  const int size = size_of(type);
  const cuuint64_t dims[3] = {cuuint64_t(s.channels), cuuint64_t(s.tokens), cuuint64_t(s.batch)};
  const cuuint64_t strides[2] = {cuuint64_t(s.tokens == 1 ? 16 : t.token_stride * size),
                                 cuuint64_t(s.batch == 1 ? 16 : t.batch_stride * size)};
  const cuuint32_t box[3] = {kGlrChannels, kGlrTokens, 1}, step[3] = {1, 1, 1};
  const CUtensorMapDataType kinds[3] = {CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                                        CU_TENSOR_MAP_DATA_TYPE_FLOAT32};
  const CUresult rc = encode(map, kinds[type], 3, t.base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                             CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? MEK_OK : fail(MEK_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed (%d)", what, int(rc));
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

}  // namespace mek

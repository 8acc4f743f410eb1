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
// publishes its own state and only then goes over its tokens (still on chip) a second time: a single-pass scan with
// decoupled look-back (D. Merrill, M. Garland, 2016).
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
// Every wait is bounded all the same (one second); what it leaves unknown -- the warp's tokens, the carried state, all that
// follows from them inside their sequence -- is then NaN.
//
// Measured at 4 x 4,096 tokens x 4,096 channels, bf16 with FP32 gates: forward 97 us = 5.5 TB/s, backward 184 - 194 us =
// 4.8 - 5.1 TB/s (copy: 6.5).  What bounds it: an SM holds four tiles (three in the backward), with its shared memory and
// its registers both full, for about 12,400 cycles each -- the number from the counter 1,750, the boxes from L2 1,700, the
// walk 2,400, the warps' pairs 1,100, the look-back 2,600, prefixes 600, the second pass 1,400, the store 850 (stamps of
// the forward before the votes on growth) -- at 61 % of the issue slots.  Tried and slower: blocks that stay and draw their next number early (235 -> 277 us at twice the
// tokens: a tile waits behind its block's present one, and its chain behind it); four or sixteen warps a block (forward
// 250 / 278, and 492 / 328 for one long chain on 512 channels instead of 334); decays in registers (267, spills);
// scalar arithmetic (276).
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

__device__ __forceinline__ float clamped(float g) {  // NaN stays
  float v;
  asm("max.NaN.f32 %0, %1, 0fC2AE0000;" : "=f"(v) : "f"(g));   // -87
  asm("min.NaN.f32 %0, %1, 0f42B1999A;" : "=f"(v) : "f"(v));   // 88.8
  return v;
}

// exp(g) = 2^n (1 + r + r^2 q(r)), r = g - n log 2: 1 + p is rounded once, so a decay next to one carries no bias.  (CUDA's
// expf is off by up to an ulp to one side there, and a thousand tokens' memory adds that up: relative error of a state
// 7e-6 with expf, 4e-7 with this.)  q of degree 4 is the minimax fit of (e^r - 1 - r) / r^2 over |r| <= log(2) / 2 in
// the error of the whole, found by reweighted least squares: off by at most 5.3e-9, by 2e-10 for |r| < 0.05.  The
// rounding of log 2 puts |n| 2e-9 into the relative error: at n = 1 the memory is a token long already.
// n sits in the low bits of the shifted product, from where one multiply-add makes 2^(n - 1), for n from -126, whose bits are
// zero (a gate at or below -87, minus infinity too, closes exactly), to 128; the factor is 2 (1 + p), the same rounding.
// (With 2^n and 1 + p the last binade of FP32, gates from 88.38 to 88.72, would be infinite.  In its place the first one
// goes: a decay below 2^-125.5 = e^-86.98 = 1.67e-38 is zero.)
__device__ __forceinline__ Two decays(Two gates) {
  const float2 v = split(gates);
  const Two g = two(clamped(v.x), clamped(v.y)), shift = two(12582912.f);
  const Two shifted = fma2(g, two(1.44269504f), shift);
  const Two n = sub2(shifted, shift), r = fma2(n, two(-0.693147181f), g);
  Two q = fma2(r, two(0.00139505253f), two(0.00836891122f));
  q = fma2(q, r, two(0.0416662060f));
  q = fma2(q, r, two(0.166665182f));
  q = fma2(q, r, two(0.5f));
  const Two e = fma2(fma2(mul2(r, r), q, r), two(2.f), two(2.f));
  const float2 m = split(shifted);
  return mul2(e, two(__int_as_float(__float_as_int(m.x) * (1 << 23) + 0x3f000000),
                     __int_as_float(__float_as_int(m.y) * (1 << 23) + 0x3f000000)));
}

// Gates may be positive, and a product of decays may then leave FP32's range where the states do not (kGrown): a state of
// zero stays zero under any growth, and a run that holds a decay of zero is closed whatever grew before or after it.  (Growth
// past the range from a state that is not zero is infinite.)  Folds wait for one another, so the two comparisons are only
// made where an A is infinite, which a vote tells beforehand (in every fold: forward 231 -> 242 us, backward 416 -> 460).
constexpr float kGlrInfinity = __builtin_huge_valf();
template <bool kGrown>
__device__ __forceinline__ float fold(float A, float B, float h) {
  return A < 0.f ? B : fmaf(kGrown && A == kGlrInfinity && h == 0.f ? 0.f : A, h, B);
}
__device__ __forceinline__ float product(float A, float A2) {
  const float p = A * A2;
  return p != p && A == A && A2 == A2 ? 0.f : p;  // zero times infinity
}
// (A, B), then (A2, B2)
template <bool kGrown>
__device__ __forceinline__ void chain(float& A, float& B, float A2, float B2) {
  B = fold<kGrown>(A2, B2, B);
  A = A < 0.f || A2 < 0.f ? kGlrReset : kGrown ? product(A, A2) : A * A2;
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

// One tensor [batch, tokens, channels] of a call: its map (kTma) or its base and strides (elements).
struct GlrTensor {
  void* base;
  int64_t batch_stride, token_stride;
};

struct GlrShape {  // a __grid_constant__ of the kernels: the functions that are not inlined take its address, not a copy's
  Sequences seq;
  int batch, tokens, channels, tiles, channel_blocks;
  int window;        // words a warp looks back over at once; 0: one warp looks at the nearest four
  int ahead;         // how many tiles later lies the one a block asks into L2
  int* counter;      // the last tile taken (-1 before the launch); NULL where there is one tile a chain
  RowWaits waits;
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

// What the warps of a block exchange.
template <int kDirections>
struct GlrShared {
  float4 pair[kDirections][kGlrWarps][32];  // the warps' (A0, B0, A1, B1)
  Two carried[32];                          // the state that enters the tile
  uint64_t arrived[kGlrWarps];              // a warp's boxes
  int2 marks[kGlrWarps];                    // nearest word not set, nearest state, among the words a warp looked at
  GlrTileAt at, ahead;                      // the block's tile, and one to ask into L2 (tile < 0: none)
  int late;
  int grown;                                // a warp's A is infinite or NaN
};

// The block's tile -- the next in order, or its own index where tiles do not wait for one another -- and the barriers.
// tile < 0: a number behind the last tile, which only a counter that something else writes to can give; the block has
// nothing to do.
template <bool kReverse, int kDirections>
__device__ __forceinline__ GlrTileAt take_tile(const GlrShape& s, GlrShared<kDirections>& sh) {
  if (threadIdx.x < 32) {
    if (threadIdx.x < kGlrWarps) mbar_init(&sh.arrived[threadIdx.x], 1);
    fence_mbar_init();
    if (threadIdx.x == 0) {
      const int index = s.counter ? atomicAdd(s.counter, 1) + 1 : int(blockIdx.x);
      sh.at = tile_at<kReverse>(s, index);
      if (unsigned(index) >= gridDim.x) sh.at.tile = -1;
      sh.ahead = tile_at<kReverse>(s, min(index, int(gridDim.x) - 1 - s.ahead) + s.ahead);
      if (index >= int(gridDim.x) - s.ahead) sh.ahead.tile = -1;
      sh.late = sh.grown = 0;
    }
  }
  __syncthreads();
  return sh.at;
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
__device__ __forceinline__ void box_prefetch(const CUtensorMap* map, int c, int t, int b) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(c), "r"(t), "r"(b)
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
__device__ __forceinline__ Two lost() { return two(__int_as_float(0x7fffffff)); }  // a state that did not come in time: NaN
struct Words {  // of a lane's two channels
  float A0, B0, A1, B1;
  __device__ __forceinline__ bool set() const {
    return __float_as_uint(A0) != 0xffffffffu && __float_as_uint(A1) != 0xffffffffu;  // no operation makes this NaN
  }
  __device__ __forceinline__ bool state() const { return A0 < 0.f && A1 < 0.f; }
  __device__ __forceinline__ bool finite() const { return A0 < kGlrInfinity && A1 < kGlrInfinity; }  // of A
  template <bool kGrown>
  __device__ __forceinline__ void onto(float (&h)[2]) const {
    h[0] = fold<kGrown>(A0, B0, h[0]), h[1] = fold<kGrown>(A1, B1, h[1]);
  }
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
  if (s.waits.tiles_withheld & kWithholdWords) return;
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

// Looking back with one warp: the nearest state among the four tiles before this one.
constexpr int kGlrNear = 4;
constexpr int kGlrFreePolls = 64;
template <bool kPair, bool kReverse>
__device__ __forceinline__ Two look_back(float* words, const GlrShape& s, const GlrTileAt& at, int before) {
  uint64_t began = 0;
  const float* row = words_at(words, s, at, at.tile);
  const int64_t step = int64_t(kReverse ? 2 : -2) * s.channels;
  for (int polls = 0;; ++polls) {
    Words v[kGlrNear];
#pragma unroll
    for (int k = 0; k < kGlrNear; ++k) {
      v[k] = {kGlrReset, 0.f, kGlrReset, 0.f};  // before the first tile: a state of zero
      if (k < before) v[k] = load_words<kPair>(row + (k + 1) * step, s, at);
    }
    bool ready = true;
    float h[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kGlrNear; ++k) {
      ready = ready && __all_sync(0xffffffffu, v[k].set());
      if (!ready) break;
      if (__all_sync(0xffffffffu, v[k].state())) {
        bool finite = true;
#pragma unroll
        for (int i = 0; i < kGlrNear; ++i) finite = finite && (i > k || v[i].finite());
        const bool grown = !__all_sync(0xffffffffu, finite);
#pragma unroll
        for (int i = kGlrNear - 1; i >= 0; --i) {
          if (i > k) continue;
          if (grown) v[i].template onto<true>(h);
          else v[i].template onto<false>(h);
        }
        return two(h[0], h[1]);
      }
    }
    if (polls >= kGlrFreePolls) {  // reading the timer costs as much as a poll: the first ones go without
      const uint64_t now = global_timer_ns();
      if (began == 0) began = now;
      // one decision for the warp: a lane that left alone would be waited for in the votes above
      if (__any_sync(0xffffffffu, now - began > s.waits.limit_ns)) return lost();
    }
  }
}

// Looking back with the whole block, for chains whose tiles in flight lie far behind one another: warp w looks at the words
// behind those of warp w - 1, which it keeps in registers, until there is a state with no unset word in front of it.
// The fold from there goes forward from warp to warp; the result is in sh.carried.
constexpr int kGlrWindow = 6;  // words of a warp
template <bool kPair, bool kReverse, int kDirections>
__device__ __forceinline__ void look_back_together(float* words, const GlrShape& s, const GlrTileAt& at,
                                                   GlrShared<kDirections>& sh, int before) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float* row = words_at(words, s, at, at.tile);
  const int64_t step = int64_t(kReverse ? 2 : -2) * s.channels;
  constexpr int kFar = 0x7fffffff;
  uint64_t began = 0;
  Words v[kGlrWindow];
  int from;
  for (int polls = 0;; ++polls) {
    int unset = kFar, state = kFar;
#pragma unroll
    for (int k = 0; k < kGlrWindow; ++k) {
      const int back = warp * s.window + k;
      v[k] = {kGlrReset, 0.f, kGlrReset, 0.f};  // before the first tile: a state of zero
      if (k < s.window && back < before) v[k] = load_words<kPair>(row + (back + 1) * step, s, at);
    }
#pragma unroll
    for (int k = 0; k < kGlrWindow; ++k) {
      if (k < s.window) {
        if (!__all_sync(0xffffffffu, v[k].set())) unset = min(unset, warp * s.window + k);
        else if (__all_sync(0xffffffffu, v[k].state())) state = min(state, warp * s.window + k);
      }
    }
    if (lane == 0) sh.marks[warp] = make_int2(unset, state);
    if (threadIdx.x == 0 && polls >= kGlrFreePolls) {
      const uint64_t now = global_timer_ns();
      if (began == 0) began = now;
      if (now - began > s.waits.limit_ns) sh.late = 1;
    }
    __syncthreads();
    const int2 mark = sh.marks[lane & (kGlrWarps - 1)];
    unset = __reduce_min_sync(0xffffffffu, mark.x), from = __reduce_min_sync(0xffffffffu, mark.y);
    if (from < unset) break;
    if (sh.late != 0) {
      sh.carried[lane] = lost();  // every warp the same
      __syncthreads();
      return;
    }
    __syncthreads();  // before the marks are set again
  }
  float h[2] = {0.f, 0.f};
  const int top = from / s.window;
  bool finite = true;
#pragma unroll
  for (int k = 0; k < kGlrWindow; ++k)
    if (k < s.window && warp * s.window + k <= from) finite = finite && v[k].finite();
  const bool grown = !__all_sync(0xffffffffu, finite);
  for (int w = top; w >= 0; --w) {
    if (warp == w) {
      if (w < top) {
        const float2 f = split(sh.carried[lane]);
        h[0] = f.x, h[1] = f.y;
      }
#pragma unroll
      for (int k = kGlrWindow - 1; k >= 0; --k)
        if (k < s.window && w * s.window + k <= from) {
          if (grown) v[k].template onto<true>(h);
          else v[k].template onto<false>(h);
        }
      sh.carried[lane] = two(h[0], h[1]);
    }
    __syncthreads();
  }
}

// The state that enters the tile (from the left; reversed: the adjoint from the right), in every warp.  Called by the
// whole block after its warp `owner` has published the tile's own pair `tile`; that warp then publishes the state.
template <bool kPair, bool kReverse, int kDirections>
__device__ __forceinline__ Two carry_in(float* words, const GlrShape& s, const GlrTileAt& at, GlrShared<kDirections>& sh,
                                        int owner, const Words& tile) {
  const int before = kReverse ? s.tiles - 1 - at.tile : at.tile;  // tiles that come before this one
  const bool mine = int(threadIdx.x >> 5) == owner;
  Two h = two(0.f);
  if (before > 0 && s.window > 0) {
    look_back_together<kPair, kReverse>(words, s, at, sh, before);
    h = sh.carried[threadIdx.x & 31];
  } else if (before > 0 && mine) {
    h = look_back<kPair, kReverse>(words, s, at, before);
  }
  if (mine && !tile.state()) {  // else it was one already
    const float2 in = split(h);
    float out[2] = {in.x, in.y};
    tile.onto<true>(out);
    publish<kPair>(words_at(words, s, at, at.tile), s, at, Words{kGlrReset, out[0], kGlrReset, out[1]});
  }
  if (before == 0 || s.window > 0) return h;
  if (mine) sh.carried[threadIdx.x & 31] = h;
  __syncthreads();
  return sh.carried[threadIdx.x & 31];
}
__device__ __forceinline__ Words words_of(const float4& v) { return {v.x, v.y, v.z, v.w}; }
template <bool kGrown>
__device__ __forceinline__ Two folded(const float4& v, Two h) {
  const float2 f = split(h);
  return two(fold<kGrown>(v.x, v.y, f.x), fold<kGrown>(v.z, v.w, f.y));
}
template <bool kGrown>
__device__ __forceinline__ void chain(Words& v, const float4& w) {
  chain<kGrown>(v.A0, v.B0, w.x, w.y);
  chain<kGrown>(v.A1, v.B1, w.z, w.w);
}
// A tile's pair, from its warps' in the order of time, and the state that enters warp `warp` when h enters the tile.
template <bool kReverse, bool kGrown>
__device__ __forceinline__ Words chained(const float4 (*pair)[32]) {
  const int lane = threadIdx.x & 31;
  Words tile = words_of(pair[kReverse ? kGlrWarps - 1 : 0][lane]);
#pragma unroll
  for (int i = 1; i < kGlrWarps; ++i) chain<kGrown>(tile, pair[kReverse ? kGlrWarps - 1 - i : i][lane]);
  return tile;
}
template <bool kReverse, bool kGrown>
__device__ __forceinline__ Two entering(const float4 (*pair)[32], int warp, Two h) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < kGlrWarps - 1; ++i) {
    const int w = kReverse ? kGlrWarps - 1 - i : i;
    if (kReverse ? w > warp : w < warp) h = folded<kGrown>(pair[w][lane], h);
  }
  return h;
}
// The same where an A is infinite or NaN.
template <bool kReverse>
static __device__ __noinline__ Words chained_grown(const float4 (*pair)[32]) { return chained<kReverse, true>(pair); }
template <bool kReverse>
static __device__ __noinline__ Two entering_grown(const float4 (*pair)[32], int warp, Two h) {
  return entering<kReverse, true>(pair, warp, h);
}

// A warp's gates and, once they are exponentiated, its decays [16][64] in FP32, in one place.  16-bit gates arrive in the
// upper half (token j's at byte 2,048 + 128 j): from token 8 on, token j's decays (byte 256 j) overwrite gates of tokens
// 2 j - 16 and 2 j - 15, none later than j.  Gradients of 16-bit gates go to the upper half again, token j's over the
// decays of token 8 + j / 2, none earlier than j on the way back.  A warp's lanes are brought together before each such
// write, so that all have read what it overwrites; FP32 gates and their gradients lie in the lane's own decay.
constexpr uint32_t kGlrDecays = kGlrTokens * kGlrChannels * sizeof(float);
template <typename G>
__device__ __forceinline__ G* gates_of(float* decays) {
  return reinterpret_cast<G*>(reinterpret_cast<uint8_t*>(decays) + kGlrDecays - kGlrBox<G>);
}
__device__ __forceinline__ Two decay_at(const float* decays, int j) {
  return *reinterpret_cast<const Two*>(decays + j * kGlrChannels + 2 * (threadIdx.x & 31));
}

template <typename G>
__device__ __forceinline__ void put_decay(float* decays, int j, Two a) {
  if (sizeof(G) < sizeof(float) && j >= kGlrTokens / 2) __syncwarp();
  *reinterpret_cast<Two*>(decays + j * kGlrChannels + 2 * (threadIdx.x & 31)) = a;
}
template <typename G>
__device__ __forceinline__ void put_gradient(float* decays, int j, Two dg) {
  if (sizeof(G) < sizeof(float)) __syncwarp();
  token(gates_of<G>(decays), j) = narrowed<G>(dg);
}

// Where sequences start and end among a warp's 16 tokens.
enum : int { kInside = 0, kOneEdge = 1, kManyEdges = 2 };
struct Edges {
  uint32_t starts, ends, live;  // live: tokens of a sequence; the others' outputs are zero and reach no live token
  int kind;                     // kInside: no boundary, all live; kOneEdge: at most one start and one end
  int start, end;               // of kOneEdge: their tokens, or -1
  int start_seq, end_seq;
  // a warp behind the last token
  __device__ __forceinline__ Edges() : starts(0), ends(0), live(0), kind(kInside), start(-1), end(-1), start_seq(0), end_seq(0) {}
  __device__ __forceinline__ Edges(const Sequences& s, const Span& span, int b, int t0) {
    const int n = min(max(s.tokens - t0, 0), kGlrTokens);
    auto below = [](int k) { return k >= 32 ? 0xffffffffu : k <= 0 ? 0u : (1u << k) - 1; };
    const uint32_t here = below(n);
    live = here & below(span.hi - t0) & ~below(span.lo - t0);
    starts = span.bounds & live;
    ends = (span.bounds >> 1) & live;
    kind = (starts | ends) == 0 && live == below(kGlrTokens) ? kInside
           : __popc(starts) <= 1 && __popc(ends) <= 1        ? kOneEdge
                                                             : kManyEdges;
    start = kind == kOneEdge ? __ffs(starts) - 1 : -1, end = kind == kOneEdge ? __ffs(ends) - 1 : -1;
    start_seq = start >= 0 ? sequence_of(s, b, t0 + start) : 0;
    end_seq = end >= 0 ? sequence_of(s, b, t0 + end) : 0;
  }
};

// One walk over the warp's tokens: gates to decays, and the fold of the run to (A, B); with gradients ds (kBack) also to
// (A, D), D the adjoint that leaves the first token to the left when nothing enters at the last.  kEdge: a sequence
// may start at edges.start from the state s0 and end at edges.end with the adjoint d1.
template <typename X, typename G, bool kBack, bool kEdge>
__device__ __forceinline__ void walk_tokens(float* decay, X* xs, X* ds, const Edges& edges, Two s0, Two d1, Two& A, Two& B,
                                            Two& D) {
  G* gates = gates_of<G>(decay);
  A = two(1.f), B = D = two(0.f);
#pragma unroll
  for (int j = 0; j < kGlrTokens; ++j) {
    const Two a = decays(widened(token(gates, j)));
    put_decay<G>(decay, j, a);
    A = mul2(A, a);
    if (kEdge && j == edges.start) B = s0;
    B = fma2(a, B, widened(token(xs, j)));
    if constexpr (kBack) {
      if (!kEdge || edges.end < 0 || j <= edges.end) D = fma2(A, widened(token(ds, j)), D);
      if (kEdge && j == edges.end) D = fma2(A, d1, D);
    }
  }
}
// The same folds where sequences start or end more than once among the tokens.
template <typename X, bool kPair>
__device__ __noinline__ Two fold_from_starts(const float* decay, X* xs, uint32_t starts, const float* __restrict__ h0,
                                             const GlrShape& s, const GlrTileAt& at, int t0) {
  Two B = two(0.f);
#pragma unroll 1
  for (int j = 0; j < kGlrTokens; ++j) {
    if ((starts >> j) & 1) B = load_state<kPair>(h0, s, at, sequence_of(s.seq, at.b, t0 + j));
    B = fma2(decay_at(decay, j), B, widened(token(xs, j)));
  }
  return B;
}
template <typename X, bool kPair>
__device__ __noinline__ Two fold_from_ends(const float* decay, X* ds, uint32_t ends, const float* __restrict__ d_final,
                                           const GlrShape& s, const GlrTileAt& at, int t0) {
  Two D = two(0.f);
#pragma unroll 1
  for (int j = kGlrTokens - 1; j >= 0; --j) {
    if ((ends >> j) & 1) D = load_state<kPair>(d_final, s, at, sequence_of(s.seq, at.b, t0 + j));
    D = mul2(decay_at(decay, j), add2(widened(token(ds, j)), D));
  }
  return D;
}
// Whether a lane's product of decays left FP32's range or met a NaN; the same for the whole warp.  The walk's A, and its D,
// which takes such products times gradients of zero, are then folded once more.
__device__ __forceinline__ bool overflowed(Two A) {
  const float2 a = split(A);
  return __any_sync(0xffffffffu, !(a.x < kGlrInfinity && a.y < kGlrInfinity));
}
static __device__ __noinline__ Two product_of(const float* decay) {
  float2 A = make_float2(1.f, 1.f);
#pragma unroll 1
  for (int j = 0; j < kGlrTokens; ++j) {
    const float2 a = split(decay_at(decay, j));
    A = make_float2(product(A.x, a.x), product(A.y, a.y));
  }
  return two(A.x, A.y);
}
__device__ __forceinline__ float4 packed(Two A, Two B) {
  const float2 a = split(A), b = split(B);
  return make_float4(a.x, b.x, a.y, b.y);
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
          int((tokens + kGlrTile - 1) / kGlrTile), int((channels + kGlrChannels - 1) / kGlrChannels), 0, 0, nullptr, row_waits()};
}

// The window: words a warp looks back over, eight warps together.  With few chains (channel blocks x batch rows) the tiles
// in flight lie one behind the other, so the nearest state may be as many tiles back as there are blocks on the GPU per
// chain; where it is at most four tiles back, one warp looks (window 0) and the others wait, which saves their
// instructions.
// Ahead: as many tiles as half the blocks on the GPU, so that a tile's boxes are in L2 when its block asks for them.  (A
// block holds its shared memory for the latency of its loads; from L2 that is 1,200 cycles instead of 2,800.)
inline void glr_window(GlrShape& s, int blocks_per_sm) {
  s.ahead = blocks_per_sm * 148 / 2;
  const int64_t chains = int64_t(s.batch) * s.channel_blocks, depth = (blocks_per_sm * 148 + chains - 1) / chains;
  s.window = int(depth >= kGlrWindow * kGlrWarps ? kGlrWindow : depth <= kGlrNear ? 0 : (depth + kGlrWarps - 1) / kGlrWarps);
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

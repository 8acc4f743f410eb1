// The gated linear recurrence, forward (see linear_recurrence.cuh).
#include "linear_recurrence.cuh"

namespace mek {

struct GlrFwdArgs {
  GlrTensor x, g, y;
  const float* h0;
  float *words, *final_state;
};

template <typename X, typename G, bool kTma>
__global__ void __launch_bounds__(kGlrWarps * 32, 4) glr_fwd_kernel(const __grid_constant__ CUtensorMap x_map,
                                                                    const __grid_constant__ CUtensorMap g_map,
                                                                    const __grid_constant__ CUtensorMap y_map,
                                                                    const GlrFwdArgs p, const __grid_constant__ GlrShape s) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ GlrShared<1> sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const GlrTileAt at = take_tile<false>(s, sh);
  if (at.tile < 0) return;
  const int t0 = at.tile * kGlrTile + warp * kGlrTokens;
  float* decay = reinterpret_cast<float*>(smem + warp * kGlrDecays);
  X* xs = reinterpret_cast<X*>(smem + kGlrWarps * kGlrDecays + warp * kGlrBox<X>);
  bool arrived = true;
  const bool any = t0 < s.tokens;  // a warp behind the last token only takes part in the block's barriers
  if constexpr (kTma) {
    if (lane == 0 && any && !((s.waits.tiles_withheld >> warp) & 1)) {
      mbar_arrive_expect(&sh.arrived[warp], kGlrBox<X> + kGlrBox<G>);
      box_load(gates_of<G>(decay), &g_map, at.c0, t0, at.b, &sh.arrived[warp]);
      box_load(xs, &x_map, at.c0, t0, at.b, &sh.arrived[warp]);
      const GlrTileAt next = sh.ahead;
      if (next.tile >= 0) {
        box_prefetch(&g_map, next.c0, next.tile * kGlrTile + warp * kGlrTokens, next.b);
        box_prefetch(&x_map, next.c0, next.tile * kGlrTile + warp * kGlrTokens, next.b);
      }
    }
  } else if (any) {
    plain_load(gates_of<G>(decay), p.g, s, at, t0);
    plain_load(xs, p.x, s, at, t0);
    __syncwarp();
  }
  const Edges edges = any ? Edges(s.seq, span_of(s.seq, t0), at.b, t0) : Edges();
  Two s0 = edges.start >= 0 ? load_state<kTma>(p.h0, s, at, edges.start_seq) : two(0.f);
  if (kTma && any) arrived = __all_sync(0xffffffffu, mbar_wait_soon(&sh.arrived[warp], 0, s.waits.limit_ns));
  if (!arrived) s0 = lost();  // whatever lies in the tile, from here on every token and state of the warp is NaN
  const Two none = two(0.f);
  Two A = two(1.f), B = none, no_adjoint;
  if (any) {
    if (edges.kind == kInside) walk_tokens<X, G, false, false>(decay, xs, xs, edges, none, none, A, B, no_adjoint);
    else walk_tokens<X, G, false, true>(decay, xs, xs, edges, s0, none, A, B, no_adjoint);
  }
  const bool grown = overflowed(A);
  if (edges.kind == kManyEdges || grown) {
    if (grown) A = product_of(decay), sh.grown = 1;
    if (edges.kind == kManyEdges) B = fold_from_starts<X, kTma>(decay, xs, edges.starts, p.h0, s, at, t0);
  }
  if (edges.starts) A = two(kGlrReset);
  if (!arrived) A = two(kGlrReset), B = lost();
  sh.pair[0][warp][lane] = packed(A, B);
  __syncthreads();
  Two h = two(0.f);
  if (s.tiles > 1) {
    Words tile;
    if (warp == 0) {
      tile = chained<false, false>(sh.pair[0]);
      if (!__all_sync(0xffffffffu, tile.finite() && sh.grown == 0)) tile = chained_grown<false>(sh.pair[0]);
      publish<kTma>(words_at(p.words, s, at, at.tile), s, at, tile);
    }
    h = carry_in<kTma, false>(p.words, s, at, sh, 0, tile);
  }
  h = sh.grown == 0 ? entering<false, false>(sh.pair[0], warp, h) : entering_grown<false>(sh.pair[0], warp, h);
  if (!arrived) h = lost();
  if (!any) return;
  if (edges.kind == kInside) {
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) {
      h = fma2(decay_at(decay, j), h, widened(token(xs, j)));
      token(xs, j) = narrowed<X>(h);
    }
  } else if (edges.kind == kOneEdge) {
    Two last = two(0.f);
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) {
      if (j == edges.start) h = s0;
      h = fma2(decay_at(decay, j), h, widened(token(xs, j)));
      if (j == edges.end) last = h;
      token(xs, j) = narrowed<X>((edges.live >> j) & 1 ? h : two(0.f));
    }
    if (p.final_state != nullptr && edges.end >= 0) store_state<kTma>(p.final_state, s, at, edges.end_seq, last);
  } else {
#pragma unroll 1
    for (int j = 0; j < kGlrTokens; ++j) {
      const int t = t0 + j;
      if ((edges.starts >> j) & 1) h = arrived ? load_state<kTma>(p.h0, s, at, sequence_of(s.seq, at.b, t)) : lost();
      h = fma2(decay_at(decay, j), h, widened(token(xs, j)));
      const bool live = (edges.live >> j) & 1;
      token(xs, j) = narrowed<X>(live ? h : two(0.f));
      if (p.final_state != nullptr && live && ((edges.ends >> j) & 1))
        store_state<kTma>(p.final_state, s, at, sequence_of(s.seq, at.b, t), h);
    }
  }
  if constexpr (kTma) {
    fence_async_smem();
    __syncwarp();
    if (lane == 0) {
      box_store(&y_map, at.c0, t0, at.b, xs);
      tma_store_commit();
      tma_store_wait_read();
    }
    if (!arrived) let_copies_land();
  } else {
    __syncwarp();
    plain_store(xs, p.y, s, at, t0);
  }
}

template <typename X, typename G>
int glr_fwd(const GlrFwdArgs& p, GlrShape s, int x_type, int g_type, bool tma, cudaStream_t stream) {
  const char* what = "linear_recurrence_fwd";
  constexpr size_t smem = kGlrWarps * (kGlrDecays + kGlrBox<X>);
  glr_window(s, 4);
  const unsigned grid = unsigned(s.tiles) * s.channel_blocks * s.batch;
  CUtensorMap x_map{}, g_map{}, y_map{};
  if (tma &&
      glr_map(&x_map, p.x, x_type, s, what) == MEK_OK &&
      glr_map(&g_map, p.g, g_type, s, what) == MEK_OK &&
      glr_map(&y_map, p.y, x_type, s, what) == MEK_OK) {
    if (int rc = want_smem(glr_fwd_kernel<X, G, true>, smem, what)) return rc;
    glr_fwd_kernel<X, G, true><<<grid, kGlrWarps * 32, smem, stream>>>(x_map, g_map, y_map, p, s);
    return launched(what);
  }
  if (int rc = want_smem(glr_fwd_kernel<X, G, false>, smem, what)) return rc;
  glr_fwd_kernel<X, G, false><<<grid, kGlrWarps * 32, smem, stream>>>(x_map, g_map, y_map, p, s);
  return launched(what);
}

}  // namespace mek

extern "C" {

int mek_linear_recurrence_tile(void) { return mek::kGlrTile; }

int mek_linear_recurrence_fwd(const void* x, int x_type, const void* g, int g_type, void* y, int64_t batch,
                              int64_t tokens, int64_t channels, int64_t x_batch_stride, int64_t x_token_stride,
                              int64_t g_batch_stride, int64_t g_token_stride, const int32_t* cu_seqlens, int64_t num_seqs,
                              const float* initial_state, float* final_state, float* states, void* stream) {
  using namespace mek;
  const char* what = "linear_recurrence_fwd";
  if (!x || !g || !y) return fail(MEK_ERR_INVALID, "%s: a null pointer", what);
  if (int rc = check_glr(what, x_type, g_type, batch, tokens, channels, num_seqs, cu_seqlens)) return rc;
  if (tokens > kGlrTile && !states) return fail(MEK_ERR_INVALID, "%s: no room for the tiles' states", what);
  if (reinterpret_cast<uintptr_t>(states) % 16 != 0) return fail(MEK_ERR_INVALID, "%s: states must be 16-byte aligned", what);
  GlrShape s = glr_shape(batch, tokens, channels, num_seqs, cu_seqlens);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const GlrFwdArgs p{{const_cast<void*>(x), x_batch_stride, x_token_stride},
                     {const_cast<void*>(g), g_batch_stride, g_token_stride},
                     {y, tokens * channels, channels},
                     initial_state, states, final_state};
  const bool tma = glr_mappable(p.x, x_type, s) && glr_mappable(p.g, g_type, s) && glr_mappable(p.y, x_type, s) &&
                   channels % 2 == 0 && (reinterpret_cast<uintptr_t>(initial_state) | reinterpret_cast<uintptr_t>(final_state)) % 8 == 0;
  if (int rc = glr_clear(what, s, states, st)) return rc;
  if (int rc = glr_empty(s, initial_state, final_state, st)) return rc;
#define MEK_GLR_FWD(X, G) glr_fwd<X, G>(p, s, x_type, g_type, tma, st)
  MEK_GLR_TYPES(MEK_GLR_FWD);
}

}  // extern "C"

// The gated linear recurrence, backward (see linear_recurrence.cuh): tiles from the last to the first.  The states inside a
// tile are recomputed from the state that entered it, which the forward's words hold; the adjoint travels through
// words of its own.
#include "linear_recurrence.cuh"

namespace mek {

struct GlrBwdArgs {
  GlrTensor dy, x, g, dx, dg;
  const float *h0, *d_final, *states;
  float *words, *dh0;
};

template <typename X, typename G, bool kTma>
__global__ void __launch_bounds__(kGlrWarps * 32, 3) glr_bwd_kernel(const __grid_constant__ CUtensorMap dy_map,
                                                                    const __grid_constant__ CUtensorMap x_map,
                                                                    const __grid_constant__ CUtensorMap g_map,
                                                                    const __grid_constant__ CUtensorMap dx_map,
                                                                    const __grid_constant__ CUtensorMap dg_map,
                                                                    const GlrBwdArgs p, const __grid_constant__ GlrShape s) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ GlrShared<2> sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const GlrTileAt at = take_tile<true>(s, sh);
  if (at.tile < 0) return;
  const int t0 = at.tile * kGlrTile + warp * kGlrTokens;
  float* decay = reinterpret_cast<float*>(smem + warp * kGlrDecays);
  X* xs = reinterpret_cast<X*>(smem + kGlrWarps * kGlrDecays + warp * kGlrBox<X>);
  X* ds = reinterpret_cast<X*>(smem + kGlrWarps * (kGlrDecays + kGlrBox<X>) + warp * kGlrBox<X>);
  G* gs = gates_of<G>(decay);
  bool arrived = true;
  const bool any = t0 < s.tokens;  // a warp behind the last token only takes part in the block's barriers
  if constexpr (kTma) {
    if (lane == 0 && any && !((s.waits.tiles_withheld >> warp) & 1)) {
      mbar_arrive_expect(&sh.arrived[warp], 2 * kGlrBox<X> + kGlrBox<G>);
      box_load(gs, &g_map, at.c0, t0, at.b, &sh.arrived[warp]);
      box_load(ds, &dy_map, at.c0, t0, at.b, &sh.arrived[warp]);
      box_load(xs, &x_map, at.c0, t0, at.b, &sh.arrived[warp]);
      const GlrTileAt next = sh.ahead;
      if (next.tile >= 0) {
        const int t = next.tile * kGlrTile + warp * kGlrTokens;
        box_prefetch(&g_map, next.c0, t, next.b);
        box_prefetch(&dy_map, next.c0, t, next.b);
        box_prefetch(&x_map, next.c0, t, next.b);
      }
    }
  } else if (any) {
    plain_load(gs, p.g, s, at, t0);
    plain_load(ds, p.dy, s, at, t0);
    plain_load(xs, p.x, s, at, t0);
    __syncwarp();
  }
  Two h = two(0.f), c = two(0.f);
  if (at.tile > 0) {
    const Words v = load_words<kTma>(words_at(const_cast<float*>(p.states), s, at, at.tile - 1), s, at);
    h = two(v.B0, v.B1);
  }
  const Edges edges = any ? Edges(s.seq, span_of(s.seq, t0), at.b, t0) : Edges();
  Two s0 = edges.start >= 0 ? load_state<kTma>(p.h0, s, at, edges.start_seq) : two(0.f);
  Two d1 = edges.end >= 0 ? load_state<kTma>(p.d_final, s, at, edges.end_seq) : two(0.f);
  if (kTma && any) arrived = __all_sync(0xffffffffu, mbar_wait_soon(&sh.arrived[warp], 0, s.waits.limit_ns));
  if (!arrived) s0 = d1 = lost();  // whatever lies in the tile, every gradient of the warp and what it hands on is NaN
  {
    Two A = two(1.f), B = two(0.f), D = two(0.f);
    if (any) {
      if (edges.kind == kInside) walk_tokens<X, G, true, false>(decay, xs, ds, edges, s0, d1, A, B, D);
      else walk_tokens<X, G, true, true>(decay, xs, ds, edges, s0, d1, A, B, D);
    }
    const bool grown = overflowed(A);
    if (edges.kind == kManyEdges || grown) {
      if (grown) A = product_of(decay), sh.grown = 1;
      if (edges.kind == kManyEdges && edges.starts) B = fold_from_starts<X, kTma>(decay, xs, edges.starts, p.h0, s, at, t0);
      if (edges.ends || grown) D = fold_from_ends<X, kTma>(decay, ds, edges.ends, p.d_final, s, at, t0);
    }
    Two R = A;
    if (edges.starts) A = two(kGlrReset);
    if (edges.ends) R = two(kGlrReset);
    if (!arrived) A = R = two(kGlrReset), B = D = lost();
    sh.pair[0][warp][lane] = packed(A, B);
    sh.pair[1][warp][lane] = packed(R, D);
  }
  __syncthreads();
  if (s.tiles > 1) {
    Words tile;
    if (warp == kGlrWarps - 1) {
      tile = chained<true, false>(sh.pair[1]);
      if (!__all_sync(0xffffffffu, tile.finite() && sh.grown == 0)) tile = chained_grown<true>(sh.pair[1]);
      publish<kTma>(words_at(p.words, s, at, at.tile), s, at, tile);
    }
    c = carry_in<kTma, true>(p.words, s, at, sh, kGlrWarps - 1, tile);
  }
  if (sh.grown == 0) {
    h = entering<false, false>(sh.pair[0], warp, h);
    c = entering<true, false>(sh.pair[1], warp, c);
  } else {
    h = entering_grown<false>(sh.pair[0], warp, h);
    c = entering_grown<true>(sh.pair[1], warp, c);
  }
  if (!arrived) h = c = lost();
  if (!any) return;
  // forward once more for the state before every token, then back with the adjoint; dx takes dy's place, dg the gates'
  Two before[kGlrTokens];
  if (edges.kind == kInside) {
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) before[j] = h, h = fma2(decay_at(decay, j), h, widened(token(xs, j)));
#pragma unroll
    for (int j = kGlrTokens - 1; j >= 0; --j) {
      const Two dh = add2(widened(token(ds, j)), c);
      c = mul2(decay_at(decay, j), dh);
      token(ds, j) = narrowed<X>(dh);
      put_gradient<G>(decay, j, mul2(c, before[j]));
    }
  } else {
    const bool one = edges.kind == kOneEdge;
    Two first = two(0.f);
#pragma unroll
    for (int j = 0; j < kGlrTokens; ++j) {
      if (j == edges.start) h = s0;
      if (!one && ((edges.starts >> j) & 1))
        h = arrived ? load_state<kTma>(p.h0, s, at, sequence_of(s.seq, at.b, t0 + j)) : lost();
      before[j] = h, h = fma2(decay_at(decay, j), h, widened(token(xs, j)));
    }
#pragma unroll
    for (int j = kGlrTokens - 1; j >= 0; --j) {
      if (j == edges.end) c = d1;
      if (!one && ((edges.ends >> j) & 1))
        c = arrived ? load_state<kTma>(p.d_final, s, at, sequence_of(s.seq, at.b, t0 + j)) : lost();
      const Two dh = add2(widened(token(ds, j)), c);
      c = mul2(decay_at(decay, j), dh);
      const bool live = (edges.live >> j) & 1;
      token(ds, j) = narrowed<X>(live ? dh : two(0.f));
      put_gradient<G>(decay, j, live ? mul2(c, before[j]) : two(0.f));
      if (j == edges.start) first = c;
      if (!one && p.dh0 != nullptr && live && ((edges.starts >> j) & 1))
        store_state<kTma>(p.dh0, s, at, sequence_of(s.seq, at.b, t0 + j), c);
    }
    if (p.dh0 != nullptr && edges.start >= 0) store_state<kTma>(p.dh0, s, at, edges.start_seq, first);
  }
  if constexpr (kTma) {
    fence_async_smem();
    __syncwarp();
    if (lane == 0) {
      box_store(&dx_map, at.c0, t0, at.b, ds);
      box_store(&dg_map, at.c0, t0, at.b, gs);
      tma_store_commit();
      tma_store_wait_read();
    }
    if (!arrived) let_copies_land();
  } else {
    __syncwarp();
    plain_store(ds, p.dx, s, at, t0);
    plain_store(gs, p.dg, s, at, t0);
  }
}

template <typename X, typename G>
int glr_bwd(const GlrBwdArgs& p, GlrShape s, int x_type, int g_type, bool tma, cudaStream_t stream) {
  const char* what = "linear_recurrence_bwd";
  constexpr size_t smem = kGlrWarps * (kGlrDecays + 2 * kGlrBox<X>);
  glr_window(s, 3);
  const unsigned grid = unsigned(s.tiles) * s.channel_blocks * s.batch;
  CUtensorMap dy_map{}, x_map{}, g_map{}, dx_map{}, dg_map{};
  if (tma &&
      glr_map(&dy_map, p.dy, x_type, s, what) == MEK_OK &&
      glr_map(&x_map, p.x, x_type, s, what) == MEK_OK &&
      glr_map(&g_map, p.g, g_type, s, what) == MEK_OK &&
      glr_map(&dx_map, p.dx, x_type, s, what) == MEK_OK &&
      glr_map(&dg_map, p.dg, g_type, s, what) == MEK_OK) {
    if (int rc = want_smem(glr_bwd_kernel<X, G, true>, smem, what)) return rc;
    glr_bwd_kernel<X, G, true><<<grid, kGlrWarps * 32, smem, stream>>>(dy_map, x_map, g_map, dx_map, dg_map, p, s);
    return launched(what);
  }
  if (int rc = want_smem(glr_bwd_kernel<X, G, false>, smem, what)) return rc;
  glr_bwd_kernel<X, G, false><<<grid, kGlrWarps * 32, smem, stream>>>(dy_map, x_map, g_map, dx_map, dg_map, p, s);
  return launched(what);
}

}  // namespace mek

extern "C" {

int mek_linear_recurrence_bwd(const void* dy, const void* x, int x_type, const void* g, int g_type, void* dx, void* dg,
                              int64_t batch, int64_t tokens, int64_t channels, int64_t x_batch_stride,
                              int64_t x_token_stride, int64_t g_batch_stride, int64_t g_token_stride,
                              const int32_t* cu_seqlens, int64_t num_seqs, const float* initial_state,
                              const float* d_final_state, const float* states, float* dh0, float* scratch, void* stream) {
  using namespace mek;
  const char* what = "linear_recurrence_bwd";
  if (!dy || !x || !g || !dx || !dg) return fail(MEK_ERR_INVALID, "%s: a null pointer", what);
  if (int rc = check_glr(what, x_type, g_type, batch, tokens, channels, num_seqs, cu_seqlens)) return rc;
  if (tokens > kGlrTile && (!scratch || !states)) return fail(MEK_ERR_INVALID, "%s: no scratch", what);
  if ((reinterpret_cast<uintptr_t>(scratch) | reinterpret_cast<uintptr_t>(states)) % 16 != 0)
    return fail(MEK_ERR_INVALID, "%s: states and scratch must be 16-byte aligned", what);
  GlrShape s = glr_shape(batch, tokens, channels, num_seqs, cu_seqlens);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t dense = tokens * channels;
  const GlrBwdArgs p{{const_cast<void*>(dy), dense, channels},
                     {const_cast<void*>(x), x_batch_stride, x_token_stride},
                     {const_cast<void*>(g), g_batch_stride, g_token_stride},
                     {dx, dense, channels},
                     {dg, dense, channels},
                     initial_state, d_final_state, states, scratch, dh0};
  const bool tma = glr_mappable(p.dy, x_type, s) && glr_mappable(p.x, x_type, s) && glr_mappable(p.g, g_type, s) &&
                   glr_mappable(p.dx, x_type, s) && glr_mappable(p.dg, g_type, s) && channels % 2 == 0 &&
                   (reinterpret_cast<uintptr_t>(initial_state) | reinterpret_cast<uintptr_t>(d_final_state) |
                    reinterpret_cast<uintptr_t>(dh0)) % 8 == 0;
  if (int rc = glr_clear(what, s, scratch, st)) return rc;
  if (int rc = glr_empty(s, d_final_state, dh0, st)) return rc;
#define MEK_GLR_BWD(X, G) glr_bwd<X, G>(p, s, x_type, g_type, tma, st)
  MEK_GLR_TYPES(MEK_GLR_BWD);
}

}  // extern "C"

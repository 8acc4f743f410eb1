// The gated linear recurrence's single-token step on a pool of states: h = exp(g) h + x per row, state updated in place.
// HBM-bound at serving batches (the state read and written, the rows read once), launch-bound below: one launch, four
// or eight channels a thread; the loads are issued before the scan for rows that share a slot.  1,024 rows x 4,096 channels:
// 15.2 us = 4.4 TB/s, one row 14 us of host time.
#include "linear_recurrence.cuh"

namespace mek {

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
    if (__syncthreads_or(before || again)) {  // as a rule no two rows share a slot
      if (__syncthreads_or(before)) return;
      again = __syncthreads_or(again);
    }
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
  if (p.wide == 8) return p.slots64 ? glr_step_of<X, G, int64_t, 8>(p, stream) : glr_step_of<X, G, int32_t, 8>(p, stream);
  if (p.wide == 4) return p.slots64 ? glr_step_of<X, G, int64_t, 4>(p, stream) : glr_step_of<X, G, int32_t, 4>(p, stream);
  return p.slots64 ? glr_step_of<X, G, int64_t, 1>(p, stream) : glr_step_of<X, G, int32_t, 1>(p, stream);
}

}  // namespace mek

extern "C" {

int mek_linear_recurrence_step(const void* x, int x_type, const void* g, int g_type, float* state, const void* slots,
                               int slots_are_int64, void* y, int64_t rows, int64_t pool, int64_t channels,
                               int64_t x_row_stride, int64_t g_row_stride, int64_t state_row_stride, void* stream) {
  using namespace mek;
  if (!x || !g || !state || !y) return fail(MEK_ERR_INVALID, "linear_recurrence_step: a null pointer");
  if (x_type < 0 || x_type > 2 || g_type < 0 || g_type > 2)
    return fail(MEK_ERR_UNSUPPORTED, "linear_recurrence_step: an element type is 0 (bf16), 1 (fp16) or 2 (fp32)");
  if (rows <= 0 || rows > 0x7fffffff || channels <= 0 || channels > (1 << 23) || pool <= 0 || pool > 0x7fffffff)
    return fail(MEK_ERR_INVALID, "linear_recurrence_step: rows, channels and the pool's slots must be positive");
  if (!slots && rows > pool)
    return fail(MEK_ERR_INVALID, "linear_recurrence_step: %lld rows and %lld states without slots", (long long)rows, (long long)pool);
  auto wide = [&](int v) {
    auto fits = [v](const void* p, int type, int64_t stride) {
      return reinterpret_cast<uintptr_t>(p) % (v * size_of(type)) == 0 && stride % v == 0;
    };
    return fits(x, x_type, x_row_stride) && fits(g, g_type, g_row_stride) && fits(state, kTypeFp32, state_row_stride) &&
           fits(y, x_type, channels);
  };
  // Four channels a thread where accesses of four are aligned; eight from 2^20 elements on, where the GPU is full and more bytes
  // a thread count (1,024 rows x 4,096: 15.2 us against 16.4), while small calls want more blocks.
  const GlrStep p{x, g, slots, y, state, x_row_stride, g_row_stride, state_row_stride, int(rows), int(pool), int(channels),
                  rows * channels >= (1 << 20) && wide(8) ? 8 : wide(4) ? 4 : 1,
                  slots_are_int64 != 0};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define MEK_GLR_STEP(X, G) glr_step<X, G>(p, st)
  MEK_GLR_TYPES(MEK_GLR_STEP);
}

}  // extern "C"

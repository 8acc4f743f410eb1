// LayerNorm over rows of any width, forward and backward, sm_100a:
//     mean = sum(x) / C,  rstd = 1 / sqrt(sum((x - mean)^2) / C + eps),  unit = (x - mean) rstd,  y = unit w + b
//     dn = dy w,  dx = rstd (dn - mean(dn) - unit mean(dn unit)),  dw = sum_rows dy unit,  db = sum_rows dy
// FP32 inside, one rounding per output.  HBM-bound: a row's elements stay in registers between the statistics and the
// output, so each tensor crosses HBM once.  The variance is taken about the mean (never as mean(x^2) - mean^2), per
// warp first and then across the warps by Chan's rule (T. Chan, G. Golub, R. LeVeque, 1979), which costs one block
// barrier a row instead of two.
//
// The weight and bias gradients: a thread owns the same columns in every row of its block and sums them in FP32
// registers; a second launch adds the blocks' sums in FP64 in block order.  The grid is a function of the extents
// alone, so identical inputs give identical bits.
//
// 8-bit checkpoint: the forward may also write unit as e4m3 codes and the backward read them in the place of x and
// mean.  |unit| <= sqrt(C), so up to 448^2 = 200,704 columns the codes need no scale.
#include <type_traits>

#include "common.cuh"
#include "rowio.cuh"

namespace mek {

constexpr int kLnSms = 148;

template <int G>
struct RowGroup {  // G threads own a row; blocks of one warp's rows hold four
  static constexpr int kThreads = G < 128 ? 128 : G;
  static constexpr int kRows = kThreads / G;
  static constexpr int kWarps = G / 32;
};

// x [rows, width] with a row stride; y and codes dense.  grid-stride over rows.
template <typename T, int VEC, int G, int NV>
__global__ void __launch_bounds__(RowGroup<G>::kThreads) layer_norm_fwd_kernel(
    const T* __restrict__ x, int64_t x_stride, const void* __restrict__ weight, const void* __restrict__ bias,
    int param_type, T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
    uint8_t* __restrict__ codes, int64_t rows, int width, float eps) {
  constexpr int kRows = RowGroup<G>::kRows, kWarps = RowGroup<G>::kWarps;
  __shared__ float2 s_part[2][kWarps];
  const int lane = threadIdx.x % G, warp = lane / 32;
  float w[NV][VEC], b[NV][VEC];
  int counts = 0;  // elements of a row this warp owns
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * G + lane) * VEC;
    counts += min(max(width - (v * G + warp * 32) * VEC, 0), 32 * VEC);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const bool in = c + i < width;
      w[v][i] = in && weight ? load_param(weight, param_type, c + i) : 1.f;
      b[v][i] = in && bias ? load_param(bias, param_type, c + i) : 0.f;
    }
  }
  const float inv_count = counts ? 1.f / float(counts) : 0.f, inv_width = 1.f / float(width);
  int phase = 0;
  for (int64_t r0 = int64_t(blockIdx.x) * kRows; r0 < rows; r0 += int64_t(gridDim.x) * kRows) {
    const int64_t r = r0 + threadIdx.x / G;
    const bool live = r < rows;  // uniform over a group; groups share barriers only when a block is one group
    float xv[NV][VEC];
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + lane) * VEC;
      if (live && c < width) unpack(*reinterpret_cast<const Vec<T, VEC>*>(x + r * x_stride + c), xv[v]);
      else
#pragma unroll
        for (int i = 0; i < VEC; ++i) xv[v][i] = 0.f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum += xv[v][i];
    }
    // of this warp's elements; rounded before it is subtracted, whether or not it is stored: the same y either way
    float mean = __fmul_rn(warp_sum(sum), inv_count), m2 = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if ((v * G + lane) * VEC < width)
#pragma unroll
        for (int i = 0; i < VEC; ++i) m2 = fmaf(xv[v][i] - mean, xv[v][i] - mean, m2);
    m2 = warp_sum(m2);
    if constexpr (kWarps > 1) {
      if (threadIdx.x % 32 == 0) s_part[phase][warp] = make_float2(mean, m2);
      __syncthreads();
      float total = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        int n = 0;
#pragma unroll
        for (int v = 0; v < NV; ++v) n += min(max(width - (v * G + k * 32) * VEC, 0), 32 * VEC);
        total = fmaf(float(n), s_part[phase][k].x, total);
      }
      mean = __fmul_rn(total, inv_width);
      m2 = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        int n = 0;
#pragma unroll
        for (int v = 0; v < NV; ++v) n += min(max(width - (v * G + k * 32) * VEC, 0), 32 * VEC);
        const float d = s_part[phase][k].x - mean;
        m2 += fmaf(float(n) * d, d, s_part[phase][k].y);
      }
      phase ^= 1;  // the other half: a slow warp may still read this one
    }
    const float rstd = rsqrtf(m2 * inv_width + eps);
    if (!live) continue;
    if (lane == 0) {
      if (mean_out) mean_out[r] = mean;
      if (rstd_out) rstd_out[r] = rstd;
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + lane) * VEC;
      if (c >= width) continue;
      float unit[VEC], out[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        unit[i] = (xv[v][i] - mean) * rstd;
        out[i] = fmaf(unit[i], w[v][i], b[v][i]);
      }
      *reinterpret_cast<Vec<T, VEC>*>(y + r * width + c) = pack<T, VEC>(out);
      if (codes) *reinterpret_cast<Vec<uint8_t, VEC>*>(codes + r * width + c) = to_e4m3(unit);
    }
  }
}

// kCodes: unit comes from the 8-bit checkpoint, x and mean are not read.  partial [gridDim.x, 2, width] (or NULL).
template <typename T, int VEC, int G, int NV, bool kCodes>
__global__ void __launch_bounds__(RowGroup<G>::kThreads) layer_norm_bwd_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, int64_t x_stride, const uint8_t* __restrict__ codes,
    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, const void* __restrict__ weight,
    int param_type, T* __restrict__ dx, float* __restrict__ partial, int64_t rows, int width) {
  constexpr int kRows = RowGroup<G>::kRows, kWarps = RowGroup<G>::kWarps;
  __shared__ float2 s_part[2][kWarps];
  const int lane = threadIdx.x % G, warp = lane / 32;
  float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = (v * G + lane) * VEC + i;
      w[v][i] = c < width && weight ? load_param(weight, param_type, c) : 1.f;
      dw[v][i] = db[v][i] = 0.f;
    }
  const float inv_width = 1.f / float(width);
  int phase = 0;
  for (int64_t r0 = int64_t(blockIdx.x) * kRows; r0 < rows; r0 += int64_t(gridDim.x) * kRows) {
    const int64_t r = r0 + threadIdx.x / G;
    const bool live = r < rows;
    const float rstd = live ? rstd_in[r] : 0.f, mean = live && !kCodes ? mean_in[r] : 0.f;
    float unit[NV][VEC], dn[NV][VEC];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + lane) * VEC;
      if (live && c < width) {
        if constexpr (kCodes) {
          from_e4m3(*reinterpret_cast<const Vec<uint8_t, VEC>*>(codes + r * width + c), unit[v]);
        } else {
          unpack(*reinterpret_cast<const Vec<T, VEC>*>(x + r * x_stride + c), unit[v]);
#pragma unroll
          for (int i = 0; i < VEC; ++i) unit[v][i] = (unit[v][i] - mean) * rstd;
        }
        unpack(*reinterpret_cast<const Vec<T, VEC>*>(dy + r * width + c), dn[v]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          dw[v][i] = fmaf(dn[v][i], unit[v][i], dw[v][i]);
          db[v][i] += dn[v][i];
          dn[v][i] *= w[v][i];
          s1 += dn[v][i];
          s2 = fmaf(dn[v][i], unit[v][i], s2);
        }
      }
    }
    s1 = warp_sum(s1), s2 = warp_sum(s2);
    if constexpr (kWarps > 1) {
      if (threadIdx.x % 32 == 0) s_part[phase][warp] = make_float2(s1, s2);
      __syncthreads();
      s1 = s2 = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) s1 += s_part[phase][k].x, s2 += s_part[phase][k].y;
      phase ^= 1;
    }
    if (!live) continue;
    s1 *= inv_width, s2 *= inv_width;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + lane) * VEC;
      if (c >= width) continue;
      float out[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[i] = rstd * (dn[v][i] - s1 - unit[v][i] * s2);
      *reinterpret_cast<Vec<T, VEC>*>(dx + r * width + c) = pack<T, VEC>(out);
    }
  }
  if (partial == nullptr) return;
  float* mine = partial + int64_t(blockIdx.x) * 2 * width;
  if constexpr (kRows == 1) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = (v * G + lane) * VEC + i;
        if (c < width) mine[c] = dw[v][i], mine[width + c] = db[v][i];
      }
  } else {  // the block's groups in order
    __shared__ float s_cols[kRows][2][G * NV * VEC];
    const int group = threadIdx.x / G;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = (v * G + lane) * VEC + i;
        s_cols[group][0][c] = dw[v][i], s_cols[group][1][c] = db[v][i];
      }
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += RowGroup<G>::kThreads) {
      float a = 0.f, d = 0.f;
#pragma unroll
      for (int k = 0; k < kRows; ++k) a += s_cols[k][0][c], d += s_cols[k][1][c];
      mine[c] = a, mine[width + c] = d;
    }
  }
}

// Column sums of partial [blocks, 2, width] in block order, FP64: 32 columns a block, eight runs of blocks.
__global__ void __launch_bounds__(256) layer_norm_param_grad_kernel(const float* __restrict__ partial, int blocks,
                                                                    int width, void* __restrict__ dw,
                                                                    void* __restrict__ db, int param_type) {
  __shared__ double s[8][32];
  const int column = threadIdx.x & 31, run = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + column;
  void* out = blockIdx.y ? db : dw;
  if (out == nullptr) return;  // uniform over the block
  const int per = (blocks + 7) / 8, lo = run * per, hi = min(lo + per, blocks);
  double sum = 0.0;
  if (c < width) {
    const float* p = partial + int64_t(blockIdx.y) * width + c;
#pragma unroll 8
    for (int k = lo; k < hi; ++k) sum += double(p[int64_t(k) * 2 * width]);
  }
  s[run][column] = sum;
  __syncthreads();
  if (run == 0 && c < width) {
#pragma unroll
    for (int k = 1; k < 8; ++k) sum += s[k][column];
    store_param(out, param_type, c, float(sum));
  }
}

// ---- rows too wide for one block's registers: the row is read again for every pass (from L2) ----------------------
constexpr int kWideThreads = 1024;
__device__ __forceinline__ float2 wide_sum(float2 v, float2* s) {
  v.x = warp_sum(v.x), v.y = warp_sum(v.y);
  __syncthreads();
  if (threadIdx.x % 32 == 0) s[threadIdx.x / 32] = v;
  __syncthreads();
  v = s[threadIdx.x % 32];
  return make_float2(warp_sum(v.x), warp_sum(v.y));
}
template <typename T>
__global__ void __launch_bounds__(kWideThreads) layer_norm_wide_fwd_kernel(
    const T* __restrict__ x, int64_t x_stride, const void* __restrict__ weight, const void* __restrict__ bias,
    int param_type, T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
    uint8_t* __restrict__ codes, int64_t rows, int width, float eps) {
  __shared__ float2 s[32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = x + r * x_stride;
    float2 sum = make_float2(0.f, 0.f);
    for (int c = threadIdx.x; c < width; c += kWideThreads) sum.x += to_float(row[c]);
    const float mean = wide_sum(sum, s).x / float(width);
    sum.x = 0.f;
    for (int c = threadIdx.x; c < width; c += kWideThreads) {
      const float d = to_float(row[c]) - mean;
      sum.x = fmaf(d, d, sum.x);
    }
    const float rstd = rsqrtf(wide_sum(sum, s).x / float(width) + eps);
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[r] = mean;
      if (rstd_out) rstd_out[r] = rstd;
    }
    for (int c = threadIdx.x; c < width; c += kWideThreads) {
      const float unit[1] = {(to_float(row[c]) - mean) * rstd};
      const float w = weight ? load_param(weight, param_type, c) : 1.f, b = bias ? load_param(bias, param_type, c) : 0.f;
      y[r * width + c] = from_float<T>(fmaf(unit[0], w, b));
      if (codes) codes[r * width + c] = to_e4m3(unit).e[0];
    }
  }
}
template <typename T>
__device__ __forceinline__ float wide_unit(const T* x_row, const uint8_t* code_row, int c, float mean, float rstd) {
  if (code_row == nullptr) return (to_float(x_row[c]) - mean) * rstd;
  Vec<uint8_t, 1> code{{code_row[c]}};
  float unit[1];
  from_e4m3(code, unit);
  return unit[0];
}
template <typename T>
__global__ void __launch_bounds__(kWideThreads) layer_norm_wide_dx_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, int64_t x_stride, const uint8_t* __restrict__ codes,
    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, const void* __restrict__ weight,
    int param_type, T* __restrict__ dx, int64_t rows, int width) {
  __shared__ float2 s[32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float rstd = rstd_in[r], mean = codes ? 0.f : mean_in[r];
    const T* x_row = codes ? nullptr : x + r * x_stride;
    const uint8_t* code_row = codes ? codes + r * width : nullptr;
    float2 sum = make_float2(0.f, 0.f);
    for (int c = threadIdx.x; c < width; c += kWideThreads) {
      const float dn = to_float(dy[r * width + c]) * (weight ? load_param(weight, param_type, c) : 1.f);
      sum.x += dn;
      sum.y = fmaf(dn, wide_unit(x_row, code_row, c, mean, rstd), sum.y);
    }
    sum = wide_sum(sum, s);
    sum.x /= float(width), sum.y /= float(width);
    for (int c = threadIdx.x; c < width; c += kWideThreads) {
      const float dn = to_float(dy[r * width + c]) * (weight ? load_param(weight, param_type, c) : 1.f);
      dx[r * width + c] = from_float<T>(rstd * (dn - sum.x - wide_unit(x_row, code_row, c, mean, rstd) * sum.y));
    }
  }
}
// partial of row block y (rows y, y + gridDim.y, ...) for 256 columns
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_wide_columns_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, int64_t x_stride, const uint8_t* __restrict__ codes,
    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, float* __restrict__ partial, int64_t rows,
    int width) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= width) return;
  float dw = 0.f, db = 0.f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float d = to_float(dy[r * width + c]);
    dw = fmaf(d, wide_unit(codes ? nullptr : x + r * x_stride, codes ? codes + r * width : nullptr, c,
                           codes ? 0.f : mean_in[r], rstd_in[r]), dw);
    db += d;
  }
  float* mine = partial + int64_t(blockIdx.y) * 2 * width;
  mine[c] = dw, mine[width + c] = db;
}

}  // namespace mek

namespace {

using namespace mek;

struct LnPlan {
  int vec, group, nv;  // group = 0: the wide kernels
  int grid;            // blocks of the backward (= rows of the partial sums)
};

// vec: elements per access, 16 bytes where every row starts on a 16-byte boundary, else one.  The smallest group
// of threads that holds a row in at most 16 elements a thread where accesses are wide, 8 where they are not.
LnPlan ln_plan(int64_t rows, int width, int type, bool aligned) {
  const int wide = type == kTypeFp32 ? 4 : 8;
  LnPlan p{aligned ? wide : 1, 0, 0, 0};
  static const int groups[] = {32, 128, 256, 512, 1024};
  const int most = p.vec > 1 ? 16 / p.vec : 8;
  for (int g : groups) {
    if (g * p.vec * most < width && !(g == 1024 && g * p.vec * 2 * most >= width)) continue;
    p.group = g;
    p.nv = 1;
    while (g * p.vec * p.nv < width) p.nv *= 2;
    break;
  }
  const int per_sm = p.group == 0 ? 2 : p.group <= 128 ? 8 : 1024 / p.group;
  const int64_t blocks = p.group == 32 ? (rows + 3) / 4 : rows;
  p.grid = int(blocks < kLnSms * per_sm ? blocks : kLnSms * per_sm);
  return p;
}

template <typename T, int VEC, int G, int NV>
int ln_fwd(const LnPlan& p, const void* x, int64_t xs, const void* w, const void* b, int pt, void* y, float* mean,
           float* rstd, uint8_t* codes, int64_t rows, int width, float eps, cudaStream_t s) {
  layer_norm_fwd_kernel<T, VEC, G, NV><<<p.grid, RowGroup<G>::kThreads, 0, s>>>(
      static_cast<const T*>(x), xs, w, b, pt, static_cast<T*>(y), mean, rstd, codes, rows, width, eps);
  return launched("layer_norm_fwd");
}
template <typename T, int VEC, int G, int NV>
int ln_bwd(const LnPlan& p, const void* dy, const void* x, int64_t xs, const uint8_t* codes, const float* mean,
           const float* rstd, const void* w, int pt, void* dx, float* partial, int64_t rows, int width,
           cudaStream_t s) {
  if (codes)
    layer_norm_bwd_kernel<T, VEC, G, NV, true><<<p.grid, RowGroup<G>::kThreads, 0, s>>>(
        static_cast<const T*>(dy), nullptr, 0, codes, mean, rstd, w, pt, static_cast<T*>(dx), partial, rows, width);
  else
    layer_norm_bwd_kernel<T, VEC, G, NV, false><<<p.grid, RowGroup<G>::kThreads, 0, s>>>(
        static_cast<const T*>(dy), static_cast<const T*>(x), xs, nullptr, mean, rstd, w, pt, static_cast<T*>(dx),
        partial, rows, width);
  return launched("layer_norm_bwd");
}

// One case per (group, vectors a thread) the plan can give for VEC.
#define MEK_LN_SHAPES(T, VEC, CALL)                                                          \
  do {                                                                                       \
    if constexpr (VEC == 1) {                                                                \
      if (p.group == 32 && p.nv == 1) return CALL(T, 1, 32, 1);                              \
      if (p.group == 32 && p.nv == 2) return CALL(T, 1, 32, 2);                              \
      if (p.group == 32 && p.nv == 4) return CALL(T, 1, 32, 4);                              \
      if (p.group == 32 && p.nv == 8) return CALL(T, 1, 32, 8);                              \
      if (p.group == 128 && p.nv == 4) return CALL(T, 1, 128, 4);                            \
      if (p.group == 128 && p.nv == 8) return CALL(T, 1, 128, 8);                            \
      if (p.group == 256 && p.nv == 8) return CALL(T, 1, 256, 8);                            \
      if (p.group == 512 && p.nv == 8) return CALL(T, 1, 512, 8);                            \
      if (p.group == 1024 && p.nv == 8) return CALL(T, 1, 1024, 8);                          \
      if (p.group == 1024 && p.nv == 16) return CALL(T, 1, 1024, 16);                        \
    } else {                                                                                 \
      constexpr int kMost = 16 / VEC;                                                        \
      if (p.group == 32 && p.nv == 1) return CALL(T, VEC, 32, 1);                            \
      if (p.group == 32 && p.nv == 2) return CALL(T, VEC, 32, 2);                            \
      if (p.group == 32 && p.nv == 4) return CALL(T, VEC, 32, 4);                            \
      if (p.group == 128 && p.nv == 1) return CALL(T, VEC, 128, 1);                          \
      if (p.group == 128 && p.nv == 2) return CALL(T, VEC, 128, 2);                          \
      if (p.group == 128 && p.nv == 4) return CALL(T, VEC, 128, 4);                          \
      if (p.group == 256 && p.nv == kMost) return CALL(T, VEC, 256, kMost);                  \
      if (p.group == 512 && p.nv == kMost) return CALL(T, VEC, 512, kMost);                  \
      if (p.group == 1024 && p.nv == kMost) return CALL(T, VEC, 1024, kMost);                \
      if (p.group == 1024 && p.nv == 2 * kMost) return CALL(T, VEC, 1024, 2 * kMost);        \
    }                                                                                        \
  } while (0)

int check_ln(const char* what, int type, int param_type, int64_t rows, int64_t width, int64_t x_stride) {
  if (type < kTypeBf16 || type > kTypeFp32 || param_type < kTypeBf16 || param_type > kTypeFp32)
    return fail(MEK_ERR_UNSUPPORTED, "%s: an element type is 0 (bf16), 1 (fp16) or 2 (fp32)", what);
  if (rows <= 0 || width <= 0 || width > (1 << 24))
    return fail(MEK_ERR_INVALID, "%s: rows=%lld must be positive and width=%lld in [1, 2^24]", what, (long long)rows,
                (long long)width);
  if (x_stride < 0) return fail(MEK_ERR_INVALID, "%s: a negative row stride", what);
  return MEK_OK;
}

bool ln_aligned(int type, int64_t width, int64_t x_stride, const void* a, const void* b, const void* c) {
  const int wide = type == kTypeFp32 ? 4 : 8;
  return width % wide == 0 && x_stride % wide == 0 &&
         (reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c)) % 16 == 0;
}

}  // namespace

extern "C" {

int mek_layer_norm_partial_rows(int64_t rows, int64_t width, int type) {
  if (rows <= 0 || width <= 0 || width > (1 << 24)) return 0;
  const LnPlan a = ln_plan(rows, int(width), type, true), b = ln_plan(rows, int(width), type, false);
  return a.grid > b.grid ? a.grid : b.grid;
}

int mek_layer_norm_fwd(const void* x, int type, const void* weight, const void* bias, int param_type, void* y,
                       float* mean, float* rstd, uint8_t* codes, int64_t rows, int64_t width, int64_t x_row_stride,
                       float eps, void* stream) {
  if (!x || !y) return fail(MEK_ERR_INVALID, "layer_norm_fwd: a null pointer");
  if (int rc = check_ln("layer_norm_fwd", type, param_type, rows, width, x_row_stride)) return rc;
  if (codes && width > 200704)
    return fail(MEK_ERR_UNSUPPORTED, "layer_norm_fwd: the 8-bit checkpoint holds rows of up to 200,704 columns");
  const LnPlan p = ln_plan(rows, int(width), type, ln_aligned(type, width, x_row_stride, x, y, nullptr) &&
                                                       reinterpret_cast<uintptr_t>(codes) % 8 == 0);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
#define MEK_LN_FWD(T, VEC, G, NV) \
  ln_fwd<T, VEC, G, NV>(p, x, x_row_stride, weight, bias, param_type, y, mean, rstd, codes, rows, int(width), eps, s)
#define MEK_LN_FWD_OF(T, WIDE)                                                                                        \
  do {                                                                                                                \
    if (p.group == 0) {                                                                                               \
      layer_norm_wide_fwd_kernel<T><<<p.grid, kWideThreads, 0, s>>>(static_cast<const T*>(x), x_row_stride, weight,   \
                                                                    bias, param_type, static_cast<T*>(y), mean, rstd, \
                                                                    codes, rows, int(width), eps);                    \
      return launched("layer_norm_fwd");                                                                              \
    }                                                                                                                 \
    if (p.vec == 1) MEK_LN_SHAPES(T, 1, MEK_LN_FWD);                                                                  \
    else MEK_LN_SHAPES(T, WIDE, MEK_LN_FWD);                                                                          \
  } while (0)
  if (type == kTypeBf16) MEK_LN_FWD_OF(__nv_bfloat16, 8);
  if (type == kTypeFp16) MEK_LN_FWD_OF(__half, 8);
  if (type == kTypeFp32) MEK_LN_FWD_OF(float, 4);
  return fail(MEK_ERR_UNSUPPORTED, "layer_norm_fwd: no kernel for width %lld", (long long)width);
}

int mek_layer_norm_bwd(const void* dy, const void* x, int type, const uint8_t* codes, const float* mean,
                       const float* rstd, const void* weight, int param_type, void* dx, float* partial, void* dw,
                       void* db, int64_t rows, int64_t width, int64_t x_row_stride, void* stream) {
  if (!dy || !rstd || !dx || (!codes && (!x || !mean))) return fail(MEK_ERR_INVALID, "layer_norm_bwd: a null pointer");
  if ((dw || db) != (partial != nullptr))
    return fail(MEK_ERR_INVALID, "layer_norm_bwd: the parameters' gradients and their partial sums go together");
  if (int rc = check_ln("layer_norm_bwd", type, param_type, rows, width, codes ? 0 : x_row_stride)) return rc;
  const LnPlan p =
      ln_plan(rows, int(width), type, ln_aligned(type, width, codes ? 0 : x_row_stride, dy, dx, codes ? nullptr : x) &&
                                          reinterpret_cast<uintptr_t>(codes) % 8 == 0);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int w = int(width);
  auto main_launch = [&]() -> int {
#define MEK_LN_BWD(T, VEC, G, NV) \
  ln_bwd<T, VEC, G, NV>(p, dy, x, x_row_stride, codes, mean, rstd, weight, param_type, dx, partial, rows, w, s)
#define MEK_LN_BWD_OF(T, WIDE)                                                                                      \
  do {                                                                                                              \
    if (p.group == 0) {                                                                                             \
      const T* xr = static_cast<const T*>(x);                                                                       \
      const T* g = static_cast<const T*>(dy);                                                                       \
      layer_norm_wide_dx_kernel<T><<<p.grid, kWideThreads, 0, s>>>(g, xr, x_row_stride, codes, mean, rstd, weight,  \
                                                                   param_type, static_cast<T*>(dx), rows, w);       \
      if (int rc = launched("layer_norm_bwd")) return rc;                                                           \
      if (partial) {                                                                                                \
        layer_norm_wide_columns_kernel<T><<<dim3((w + 255) / 256, p.grid), 256, 0, s>>>(g, xr, x_row_stride, codes, \
                                                                                        mean, rstd, partial, rows, w); \
        return launched("layer_norm_bwd (columns)");                                                                \
      }                                                                                                             \
      return MEK_OK;                                                                                                \
    }                                                                                                               \
    if (p.vec == 1) MEK_LN_SHAPES(T, 1, MEK_LN_BWD);                                                                \
    else MEK_LN_SHAPES(T, WIDE, MEK_LN_BWD);                                                                        \
  } while (0)
    if (type == kTypeBf16) MEK_LN_BWD_OF(__nv_bfloat16, 8);
    if (type == kTypeFp16) MEK_LN_BWD_OF(__half, 8);
    if (type == kTypeFp32) MEK_LN_BWD_OF(float, 4);
    return fail(MEK_ERR_UNSUPPORTED, "layer_norm_bwd: no kernel for width %lld", (long long)width);
  };
  if (int rc = main_launch()) return rc;
  if (partial) {
    layer_norm_param_grad_kernel<<<dim3((w + 31) / 32, 2), 256, 0, s>>>(partial, p.grid, w, dw, db, param_type);
    return launched("layer_norm_bwd (parameters)");
  }
  return MEK_OK;
}

}  // extern "C"

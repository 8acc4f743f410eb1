// SiLU-gated RMSNorm over rows of 128, forward and backward, sm_100a: the output norm of the GDN layer,
//     rstd = 1 / sqrt(mean(x^2) + eps),   y = bf16(((x rstd) w) silu(z))                               (FP32 inside)
// (reference: miles_ext_kernels/cake/_impl/gated_rmsnorm/ops.py:8-24; closed-form backward as in
// tests/cake/gated_rmsnorm/inputs.py:75-95).  HBM-bound row work: one warp per row, 8 bytes per lane and tensor, x
// and the gate z read where they lie (each with its own token and head stride: z is usually a column slice of the
// layer's input projection).
//
// The weight gradient sums a term per row.  Every reduction has a fixed order: a warp adds the terms of its rows in
// row order (FP32), a block adds its 8 warps in warp order (FP32), and a second launch adds the blocks' partial sums
// in block order in FP64.  The number of blocks is a function of the row count alone, so identical inputs give
// identical bits.
//
// 8-bit checkpoint: the forward may also write what the backward needs as e4m3 codes -- the normalised row n = x rstd,
// whose values stay below sqrt(128) and need no scale, and z under one power of two a row (exact to divide by, so
// the code's rounding is the only error) -- and the backward read them in the place of x and z: 2 bytes an element kept
// instead of 4.  1,048,576 rows: forward 217 us = 4.9 TB/s, backward 238 us = 4.5 TB/s (copy: 6.5), bound by instructions
// (67 - 70 % of the issue slots: two MUFU operations and about 20 others an element).
#include "common.cuh"
#include "rowio.cuh"
#include "umma.cuh"

namespace mek {

constexpr int kNormRowsPerBlock = 32;  // 8 warps x 2 half-warps x 2 rows in flight
constexpr int kNormMaxBlocks = 148 * 4;

struct RowView {
  const __nv_bfloat16* base;
  int64_t token_stride, head_stride;
  __device__ __forceinline__ const __nv_bfloat16* row(int64_t token, int64_t head) const {
    return base + token * token_stride + head * head_stride;
  }
};
// Rows r0 and r0 + 1 (the last row for what lies past it) as (token, head): one division for both.
struct TwoRows {
  int64_t token[2], head[2];
  __device__ __forceinline__ TwoRows(int64_t r0, int64_t rows, int heads) {
    const int64_t r = r0 < rows ? r0 : rows - 1;
    token[0] = r / heads, head[0] = r - token[0] * heads;
    const bool turn = head[0] + 1 == heads, more = r0 + 1 < rows;
    token[1] = token[0] + (more && turn ? 1 : 0);
    head[1] = !more ? head[0] : turn ? 0 : head[0] + 1;
  }
};

// A half-warp owns a row: 16 lanes x 16 bytes.
__device__ __forceinline__ void load8(const __nv_bfloat16* p, int l16, float* v) {
  const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p) + l16);
  const float2 a = unpack_bf16(raw.x), b = unpack_bf16(raw.y), c = unpack_bf16(raw.z), d = unpack_bf16(raw.w);
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, int l16, const float* v) {
  reinterpret_cast<uint4*>(p)[l16] =
      make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}
__device__ __forceinline__ float half_warp_sum(float x) {
#pragma unroll
  for (int m = 8; m >= 1; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
  return x;
}

__device__ __forceinline__ float half_warp_max(float x) {
#pragma unroll
  for (int m = 8; m >= 1; m >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, m));
  return x;
}

// The smallest e >= -126 with most <= 448 2^e, from the bits of most >= 0 (448 = 0.875 2^9).
__device__ __forceinline__ int e4m3_exponent(float most) {
  const int bits = __float_as_int(most);
  return max((bits >> 23) - 135 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0), -126);
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// A row of the checkpoint: codes of n and of z 2^-e, e (biased by 127), rstd.
struct NormCheckpoint {
  uint8_t *n_codes, *z_codes, *z_exponent;
  float* rstd;
};

// kKeep: the checkpoint is written too; y does not depend on it.
template <bool kKeep>
__global__ void __launch_bounds__(256) gated_rmsnorm_fwd_kernel(RowView x, RowView z, const __nv_bfloat16* __restrict__ w,
                                                                __nv_bfloat16* __restrict__ y, int64_t rows, int heads,
                                                                float eps, NormCheckpoint keep) {
  const int l16 = threadIdx.x & 15, half = threadIdx.x >> 4;  // 16 half-warps per block, 2 rows each
  const int64_t r0 = int64_t(blockIdx.x) * kNormRowsPerBlock + half * 2;
  float wv[8], xv[2][8], zv[2][8];
  load8(w, l16, wv);
  const TwoRows at(r0, rows, heads);
#pragma unroll
  for (int i = 0; i < 2; ++i) {  // both rows' loads in flight before any arithmetic
    load8(x.row(at.token[i], at.head[i]), l16, xv[i]);
    load8(z.row(at.token[i], at.head[i]), l16, zv[i]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float ss = 0.f, out[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(xv[i][j], xv[i][j], ss);
    const float rstd = rsqrtf(half_warp_sum(ss) * (1.0f / 128.0f) + eps);
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = ((xv[i][j] * rstd) * wv[j]) * __fdividef(zv[i][j], 1.0f + __expf(-zv[i][j]));
    if (r0 + i < rows) store8(y + (r0 + i) * 128, l16, out);
    if constexpr (kKeep) {
      float most = 0.f, n[8], scaled[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) most = fmaxf(most, isfinite(zv[i][j]) ? fabsf(zv[i][j]) : 0.f);
      const int e = e4m3_exponent(half_warp_max(most));
      const float down = power_of_two(-e);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        n[j] = xv[i][j] * rstd;
        scaled[j] = isfinite(zv[i][j]) ? zv[i][j] * down : __int_as_float(0x7fffffff);  // e4m3 has NaN, no infinity
      }
      if (r0 + i < rows) {
        const int64_t r = r0 + i;
        store_codes(keep.n_codes + r * 128 + l16 * 8, n);
        store_codes(keep.z_codes + r * 128 + l16 * 8, scaled);
        if (l16 == 0) keep.z_exponent[r] = uint8_t(e + 127), keep.rstd[r] = rstd;
      }
    }
  }
}

// The backward from the checkpoint; formulas as below with n and z as the codes hold them.  A half-warp's row of the next
// group is loaded, as it lies in memory, as soon as the present one is decoded.
struct KeptRow {
  Codes<8> n, z;
  uint4 dy;
  float rstd;
  uint8_t exponent;
  __device__ __forceinline__ void load(const NormCheckpoint& kept, const __nv_bfloat16* dy_in, int64_t r, int l16) {
    n = load_codes<8>(kept.n_codes + r * 128 + l16 * 8);
    z = load_codes<8>(kept.z_codes + r * 128 + l16 * 8);
    dy = __ldg(reinterpret_cast<const uint4*>(dy_in + r * 128) + l16);
    rstd = kept.rstd[r];
    exponent = kept.z_exponent[r];
  }
};
__global__ void __launch_bounds__(256, 3) gated_rmsnorm_bwd_kept_kernel(const __nv_bfloat16* __restrict__ dy,
                                                                        NormCheckpoint kept,
                                                                        const __nv_bfloat16* __restrict__ w,
                                                                        __nv_bfloat16* __restrict__ dx,
                                                                        __nv_bfloat16* __restrict__ dz,
                                                                        float* __restrict__ dw_partial, int64_t rows) {
  __shared__ float s_dw[16][128];
  const int l16 = threadIdx.x & 15, half = threadIdx.x >> 4;
  float wv[8], acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  load8(w, l16, wv);
  const int64_t step = int64_t(gridDim.x) * kNormRowsPerBlock, first = int64_t(blockIdx.x) * kNormRowsPerBlock;
  KeptRow row[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) row[i].load(kept, dy, min(first + half * 2 + i, rows - 1), l16);
  for (int64_t group = first; group < rows; group += step) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t r = group + half * 2 + i;
      const bool live = r < rows;  // uniform over the half-warp
      const float up = power_of_two(int(row[i].exponent) - 127), rstd = row[i].rstd;
      float n[8], zv[8], gv[8], dn[8], dzv[8], dxv[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 a = code_pair(row[i].n, q), b = code_pair(row[i].z, q);
        n[2 * q] = a.x, n[2 * q + 1] = a.y, zv[2 * q] = b.x, zv[2 * q + 1] = b.y;
      }
      const float2 g0 = unpack_bf16(row[i].dy.x), g1 = unpack_bf16(row[i].dy.y), g2 = unpack_bf16(row[i].dy.z),
                   g3 = unpack_bf16(row[i].dy.w);
      gv[0] = g0.x, gv[1] = g0.y, gv[2] = g1.x, gv[3] = g1.y, gv[4] = g2.x, gv[5] = g2.y, gv[6] = g3.x, gv[7] = g3.y;
      if (r + step < rows) row[i].load(kept, dy, r + step, l16);
      float dot = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float z = zv[j] * up;
        const float s = __fdividef(1.0f, 1.0f + __expf(-z));
        const float a = gv[j] * (z * s);
        dn[j] = a * wv[j];
        dot = fmaf(dn[j], n[j], dot);
        dzv[j] = gv[j] * n[j] * wv[j] * s * (1.0f + z * (1.0f - s));
        if (live) acc[j] = fmaf(a, n[j], acc[j]);
      }
      const float mean = half_warp_sum(dot) * (1.0f / 128.0f);
#pragma unroll
      for (int j = 0; j < 8; ++j) dxv[j] = rstd * (dn[j] - n[j] * mean);
      if (live) {
        store8(dx + r * 128, l16, dxv);
        store8(dz + r * 128, l16, dzv);
      }
    }
  }
  if (dw_partial == nullptr) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) s_dw[half][l16 * 8 + j] = acc[j];
  __syncthreads();
  if (threadIdx.x < 128) {
    float sum = 0.f;
#pragma unroll
    for (int hw = 0; hw < 16; ++hw) sum += s_dw[hw][threadIdx.x];
    dw_partial[int64_t(blockIdx.x) * 128 + threadIdx.x] = sum;
  }
}

// dx = rstd dn - x rstd^3 mean(dn x), dn = dy silu(z) w;  dz = dy n w s (1 + z (1 - s)), n = x rstd, s = sigmoid(z);
// dw += dy silu(z) n.  Block b takes the row groups b, b + gridDim.x, ...
__global__ void __launch_bounds__(256) gated_rmsnorm_bwd_kernel(const __nv_bfloat16* __restrict__ dy, RowView x, RowView z,
                                                                const __nv_bfloat16* __restrict__ w,
                                                                __nv_bfloat16* __restrict__ dx,
                                                                __nv_bfloat16* __restrict__ dz,
                                                                float* __restrict__ dw_partial, int64_t rows, int heads,
                                                                float eps) {
  __shared__ float s_dw[16][128];
  const int l16 = threadIdx.x & 15, half = threadIdx.x >> 4;
  float wv[8], acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  load8(w, l16, wv);
  for (int64_t group = blockIdx.x; group * kNormRowsPerBlock < rows; group += gridDim.x) {
    const int64_t r0 = group * kNormRowsPerBlock + half * 2;
    float xv[2][8], zv[2][8], gv[2][8];
    const TwoRows at(r0, rows, heads);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t r = r0 + i < rows ? r0 + i : rows - 1;
      load8(x.row(at.token[i], at.head[i]), l16, xv[i]);
      load8(z.row(at.token[i], at.head[i]), l16, zv[i]);
      load8(dy + r * 128, l16, gv[i]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool live = r0 + i < rows;  // uniform over the half-warp
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(xv[i][j], xv[i][j], ss);
      const float rstd = rsqrtf(half_warp_sum(ss) * (1.0f / 128.0f) + eps);
      float dot = 0.f, dn[8], dzv[8], dxv[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float s = __fdividef(1.0f, 1.0f + __expf(-zv[i][j]));
        const float a = gv[i][j] * (zv[i][j] * s);
        const float n = xv[i][j] * rstd;
        dn[j] = a * wv[j];
        dot = fmaf(dn[j], xv[i][j], dot);
        dzv[j] = gv[i][j] * n * wv[j] * s * (1.0f + zv[i][j] * (1.0f - s));
        if (live) acc[j] = fmaf(a, n, acc[j]);
      }
      const float mean = half_warp_sum(dot) * (1.0f / 128.0f);
      const float r3 = rstd * rstd * rstd;
#pragma unroll
      for (int j = 0; j < 8; ++j) dxv[j] = rstd * dn[j] - xv[i][j] * r3 * mean;
      if (live) {
        store8(dx + (r0 + i) * 128, l16, dxv);
        store8(dz + (r0 + i) * 128, l16, dzv);
      }
    }
  }
  if (dw_partial == nullptr) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) s_dw[half][l16 * 8 + j] = acc[j];
  __syncthreads();
  if (threadIdx.x < 128) {
    float sum = 0.f;
#pragma unroll
    for (int hw = 0; hw < 16; ++hw) sum += s_dw[hw][threadIdx.x];
    dw_partial[int64_t(blockIdx.x) * 128 + threadIdx.x] = sum;
  }
}

__global__ void __launch_bounds__(128) gated_rmsnorm_dw_kernel(const float* __restrict__ dw_partial, int blocks,
                                                               __nv_bfloat16* __restrict__ dw) {
  double sum = 0.0;
  for (int b = 0; b < blocks; ++b) sum += double(dw_partial[int64_t(b) * 128 + threadIdx.x]);
  dw[threadIdx.x] = __float2bfloat16_rn(float(sum));
}

// The same sum for the checkpoint's backward in eight runs of blocks side by side, then the runs in order: one chain of
// 592 FP64 additions takes 29 us, the runs 10.  (The plain backward keeps the one chain: another order of the sum could turn
// the last bit of a weight gradient that callers have had from it.)
constexpr int kNormRuns = 8;
__global__ void __launch_bounds__(128 * kNormRuns) gated_rmsnorm_dw_runs_kernel(const float* __restrict__ dw_partial,
                                                                                int blocks,
                                                                                __nv_bfloat16* __restrict__ dw) {
  __shared__ double s[kNormRuns][128];
  const int column = threadIdx.x & 127, run = threadIdx.x >> 7;
  const int per = (blocks + kNormRuns - 1) / kNormRuns, lo = run * per, hi = min(lo + per, blocks);
  double sum = 0.0;
#pragma unroll 8
  for (int b = lo; b < hi; ++b) sum += double(dw_partial[int64_t(b) * 128 + column]);
  s[run][column] = sum;
  __syncthreads();
  if (run != 0) return;
#pragma unroll
  for (int k = 1; k < kNormRuns; ++k) sum += s[k][column];
  dw[column] = __float2bfloat16_rn(float(sum));
}

}  // namespace mek

namespace {

int norm_blocks(int64_t rows) {
  const int64_t groups = (rows + mek::kNormRowsPerBlock - 1) / mek::kNormRowsPerBlock;
  return int(groups < mek::kNormMaxBlocks ? groups : mek::kNormMaxBlocks);
}

int check_norm(const char* what, int64_t rows, int heads, int64_t xt, int64_t xh, int64_t zt, int64_t zh, const void* x,
               const void* z) {
  using namespace mek;
  if (rows <= 0 || heads <= 0 || rows % heads != 0)
    return fail(MEK_ERR_INVALID, "%s: rows=%lld must be a positive multiple of heads=%d", what, (long long)rows, heads);
  if ((xt | xh | zt | zh) % 8 != 0 || xh < 0 || zh < 0 || xt < 0 || zt < 0)
    return fail(MEK_ERR_INVALID, "%s: token and head strides must be non-negative multiples of 8 elements", what);
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(z)) % 16 != 0)
    return fail(MEK_ERR_INVALID, "%s: x and z must be 16-byte aligned", what);
  return MEK_OK;
}

// What the kernels read and write as dense rows, 16 bytes an access.
int check_dense(const char* what, const void* a, const void* b, const void* c = nullptr, const void* d = nullptr) {
  using namespace mek;
  auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  if ((bits(a) | bits(b) | bits(c) | bits(d)) % 16 != 0)
    return fail(MEK_ERR_INVALID, "%s: the weight, y, dy, dx and dz must be 16-byte aligned", what);
  return MEK_OK;
}

int check_checkpoint(const char* what, const mek::NormCheckpoint& c) {
  using namespace mek;
  if (!c.n_codes || !c.z_codes || !c.z_exponent || !c.rstd) return fail(MEK_ERR_INVALID, "%s: a null pointer", what);
  if ((reinterpret_cast<uintptr_t>(c.n_codes) | reinterpret_cast<uintptr_t>(c.z_codes)) % 8 != 0)
    return fail(MEK_ERR_INVALID, "%s: the codes must be 8-byte aligned", what);
  return MEK_OK;
}

int norm_fwd(const char* what, const void* x, const void* z, const void* weight, void* y,
             const mek::NormCheckpoint* keep, int64_t rows, int heads, int64_t x_token_stride, int64_t x_head_stride,
             int64_t z_token_stride, int64_t z_head_stride, float eps, void* stream) {
  using namespace mek;
  if (!x || !z || !weight || !y) return fail(MEK_ERR_INVALID, "%s: a null pointer", what);
  if (int rc = check_norm(what, rows, heads, x_token_stride, x_head_stride, z_token_stride, z_head_stride, x, z))
    return rc;
  if (int rc = check_dense(what, weight, y)) return rc;
  const RowView xv{static_cast<const __nv_bfloat16*>(x), x_token_stride, x_head_stride};
  const RowView zv{static_cast<const __nv_bfloat16*>(z), z_token_stride, z_head_stride};
  const unsigned grid = unsigned((rows + kNormRowsPerBlock - 1) / kNormRowsPerBlock);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const __nv_bfloat16* w = static_cast<const __nv_bfloat16*>(weight);
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(y);
  if (keep) gated_rmsnorm_fwd_kernel<true><<<grid, 256, 0, s>>>(xv, zv, w, out, rows, heads, eps, *keep);
  else gated_rmsnorm_fwd_kernel<false><<<grid, 256, 0, s>>>(xv, zv, w, out, rows, heads, eps, NormCheckpoint{});
  return launched(what);
}

}  // namespace

extern "C" {

int mek_gated_rmsnorm_partial_rows(int64_t rows) { return rows > 0 ? norm_blocks(rows) : 0; }

int mek_gated_rmsnorm_fwd(const void* x, const void* z, const void* weight, void* y, int64_t rows, int heads,
                          int64_t x_token_stride, int64_t x_head_stride, int64_t z_token_stride, int64_t z_head_stride,
                          float eps, void* stream) {
  return norm_fwd("gated_rmsnorm_fwd", x, z, weight, y, nullptr, rows, heads, x_token_stride, x_head_stride,
                  z_token_stride, z_head_stride, eps, stream);
}

int mek_gated_rmsnorm_fwd_keep(const void* x, const void* z, const void* weight, void* y, uint8_t* n_codes,
                               uint8_t* z_codes, uint8_t* z_exponent, float* rstd, int64_t rows, int heads,
                               int64_t x_token_stride, int64_t x_head_stride, int64_t z_token_stride,
                               int64_t z_head_stride, float eps, void* stream) {
  const mek::NormCheckpoint keep{n_codes, z_codes, z_exponent, rstd};
  if (int rc = check_checkpoint("gated_rmsnorm_fwd_keep", keep)) return rc;
  return norm_fwd("gated_rmsnorm_fwd_keep", x, z, weight, y, &keep, rows, heads, x_token_stride, x_head_stride,
                  z_token_stride, z_head_stride, eps, stream);
}

int mek_gated_rmsnorm_bwd_kept(const void* dy, const uint8_t* n_codes, const uint8_t* z_codes,
                               const uint8_t* z_exponent, const float* rstd, const void* weight, void* dx, void* dz,
                               float* dw_partial, void* dw, int64_t rows, void* stream) {
  using namespace mek;
  if (!dy || !weight || !dx || !dz) return fail(MEK_ERR_INVALID, "gated_rmsnorm_bwd_kept: a null pointer");
  const NormCheckpoint kept{const_cast<uint8_t*>(n_codes), const_cast<uint8_t*>(z_codes),
                            const_cast<uint8_t*>(z_exponent), const_cast<float*>(rstd)};
  if (int rc = check_checkpoint("gated_rmsnorm_bwd_kept", kept)) return rc;
  if ((dw == nullptr) != (dw_partial == nullptr))
    return fail(MEK_ERR_INVALID, "gated_rmsnorm_bwd_kept: dw and its partial sums go together");
  if (int rc = check_dense("gated_rmsnorm_bwd_kept", weight, dy, dx, dz)) return rc;
  if (rows <= 0) return fail(MEK_ERR_INVALID, "gated_rmsnorm_bwd_kept: rows=%lld must be positive", (long long)rows);
  const int blocks = norm_blocks(rows);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  gated_rmsnorm_bwd_kept_kernel<<<blocks, 256, 0, s>>>(static_cast<const __nv_bfloat16*>(dy), kept,
                                                       static_cast<const __nv_bfloat16*>(weight),
                                                       static_cast<__nv_bfloat16*>(dx), static_cast<__nv_bfloat16*>(dz),
                                                       dw_partial, rows);
  if (int rc = launched("gated_rmsnorm_bwd_kept")) return rc;
  if (dw != nullptr) {
    gated_rmsnorm_dw_runs_kernel<<<1, 128 * kNormRuns, 0, s>>>(dw_partial, blocks, static_cast<__nv_bfloat16*>(dw));
    return launched("gated_rmsnorm_bwd_kept (weight gradient)");
  }
  return MEK_OK;
}

int mek_gated_rmsnorm_bwd(const void* dy, const void* x, const void* z, const void* weight, void* dx, void* dz,
                          float* dw_partial, void* dw, int64_t rows, int heads, int64_t x_token_stride,
                          int64_t x_head_stride, int64_t z_token_stride, int64_t z_head_stride, float eps,
                          void* stream) {
  using namespace mek;
  if (!dy || !x || !z || !weight || !dx || !dz) return fail(MEK_ERR_INVALID, "gated_rmsnorm_bwd: a null pointer");
  if ((dw == nullptr) != (dw_partial == nullptr))
    return fail(MEK_ERR_INVALID, "gated_rmsnorm_bwd: dw and its partial sums go together");
  if (int rc = check_norm("gated_rmsnorm_bwd", rows, heads, x_token_stride, x_head_stride, z_token_stride,
                          z_head_stride, x, z))
    return rc;
  if (int rc = check_dense("gated_rmsnorm_bwd", weight, dy, dx, dz)) return rc;
  const RowView xv{static_cast<const __nv_bfloat16*>(x), x_token_stride, x_head_stride};
  const RowView zv{static_cast<const __nv_bfloat16*>(z), z_token_stride, z_head_stride};
  const int blocks = norm_blocks(rows);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  gated_rmsnorm_bwd_kernel<<<blocks, 256, 0, s>>>(static_cast<const __nv_bfloat16*>(dy), xv, zv,
                                                  static_cast<const __nv_bfloat16*>(weight),
                                                  static_cast<__nv_bfloat16*>(dx), static_cast<__nv_bfloat16*>(dz),
                                                  dw_partial, rows, heads, eps);
  if (int rc = launched("gated_rmsnorm_bwd")) return rc;
  if (dw != nullptr) {
    gated_rmsnorm_dw_kernel<<<1, 128, 0, s>>>(dw_partial, blocks, static_cast<__nv_bfloat16*>(dw));
    return launched("gated_rmsnorm_bwd (weight gradient)");
  }
  return MEK_OK;
}

}  // extern "C"

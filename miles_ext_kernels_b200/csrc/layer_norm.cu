// LayerNorm over rows of any width, forward and backward, sm_100a:
//     mean = sum(x) / C,  rstd = 1 / sqrt(sum((x - mean)^2) / C + eps),  unit = (x - mean) rstd,  y = unit w + b
//     dn = dy w,  dx = rstd (dn - mean(dn) - unit mean(dn unit)),  dw = sum_rows dy unit,  db = sum_rows dy
// FP32 inside, one rounding per output.  HBM-bound: a row's elements stay in registers between the statistics and the
// output, so each tensor crosses HBM once.  The variance is taken about the mean (never as mean(x^2) - mean^2), per
// warp first and then across the warps by Chan's rule (T. Chan, G. Golub, R. LeVeque, 1979), which costs one block
// barrier a row instead of two.
//
// The weight and bias gradients: a thread owns the same columns in every row of its block and sums them in FP32
// registers; a second launch adds the blocks' sums in FP64 in a fixed order.  The grid is a function of the extents and
// of the rows' alignment, so identical inputs give identical bits.
//
// Arithmetic on packed pairs of FP32 (half the instructions; a row of 16 elements a thread took 427 of them scalar, which
// bounded it), rows of a whole block streamed by bulk copies, narrow rows side by side in a warp.  Measured, bf16:
// 32,768 x 4,096 forward 110 us = 4.9 TB/s, backward 155 us = 5.2 TB/s with the last sums (copy: 6.5); 16,384 x 8,192
// with the checkpoint 139 + 149 us; 65,536 x 2,048 98 + 150.  What bounds it: the chain of a row's phases (wait, sums,
// shuffles, barrier, output) with three blocks an SM (backward: two), at 60 % of the issue slots; below 512 columns the
// instructions of a row.
//
// 8-bit checkpoint: the forward may also write unit as e4m3 codes and the backward read them in the place of x and
// mean.  |unit| <= sqrt(C), so up to 448^2 = 200,704 columns the codes need no scale.
#include <type_traits>

#include "common.cuh"
#include "rowio.cuh"
#include "tma.cuh"
#include "umma.cuh"

namespace mek {

constexpr int kLnSms = 148;

constexpr int kLnMaxSlots = 8;

// How a group of G threads holds a row: NV accesses of VEC elements a thread, in packed pairs.  Pair q of a thread:
// neighbouring columns of one access, or (VEC = 1, NV even) the columns of two accesses.
template <typename T, int VEC, int G, int NV>
struct RowShape {
  static constexpr int kThreads = G < 128 ? 128 : G, kRows = kThreads / G, kWarps = G < 32 ? 1 : G / 32;
  static constexpr int kPairs = NV * VEC / 2, kSide = G < 32 ? 32 / G : 1;  // rows a warp holds side by side
  static_assert(NV * VEC % 2 == 0, "pairs");
  static __device__ __forceinline__ int column(int lane, int q, int i) {
    if constexpr (VEC == 1) return (2 * q + i) * G + lane;
    else return (q / (VEC / 2) * G + lane) * VEC + q % (VEC / 2) * 2 + i;
  }
  // elements of a row of `width` that warp w of the group holds
  static __device__ __forceinline__ int count(int w, int width) {
    int n = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) n += min(max(width - (v * G + w * 32) * VEC, 0), min(G, 32) * VEC);
    return n;
  }
};

// A thread's part of a row as it lies in memory (zeros past the row's end), and its pairs.
template <typename E, int VEC, int G, int NV>
struct RowPart {
  Vec<E, VEC> raw[NV];
  __device__ __forceinline__ void load(const E* row, int lane, int width) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + lane) * VEC;
      if (c < width) raw[v] = *reinterpret_cast<const Vec<E, VEC>*>(row + c);
      else
#pragma unroll
        for (int i = 0; i < VEC; ++i) raw[v].e[i] = from_float<E>(0.f);
    }
  }
  __device__ __forceinline__ Two pair(int q) const {
    Vec<E, 2> two_of;
    if constexpr (VEC == 1) two_of = {{raw[2 * q].e[0], raw[2 * q + 1].e[0]}};
    else two_of = {{raw[q / (VEC / 2)].e[q % (VEC / 2) * 2], raw[q / (VEC / 2)].e[q % (VEC / 2) * 2 + 1]}};
    return widened(two_of);
  }
};
template <int VEC, int G, int NV>
struct RowPart<uint8_t, VEC, G, NV> {
  Codes<VEC> raw[NV];
  __device__ __forceinline__ void load(const uint8_t* row, int lane, int width) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + lane) * VEC;
      if (c < width) raw[v] = load_codes<VEC>(row + c);
      else raw[v].clear();
    }
  }
  __device__ __forceinline__ Two pair(int q) const {
    if constexpr (VEC == 1) {
      return two(code_value(raw[2 * q].byte), code_value(raw[2 * q + 1].byte));
    } else {
      const float2 f = code_pair(raw[q / (VEC / 2)], q % (VEC / 2));
      return two(f.x, f.y);
    }
  }
};
template <typename E, int VEC, int G, int NV, typename Value>  // value(q) -> Two
__device__ __forceinline__ void store_row(E* row, int lane, int width, Value value) {
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * G + lane) * VEC;
    if constexpr (VEC == 1) {
      if (v % 2) continue;
      const float2 f = split(value(v / 2));
      if (c < width) row[c] = from_float<E>(f.x);
      if (c + G < width) row[c + G] = from_float<E>(f.y);
    } else {
      if (c >= width) continue;
      float f[VEC];
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        const float2 p = split(value(v * (VEC / 2) + i));
        f[2 * i] = p.x, f[2 * i + 1] = p.y;
      }
      *reinterpret_cast<Vec<E, VEC>*>(row + c) = pack<E, VEC>(f);
    }
  }
}
template <int VEC, int G, int NV, typename Value>
__device__ __forceinline__ void store_row_codes(uint8_t* row, int lane, int width, Value value) {
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * G + lane) * VEC;
    if constexpr (VEC == 1) {
      if (v % 2) continue;
      const float2 f = split(value(v / 2));
      const float a[1] = {f.x}, b[1] = {f.y};
      if (c < width) store_codes(row + c, a);
      if (c + G < width) store_codes(row + c + G, b);
    } else {
      if (c >= width) continue;
      float f[VEC];
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) {
        const float2 p = split(value(v * (VEC / 2) + i));
        f[2 * i] = p.x, f[2 * i + 1] = p.y;
      }
      store_codes(row + c, f);
    }
  }
}

// Over the lanes of a group inside a warp.
template <int G>
__device__ __forceinline__ float lane_sum(float x) {
#pragma unroll
  for (int m = min(G, 32) / 2; m >= 1; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
  return x;
}

// Sums over a group of two values, the warps' sums through shared memory (`phase` alternates: one barrier a row).
template <int G>
__device__ __forceinline__ float2 group_sum(float a, float b, float2 (*part)[32], int phase) {
  a = lane_sum<G>(a), b = lane_sum<G>(b);
  if constexpr (G <= 32) return make_float2(a, b);
  if (threadIdx.x % 32 == 0) part[phase][threadIdx.x / 32] = make_float2(a, b);
  __syncthreads();
  if constexpr (G <= 256) {
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < G / 32; ++w) a += part[phase][w].x, b += part[phase][w].y;
    return make_float2(a, b);
  } else {
    const float2 p = threadIdx.x % 32 < G / 32 ? part[phase][threadIdx.x % 32] : make_float2(0.f, 0.f);
    return make_float2(warp_sum(p.x), warp_sum(p.y));
  }
}

// Where a block's rows come from.  Rows of wide accesses that take a whole block are streamed through shared memory: one
// thread asks for the next rows with bulk copies, `slots` rows ahead, so the loads in flight depend neither on registers
// nor on how far the block is inside a row.  Other rows are loaded a row ahead into registers.
__device__ __forceinline__ void bulk_load(void* to, const void* from, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(to)),
               "l"(from), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
template <int VEC, int G>
constexpr bool kLnStreams = VEC > 1 && G >= 128;
// Rows ahead in registers: where a warp holds rows of its own, four of up to 16 bytes a thread or two of more (narrow rows
// would keep few bytes in flight otherwise), else one.
template <typename T, int VEC, int G, int NV>
constexpr int kLnDepth = G >= 128 ? 1 : NV * VEC * int(sizeof(T)) <= 16 ? 4 : 2;
// Blocks an SM: about 80 registers a thread for the forward, 128 for the backward, whose sums take a third of them (a group
// of 1,024 has 64 either way).
template <int G>
constexpr int kLnFwdBlocks = G <= 32 ? 5 : G == 128 ? 6 : G == 256 ? 3 : 1;
template <int G>
constexpr int kLnBwdBlocks = G <= 128 ? 4 : G == 256 ? 2 : 1;
// The widest rows leave no registers for the parameters, which stay in shared memory: 32 elements a thread of 128 registers
// (16-bit rows; with 1,024 threads of 64 registers the backward took 343 us for 8,192 x 16,384, so it takes 332), or 1,024
// threads.  Both spill in the backward all the same (bytes stored a thread): 278 - 348 with 512 threads, 576 - 596 where the
// codes cannot be streamed; 222 - 516 with 1,024 threads of FP32; 60 - 686 with 1,024 threads and one element an access.
// So do, of the narrower forms, FP32 rows of one warp x 16 elements (backward 280, forward 140) and, in the forward, odd
// 16-bit rows side by side in a warp (122 - 134).
template <int VEC, int G, int NV>
constexpr bool kLnParamsShared = G == 1024 || NV * VEC == 32;

// The parameters of a thread's columns, FP32.
template <typename T, int VEC, int G, int NV>
struct RowParams {
  typedef RowShape<T, VEC, G, NV> Shape;
  Two kept[kLnParamsShared<VEC, G, NV> ? 1 : Shape::kPairs];
  const float* shared;
  int last;  // columns past the row's end read its last parameters, and nobody what comes of it
  __device__ __forceinline__ void load(const void* p, int type, float missing, float* room, int lane, int width) {
    shared = room, last = VEC == 1 ? width - 1 : width - 2;
    if constexpr (kLnParamsShared<VEC, G, NV>) {
      for (int c = lane; c < width; c += G) room[c] = p ? load_param(p, type, c) : missing;
    } else {
#pragma unroll
      for (int q = 0; q < Shape::kPairs; ++q) {
        float f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int c = Shape::column(lane, q, i);
          f[i] = p && c < width ? load_param(p, type, c) : missing;
        }
        kept[q] = two(f[0], f[1]);
      }
    }
  }
  __device__ __forceinline__ Two pair(int q, int lane) const {
    if constexpr (!kLnParamsShared<VEC, G, NV>) return kept[q];
    else if constexpr (VEC == 1)
      return two(shared[min(Shape::column(lane, q, 0), last)], shared[min(Shape::column(lane, q, 1), last)]);
    else return *reinterpret_cast<const Two*>(shared + min(Shape::column(lane, q, 0), last));
  }
};

// x [rows, width] with a row stride; y and codes dense.  Block b takes rows (or groups of rows) b, b + gridDim.x, ...
template <typename T, int VEC, int G, int NV>
__global__ void __launch_bounds__(RowShape<T, VEC, G, NV>::kThreads, kLnFwdBlocks<G>) layer_norm_fwd_kernel(
    const T* __restrict__ x, int64_t x_stride, const void* __restrict__ weight, const void* __restrict__ bias,
    int param_type, T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
    uint8_t* __restrict__ codes, int64_t rows, int width, float eps, int slots, const RowWaits waits) {
  typedef RowShape<T, VEC, G, NV> Shape;
  constexpr bool kStream = kLnStreams<VEC, G>;
  constexpr int kPairs = Shape::kPairs;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 s_part[2][32];
  __shared__ float s_count[32];
  __shared__ uint64_t s_full[kLnMaxSlots];
  const int lane = threadIdx.x % G, warp = lane / 32;
  const uint32_t bytes = uint32_t(width) * sizeof(T);
  const int64_t first = int64_t(blockIdx.x) * Shape::kRows + threadIdx.x / G, step = int64_t(gridDim.x) * Shape::kRows;
  const int64_t served = rows < waits.rows_served ? rows : waits.rows_served;
  if (kStream && threadIdx.x == 0) {
    for (int k = 0; k < slots; ++k) mbar_init(&s_full[k], 1);
    fence_mbar_init();
    for (int k = 0; k < slots && first + k * step < served; ++k) {
      mbar_arrive_expect(&s_full[k], bytes);
      bulk_load(smem + k * bytes, x + (first + k * step) * x_stride, bytes, &s_full[k]);
    }
  }
  float* room = reinterpret_cast<float*>(smem + size_t(kStream ? slots : 0) * bytes);
  RowParams<T, VEC, G, NV> w, b;
  w.load(weight, param_type, 1.f, room, lane, width);
  b.load(bias, param_type, 0.f, room + width, lane, width);
  if (threadIdx.x < Shape::kWarps) s_count[threadIdx.x] = float(Shape::count(threadIdx.x, width));
  const int count = Shape::count(warp, width);
  const float inv_count = count ? 1.f / float(count) : 0.f, inv_width = 1.f / float(width);
  const bool full = Shape::column(lane, kPairs - 1, 1) < width;  // no column past the row's end
  constexpr int kDepth = kStream ? 1 : kLnDepth<T, VEC, G, NV>;
  RowPart<T, VEC, G, NV> parts[kDepth];
  if constexpr (!kStream) {
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
      if (Shape::kSide > 1) parts[k].load(x, lane, 0);  // zeros where a warp's last rows are not all there
      if (first + k * step < rows) parts[k].load(x + (first + k * step) * x_stride, lane, width);
    }
  }
  __syncthreads();
  int slot = 0, parity = 0, phase = 0;
  bool failed = false;  // a wait ran out: the rows from there on are NaN, and nothing waits again
  auto one_row = [&](int64_t r, RowPart<T, VEC, G, NV>& part) {
    const bool live = Shape::kSide == 1 || r < rows;  // rows side by side in a warp go through its shuffles together
    if constexpr (kStream) {
      if (!failed) failed = !mbar_wait_soon(&s_full[slot], parity, waits.limit_ns);
      part.load(reinterpret_cast<const T*>(smem + slot * bytes), lane, width);
    }
    Two xv[kPairs], sum = two(0.f);
#pragma unroll
    for (int q = 0; q < kPairs; ++q) xv[q] = part.pair(q), sum = add2(sum, xv[q]);
    if constexpr (!kStream)
      if (r + kDepth * step < rows) part.load(x + (r + kDepth * step) * x_stride, lane, width);
    // this warp's mean and squares about it; a mean is rounded before it is subtracted, whether or not it is stored: the
    // same y either way
    float2 s = split(sum);
    if (failed) s.x = __int_as_float(0x7fffffff);
    float total = lane_sum<G>(s.x + s.y);
    float mean = __fmul_rn(total, inv_count);
    Two squares = two(0.f);
    const Two mean2 = two(mean);
    if (full) {
#pragma unroll
      for (int q = 0; q < kPairs; ++q) {
        const Two d = sub2(xv[q], mean2);
        squares = fma2(d, d, squares);
      }
    } else {
#pragma unroll
      for (int q = 0; q < kPairs; ++q) {
        const float2 d = split(sub2(xv[q], mean2));
        const Two in = two(Shape::column(lane, q, 0) < width ? d.x : 0.f, Shape::column(lane, q, 1) < width ? d.y : 0.f);
        squares = fma2(in, in, squares);
      }
    }
    s = split(squares);
    float m2 = lane_sum<G>(s.x + s.y);
    if constexpr (G > 32) {  // the warps' by Chan's rule
      if (threadIdx.x % 32 == 0) s_part[phase][warp] = make_float2(mean, m2);
      __syncthreads();
      if (kStream && threadIdx.x == 0 && !failed && r + slots * step < served) {  // everybody has the row in registers
        mbar_arrive_expect(&s_full[slot], bytes);
        bulk_load(smem + slot * bytes, x + (r + slots * step) * x_stride, bytes, &s_full[slot]);
      }
      if constexpr (G <= 256) {
        total = m2 = 0.f;
#pragma unroll
        for (int k = 0; k < Shape::kWarps; ++k) total = fmaf(s_part[phase][k].x, s_count[k], total);
        mean = __fmul_rn(total, inv_width);
#pragma unroll
        for (int k = 0; k < Shape::kWarps; ++k) {
          const float d = s_part[phase][k].x - mean;
          m2 += fmaf(s_count[k] * d, d, s_part[phase][k].y);
        }
      } else {
        const bool in = threadIdx.x % 32 < Shape::kWarps;
        const float2 p = in ? s_part[phase][threadIdx.x % 32] : make_float2(0.f, 0.f);
        const float n = in ? s_count[threadIdx.x % 32] : 0.f;
        mean = __fmul_rn(warp_sum(p.x * n), inv_width);
        const float d = p.x - mean;
        m2 = warp_sum(fmaf(n * d, d, p.y));
      }
    }
    const float rstd = rsqrtf(m2 * inv_width + eps);
    if (lane == 0 && live) {
      if (mean_out) mean_out[r] = mean;
      if (rstd_out) rstd_out[r] = rstd;
    }
    const Two m = two(mean), scale = two(rstd);
#pragma unroll
    for (int q = 0; q < kPairs; ++q) xv[q] = mul2(sub2(xv[q], m), scale);  // unit
    if (live) {
      store_row<T, VEC, G, NV>(y + r * width, lane, width, [&](int q) { return fma2(xv[q], w.pair(q, lane), b.pair(q, lane)); });
      if (codes) store_row_codes<VEC, G, NV>(codes + r * width, lane, width, [&](int q) { return xv[q]; });
    }
    if (kStream && ++slot == slots) slot = 0, parity ^= 1;
    phase ^= 1;
  };
  const int side = Shape::kSide == 1 ? 0 : int(threadIdx.x % 32) / G;
  for (int64_t r = first; r - side < rows; r += kDepth * step) {
#pragma unroll
    for (int k = 0; k < kDepth; ++k)
      if (r - side + k * step < rows) one_row(r + k * step, parts[k]);
  }
  if (kStream && failed) let_copies_land();
}

// kCodes: unit comes from the 8-bit checkpoint, x and mean are not read.  partial [gridDim.x, 2, width] (or NULL).
// A row stays in registers, as it came, between the sums and dx.
template <typename T, int VEC, int G, int NV, bool kCodes, bool kStream>
__global__ void __launch_bounds__(RowShape<T, VEC, G, NV>::kThreads, kLnBwdBlocks<G>) layer_norm_bwd_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, int64_t x_stride, const uint8_t* __restrict__ codes,
    const float* __restrict__ mean_in, const float* __restrict__ rstd_in, const void* __restrict__ weight,
    int param_type, T* __restrict__ dx, float* __restrict__ partial, int64_t rows, int width, int slots,
    const RowWaits waits) {
  typedef RowShape<T, VEC, G, NV> Shape;
  typedef typename std::conditional<kCodes, uint8_t, T>::type Kept;
  constexpr int kPairs = Shape::kPairs;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 s_part[2][32];
  __shared__ uint64_t s_full[kLnMaxSlots];
  const int lane = threadIdx.x % G;
  const uint32_t dy_bytes = uint32_t(width) * sizeof(T), kept_bytes = uint32_t(width) * sizeof(Kept);
  const uint32_t bytes = dy_bytes + kept_bytes;
  const int64_t first = int64_t(blockIdx.x) * Shape::kRows + threadIdx.x / G, step = int64_t(gridDim.x) * Shape::kRows;
  const int64_t served = rows < waits.rows_served ? rows : waits.rows_served;
  auto kept_row = [&](int64_t r) -> const Kept* {
    if constexpr (kCodes) return codes + r * width;
    else return x + r * x_stride;
  };
  auto fill = [&](int slot, int64_t r) {
    uint8_t* to = smem + slot * bytes;
    mbar_arrive_expect(&s_full[slot], bytes);
    bulk_load(to, dy + r * width, dy_bytes, &s_full[slot]);
    bulk_load(to + dy_bytes, kept_row(r), kept_bytes, &s_full[slot]);
  };
  if (kStream && threadIdx.x == 0) {
    for (int k = 0; k < slots; ++k) mbar_init(&s_full[k], 1);
    fence_mbar_init();
    for (int k = 0; k < slots && first + k * step < served; ++k) fill(k, first + k * step);
  }
  RowParams<T, VEC, G, NV> w;
  w.load(weight, param_type, 1.f, reinterpret_cast<float*>(smem + size_t(kStream ? slots : 0) * bytes), lane, width);
  Two dw[kPairs], db[kPairs];
#pragma unroll
  for (int q = 0; q < kPairs; ++q) dw[q] = db[q] = two(0.f);
  const float inv_width = 1.f / float(width);
  constexpr int kDepth = kStream || G >= 128 ? 1 : kLnDepth<T, VEC, G, NV> / 2;
  float ahead_rstd[kDepth], ahead_mean[kDepth];  // the statistics are ahead as well
  RowPart<T, VEC, G, NV> g_parts[kDepth];
  RowPart<Kept, VEC, G, NV> k_parts[kDepth];
  auto ahead = [&](int64_t r, int k) {
    if (r >= rows) return;
    ahead_rstd[k] = rstd_in[r];
    if constexpr (!kCodes) ahead_mean[k] = mean_in[r];
    if constexpr (!kStream) g_parts[k].load(dy + r * width, lane, width), k_parts[k].load(kept_row(r), lane, width);
  };
#pragma unroll
  for (int k = 0; k < kDepth; ++k) {
    ahead_rstd[k] = ahead_mean[k] = 0.f;
    if constexpr (Shape::kSide > 1) g_parts[k].load(dy, lane, 0), k_parts[k].load(kept_row(0), lane, 0);
    ahead(first + k * step, k);
  }
  __syncthreads();
  int slot = 0, parity = 0, phase = 0;
  bool failed = false;
  auto one_row = [&](int64_t r, int k) {
    const bool live = Shape::kSide == 1 || r < rows;
    const float rstd = ahead_rstd[k];
    const Two mean = two(ahead_mean[k]), scale = two(rstd);
    RowPart<T, VEC, G, NV> g_part;
    RowPart<Kept, VEC, G, NV> k_part;
    if constexpr (kStream) {
      if (!failed) failed = !mbar_wait_soon(&s_full[slot], parity, waits.limit_ns);
      g_part.load(reinterpret_cast<const T*>(smem + slot * bytes), lane, width);
      k_part.load(reinterpret_cast<const Kept*>(smem + slot * bytes + dy_bytes), lane, width);
    } else {
      g_part = g_parts[k], k_part = k_parts[k];
    }
    ahead(r + kDepth * step, k);
    if (Shape::kSide > 1 && !live) g_part.load(dy, lane, 0), k_part.load(kept_row(0), lane, 0);  // zeros add nothing
    auto unit = [&](int q) {
      const Two v = k_part.pair(q);
      if constexpr (kCodes) return v;
      else return mul2(sub2(v, mean), scale);
    };
    Two s1 = two(0.f), s2 = two(0.f);
#pragma unroll
    for (int q = 0; q < kPairs; ++q) {  // past the row's end dy is zero
      const Two u = unit(q), g = g_part.pair(q), dn = mul2(g, w.pair(q, lane));
      dw[q] = fma2(g, u, dw[q]);
      db[q] = add2(db[q], g);
      s1 = add2(s1, dn);
      s2 = fma2(dn, u, s2);
    }
    const float2 a = split(s1), c = split(s2);
    const float2 sums = group_sum<G>(failed ? __int_as_float(0x7fffffff) : a.x + a.y, c.x + c.y, s_part, phase);
    if (kStream && threadIdx.x == 0 && !failed && r + slots * step < served) fill(slot, r + slots * step);  // all have read the row
    const Two m1 = two(sums.x * inv_width), m2 = two(-(sums.y * inv_width));
    if (live) store_row<T, VEC, G, NV>(dx + r * width, lane, width, [&](int q) {
      return mul2(fma2(unit(q), m2, sub2(mul2(g_part.pair(q), w.pair(q, lane)), m1)), scale);
    });
    if (kStream && ++slot == slots) slot = 0, parity ^= 1;
    phase ^= 1;
  };
  const int side = Shape::kSide == 1 ? 0 : int(threadIdx.x % 32) / G;
  for (int64_t r = first; r - side < rows; r += kDepth * step) {
#pragma unroll
    for (int k = 0; k < kDepth; ++k)
      if (r - side + k * step < rows) one_row(r + k * step, k);
  }
  if (kStream && failed) {
    let_copies_land();
#pragma unroll
    for (int q = 0; q < kPairs; ++q) dw[q] = db[q] = two(__int_as_float(0x7fffffff));  // they hold whatever lay in the slots
  }
  if (partial == nullptr) return;
  float* mine = partial + int64_t(blockIdx.x) * 2 * width;
  if constexpr (Shape::kRows == 1) {
#pragma unroll
    for (int q = 0; q < kPairs; ++q) {
      const float2 a = split(dw[q]), c = split(db[q]);
      const int c0 = Shape::column(lane, q, 0), c1 = Shape::column(lane, q, 1);
      if (c0 < width) mine[c0] = a.x, mine[width + c0] = c.x;
      if (c1 < width) mine[c1] = a.y, mine[width + c1] = c.y;
    }
  } else {  // the block's groups in order
    __shared__ float s_cols[Shape::kRows][2][G * NV * VEC];
    const int group = threadIdx.x / G;
#pragma unroll
    for (int q = 0; q < kPairs; ++q) {
      const float2 a = split(dw[q]), c = split(db[q]);
      const int c0 = Shape::column(lane, q, 0), c1 = Shape::column(lane, q, 1);
      s_cols[group][0][c0] = a.x, s_cols[group][1][c0] = c.x;
      s_cols[group][0][c1] = a.y, s_cols[group][1][c1] = c.y;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += Shape::kThreads) {
      float a = 0.f, d = 0.f;
#pragma unroll
      for (int k = 0; k < Shape::kRows; ++k) a += s_cols[k][0][c], d += s_cols[k][1][c];
      mine[c] = a, mine[width + c] = d;
    }
  }
}

// Column sums of partial [blocks, 2, width] in block order, FP64: 32 columns a block, a warp per run of blocks, so that few
// additions wait for one another (32,768 x 4,096 bf16: the backward 156.5 us with eight runs, 153.5 with 32).
constexpr int kLnRuns = 32;
__global__ void __launch_bounds__(32 * kLnRuns) layer_norm_param_grad_kernel(const float* __restrict__ partial, int blocks,
                                                                             int width, void* __restrict__ dw,
                                                                             void* __restrict__ db, int param_type) {
  __shared__ double s[kLnRuns][32];
  const int column = threadIdx.x & 31, run = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + column;
  void* out = blockIdx.y ? db : dw;
  if (out == nullptr) return;  // uniform over the block
  const int per = (blocks + kLnRuns - 1) / kLnRuns, lo = run * per, hi = min(lo + per, blocks);
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
    for (int k = 1; k < kLnRuns; ++k) sum += s[k][column];
    store_param(out, param_type, c, float(sum));
  }
}

// ---- rows too wide for one block (16-bit: over 16,384 columns; FP32: over 13,440 forward, 10,752 backward, whose parameters
// and two rows in flight no longer fit the shared memory): the row is read again for every pass, from L2 (4,096 x 20,000
// bf16: forward 183 us, backward 462).
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
      if (codes) store_codes(codes + r * width + c, unit);
    }
  }
}
template <typename T>
__device__ __forceinline__ float wide_unit(const T* x_row, const uint8_t* code_row, int c, float mean, float rstd) {
  if (code_row == nullptr) return (to_float(x_row[c]) - mean) * rstd;
  return code_value(code_row[c]);
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
  int grid, slots;     // slots > 0: the rows are streamed
};

// vec: elements per access, 16 bytes where every row starts on a 16-byte boundary, else one.  The smallest group
// of threads that holds a row in at most 16 elements a thread where accesses are wide, 8 (at last 16) where they are
// not (8 elements in a part of a warp).  A row of wide accesses that takes a whole block is streamed (kept_size: bytes an element of what the backward
// reads besides dy, 0 for the forward): as many rows in flight as 160 KB an SM hold, two to eight.
LnPlan ln_plan(int64_t rows, int width, int type, bool aligned, int kept_size) {
  const int size = type == kTypeFp32 ? 4 : 2;
  LnPlan p{aligned ? 16 / size : 1, 0, 0, 0, 0};
  static const int groups[] = {8, 16, 32, 128, 256, 512, 1024};
  for (int g : groups) {
    const int most = p.vec == 1 ? (g == 1024 ? 16 : 8) : (g < 32 ? 8 : p.vec == 8 && g == 512 ? 32 : 16) / p.vec;
    if (g * p.vec * most < width) continue;
    p.group = g;
    p.nv = p.vec == 1 ? 2 : 1;
    while (g * p.vec * p.nv < width) p.nv *= 2;
    break;
  }
  int blocks = p.group == 0 || p.group == 256 ? 2 : p.group <= 128 ? kLnBwdBlocks<128> : 1;
  if (kept_size == 0 && p.group > 0)
    blocks = p.group <= 32 ? kLnFwdBlocks<32> : p.group == 128 ? kLnFwdBlocks<128> : p.group == 256 ? kLnFwdBlocks<256> : 1;
  if (p.vec > 1 && p.group >= 128 && (kept_size != 1 || width % 16 == 0)) {  // bulk copies move multiples of 16 bytes
    const bool shared = p.group == 1024 || p.vec * p.nv == 32;
    const int64_t bytes = int64_t(width) * (size + kept_size), params = shared ? width * (kept_size ? 4 : 8) : 0;
    const int64_t fit = ((shared ? 210 << 10 : 160 << 10) - params) / (blocks * bytes);
    p.slots = int(fit > kLnMaxSlots ? kLnMaxSlots : fit);
    if (p.slots < 2) p.group = p.slots = 0, blocks = 2;
  }
  const int64_t most_blocks = p.group && p.group <= 32 ? (rows * p.group + 127) / 128 : rows;
  p.grid = int(most_blocks < kLnSms * blocks ? most_blocks : kLnSms * blocks);
  return p;
}

template <typename T, int VEC, int G, int NV>
int ln_fwd(const LnPlan& p, const void* x, int64_t xs, const void* w, const void* b, int pt, void* y, float* mean,
           float* rstd, uint8_t* codes, int64_t rows, int width, float eps, cudaStream_t s) {
  const size_t smem = size_t(p.slots) * width * sizeof(T) + (kLnParamsShared<VEC, G, NV> ? size_t(width) * 8 : 0);
  if (smem > 40 << 10)  // with the static part it may pass the 48 KB a launch has without asking
    if (int rc = want_smem(layer_norm_fwd_kernel<T, VEC, G, NV>, smem, "layer_norm_fwd")) return rc;
  layer_norm_fwd_kernel<T, VEC, G, NV><<<p.grid, RowShape<T, VEC, G, NV>::kThreads, smem, s>>>(
      static_cast<const T*>(x), xs, w, b, pt, static_cast<T*>(y), mean, rstd, codes, rows, width, eps, p.slots,
      row_waits());
  return launched("layer_norm_fwd");
}
template <typename T, int VEC, int G, int NV, bool kCodes, bool kStream>
int ln_bwd_of(const LnPlan& p, const void* dy, const void* x, int64_t xs, const uint8_t* codes, const float* mean,
              const float* rstd, const void* w, int pt, void* dx, float* partial, int64_t rows, int width, cudaStream_t s) {
  const size_t row = size_t(width) * (sizeof(T) + (kCodes ? 1 : sizeof(T)));
  const size_t smem = p.slots * row + (kLnParamsShared<VEC, G, NV> ? size_t(width) * 4 : 0);
  if (smem > 40 << 10)
    if (int rc = want_smem(layer_norm_bwd_kernel<T, VEC, G, NV, kCodes, kStream>, smem, "layer_norm_bwd")) return rc;
  layer_norm_bwd_kernel<T, VEC, G, NV, kCodes, kStream><<<p.grid, RowShape<T, VEC, G, NV>::kThreads, smem, s>>>(
      static_cast<const T*>(dy), static_cast<const T*>(x), xs, codes, mean, rstd, w, pt, static_cast<T*>(dx), partial, rows,
      width, p.slots, row_waits());
  return launched("layer_norm_bwd");
}
template <typename T, int VEC, int G, int NV>
int ln_bwd(const LnPlan& p, const void* dy, const void* x, int64_t xs, const uint8_t* codes, const float* mean,
           const float* rstd, const void* w, int pt, void* dx, float* partial, int64_t rows, int width,
           cudaStream_t s) {
#define MEK_LN_OF(CODES, STREAM) \
  ln_bwd_of<T, VEC, G, NV, CODES, STREAM>(p, dy, x, xs, codes, mean, rstd, w, pt, dx, partial, rows, width, s)
  constexpr bool kStream = kLnStreams<VEC, G>;
  if (!codes) return MEK_LN_OF(false, kStream);
  if (kStream && p.slots == 0) return MEK_LN_OF(true, false);  // rows of codes that bulk copies cannot move
  return MEK_LN_OF(true, kStream);
#undef MEK_LN_OF
}

// One case per (group, vectors a thread) the plan can give for VEC.
#define MEK_LN_SHAPES(T, VEC, CALL)                                                          \
  do {                                                                                       \
    if constexpr (VEC == 1) {                                                                \
      if (p.group == 8 && p.nv == 2) return CALL(T, 1, 8, 2);                                \
      if (p.group == 8 && p.nv == 4) return CALL(T, 1, 8, 4);                                \
      if (p.group == 8 && p.nv == 8) return CALL(T, 1, 8, 8);                                \
      if (p.group == 16 && p.nv == 8) return CALL(T, 1, 16, 8);                              \
      if (p.group == 32 && p.nv == 8) return CALL(T, 1, 32, 8);                              \
      if (p.group == 128 && p.nv == 4) return CALL(T, 1, 128, 4);                            \
      if (p.group == 128 && p.nv == 8) return CALL(T, 1, 128, 8);                            \
      if (p.group == 256 && p.nv == 8) return CALL(T, 1, 256, 8);                            \
      if (p.group == 512 && p.nv == 8) return CALL(T, 1, 512, 8);                            \
      if (p.group == 1024 && p.nv == 8) return CALL(T, 1, 1024, 8);                          \
      if (p.group == 1024 && p.nv == 16) return CALL(T, 1, 1024, 16);                        \
    } else {                                                                                 \
      constexpr int kMost = 16 / VEC;                                                        \
      if (p.group == 8 && p.nv == 1) return CALL(T, VEC, 8, 1);                              \
      if (p.group == 32 && p.nv == 2) return CALL(T, VEC, 32, 2);                            \
      if (p.group == 128 && p.nv == 2) return CALL(T, VEC, 128, 2);                          \
      if constexpr (VEC == 4) {                                                              \
        if (p.group == 8 && p.nv == 2) return CALL(T, VEC, 8, 2);                            \
        if (p.group == 16 && p.nv == 2) return CALL(T, VEC, 16, 2);                          \
        if (p.group == 32 && p.nv == 4) return CALL(T, VEC, 32, 4);                          \
        if (p.group == 128 && p.nv == 4) return CALL(T, VEC, 128, 4);                        \
      } else {                                                                               \
        if (p.group == 16 && p.nv == 1) return CALL(T, VEC, 16, 1);                          \
        if (p.group == 32 && p.nv == 1) return CALL(T, VEC, 32, 1);                          \
        if (p.group == 128 && p.nv == 1) return CALL(T, VEC, 128, 1);                        \
      }                                                                                      \
      if (p.group == 256 && p.nv == kMost) return CALL(T, VEC, 256, kMost);                  \
      if (p.group == 512 && p.nv == kMost) return CALL(T, VEC, 512, kMost);                  \
      if constexpr (VEC == 4) {                                                              \
        if (p.group == 1024 && p.nv == 4) return CALL(T, VEC, 1024, 4);                      \
      } else {                                                                               \
        if (p.group == 512 && p.nv == 4) return CALL(T, VEC, 512, 4);                        \
      }                                                                                      \
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
  int most = 0;
  for (int kept : {1, type == kTypeFp32 ? 4 : 2})
    for (bool aligned : {false, true}) {
      const LnPlan p = ln_plan(rows, int(width), type, aligned, kept);
      if (p.grid > most) most = p.grid;
    }
  return most;
}

int mek_layer_norm_fwd(const void* x, int type, const void* weight, const void* bias, int param_type, void* y,
                       float* mean, float* rstd, uint8_t* codes, int64_t rows, int64_t width, int64_t x_row_stride,
                       float eps, void* stream) {
  if (!x || !y) return fail(MEK_ERR_INVALID, "layer_norm_fwd: a null pointer");
  if (int rc = check_ln("layer_norm_fwd", type, param_type, rows, width, x_row_stride)) return rc;
  if (codes && width > 200704)
    return fail(MEK_ERR_UNSUPPORTED, "layer_norm_fwd: the 8-bit checkpoint holds rows of up to 200,704 columns");
  const LnPlan p = ln_plan(rows, int(width), type, ln_aligned(type, width, x_row_stride, x, y, nullptr) &&
                                                       reinterpret_cast<uintptr_t>(codes) % 8 == 0, 0);
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
                                          reinterpret_cast<uintptr_t>(codes) % 16 == 0,
              codes ? 1 : type == kTypeFp32 ? 4 : 2);
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
    layer_norm_param_grad_kernel<<<dim3((w + 31) / 32, 2), 32 * kLnRuns, 0, s>>>(partial, p.grid, w, dw, db, param_type);
    return launched("layer_norm_bwd (parameters)");
  }
  return MEK_OK;
}

}  // extern "C"

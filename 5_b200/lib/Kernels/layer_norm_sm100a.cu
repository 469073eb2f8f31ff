// Layer norm over the rows of a matrix, forward and backward, for sm_100a.
//
//   mean_r = sum_c x / C,  rstd_r = 1 / sqrt(sum_c (x - mean_r)^2 / C + eps),  n = (x - mean_r) rstd_r
//   forward:   y = n w + b                                  (w, b: one value per column, each optional)
//   backward:  a = dy w
//              dx = rstd_r (a - sum_c a / C - n sum_c (a n) / C)
//              dw = sum_r dy n,   db = sum_r dy
//
// All sums are float32; the variance is taken of the differences from the mean, which a row held in
// registers makes free and which does not cancel when the mean is large. One rounding on each store.
//
// Both kernels are bound by HBM: forward reads x and writes y, backward reads x and dy and writes dx,
// and a row is read once because its values stay in the registers of the threads that loaded them
// between the reduction and the store. A row belongs to one warp when 32 lanes hold it, to one CTA
// otherwise.
//
// The backward kernel is persistent: a CTA walks the rows blockIdx.x, blockIdx.x + gridDim.x, ... with
// every thread keeping the same columns, so that the sums over rows, dw and db, build up in registers;
// a CTA then writes one row of partial sums and a second kernel adds those rows in their order. No
// atomics: the result does not depend on which CTA runs when.
//
// Rows that are too long for the registers of a CTA are walked several times (the later walks mostly
// hit the L2); dw and db then come from a kernel of their own that walks columns.
//
// Large matrices go through persistent kernels whose rows arrive in shared memory by bulk copies some rows
// ahead (below). Measured: 16384 x 4096 bfloat16 forward 54.5 us (4.9 TB/s), backward 115 us (3.5 TB/s); 4000 x
// 8192 float32 49.4 us (5.3 TB/s) and 91 us (4.3 TB/s). What holds the 16-bit ones back is no longer memory
// but arithmetic and its latency (0.6 instructions a cycle and scheduler with four warps, the registers being
// full), which is why the sums and the scaling work on pairs of floats in one instruction.
#include "device_checks.cuh"
#include "gemm_launch.h"
#include "sm100_ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace hc {
namespace sm100 {

namespace norm {

constexpr int kMaxThreads = 1024;
constexpr int kWarpRowWarps = 8;  // warps of a CTA whose warps own a row each

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// kVec consecutive elements as they lie in memory (one access of up to 16 bytes).
template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) Pack {
  T v[kVec];
};

template <typename T, int kVec>
__device__ __forceinline__ Pack<T, kVec> zero_pack() {
  Pack<T, kVec> p;
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    p.v[i] = from_float<T>(0.0f);
  return p;
}

// Elements [c, c + kVec) of a row of `cols`; those past its end are zero. `row + c` is aligned for a
// Pack when kVec > 1 (the launcher takes kVec = 1 otherwise).
template <typename T, int kVec>
__device__ __forceinline__ Pack<T, kVec> load_pack(const T *row, long long c, long long cols) {
  if (c + kVec <= cols)
    return *reinterpret_cast<const Pack<T, kVec> *>(row + c);
  Pack<T, kVec> p = zero_pack<T, kVec>();
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    if (c + i < cols)
      p.v[i] = row[c + i];
  return p;
}

template <typename T, int kVec>
__device__ __forceinline__ void store_pack(T *row, long long c, long long cols, const Pack<T, kVec> &p) {
  if (c + kVec <= cols) {
    *reinterpret_cast<Pack<T, kVec> *>(row + c) = p;
    return;
  }
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    if (c + i < cols)
      row[c + i] = p.v[i];
}

// kVec values of a weight or bias vector as floats; `fallback` where there is none (null) or past the
// end. The vectors need not be aligned like the rows: they are read element by element if not.
template <typename P, int kVec>
__device__ __forceinline__ void load_params(float (&out)[kVec], const P *p, long long c, long long cols, bool aligned,
                                            float fallback) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      out[i] = fallback;
    return;
  }
  if (aligned && c + kVec <= cols) {
    constexpr int kPiece = sizeof(P) * kVec > 16 ? 16 / static_cast<int>(sizeof(P)) : kVec;
#pragma unroll
    for (int j = 0; j < kVec; j += kPiece) {
      const Pack<P, kPiece> v = *reinterpret_cast<const Pack<P, kPiece> *>(p + c + j);
#pragma unroll
      for (int i = 0; i < kPiece; ++i)
        out[j + i] = to_float(v.v[i]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    out[i] = c + i < cols ? to_float(p[c + i]) : fallback;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the threads that own a row: a warp, or the whole CTA through `shared` (32 floats; a second
// call needs another array or a barrier in between).
template <bool kWarpRow>
__device__ __forceinline__ float row_sum(float v, float *shared) {
  v = warp_sum(v);
  if (kWarpRow)
    return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (blockDim.x + 31) >> 5;
  if (lane == 0)
    shared[warp] = v;
  __syncthreads();
  if (warps <= 8) {  // (the same for the whole CTA)
    v = lane < warps ? shared[lane] : 0.0f;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1)
      v += __shfl_xor_sync(0xffffffffu, v, o);
    return __shfl_sync(0xffffffffu, v, 0);
  }
  return warp_sum(lane < warps ? shared[lane] : 0.0f);
}

struct Forward {
  const void *x, *weight, *bias;
  void *y;
  float *mean, *rstd;
  long long rows, cols, ldx, ldy;
  float eps;
  int params_aligned;
};

// ---------------------------------------------------------------- forward -----------

template <typename T, typename P, int kVec, int kPacks, bool kWarpRow>
__global__ void __launch_bounds__(kWarpRow ? 32 * kWarpRowWarps : kMaxThreads)
layer_norm_kernel(const Forward f) {
  __shared__ float sums[2][32];
  const int step = kWarpRow ? 32 : blockDim.x;
  const int t = kWarpRow ? (threadIdx.x & 31) : threadIdx.x;
  const long long r = kWarpRow ? static_cast<long long>(blockIdx.x) * kWarpRowWarps + (threadIdx.x >> 5) : blockIdx.x;
  if (kWarpRow && r >= f.rows)
    return;
  const long long cols = f.cols;
  const T *x = static_cast<const T *>(f.x) + r * f.ldx;
  float v[kPacks][kVec];
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < kPacks; ++j) {
    const Pack<T, kVec> p = load_pack<T, kVec>(x, static_cast<long long>(t + j * step) * kVec, cols);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      v[j][i] = to_float(p.v[i]);
      sum += v[j][i];
    }
  }
  const float inv = 1.0f / static_cast<float>(cols);
  const float mean = row_sum<kWarpRow>(sum, sums[0]) * inv;
  float square = 0.0f;
#pragma unroll
  for (int j = 0; j < kPacks; ++j) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      v[j][i] -= mean;
      if (static_cast<long long>(t + j * step) * kVec + i < cols)
        square = fmaf(v[j][i], v[j][i], square);
    }
  }
  const float rstd = rsqrtf(row_sum<kWarpRow>(square, sums[1]) * inv + f.eps);
  T *y = static_cast<T *>(f.y) + r * f.ldy;
#pragma unroll
  for (int j = 0; j < kPacks; ++j) {
    const long long c = static_cast<long long>(t + j * step) * kVec;
    if (c >= cols)
      break;
    float w[kVec], b[kVec];
    load_params<P, kVec>(w, static_cast<const P *>(f.weight), c, cols, f.params_aligned != 0, 1.0f);
    load_params<P, kVec>(b, static_cast<const P *>(f.bias), c, cols, f.params_aligned != 0, 0.0f);
    Pack<T, kVec> out;
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      out.v[i] = from_float<T>(fmaf(v[j][i] * rstd, w[i], b[i]));
    store_pack<T, kVec>(y, c, cols, out);
  }
  if (t == 0) {
    if (f.mean != nullptr)
      f.mean[r] = mean;
    if (f.rstd != nullptr)
      f.rstd[r] = rstd;
  }
}

// Rows too long for a CTA's registers: three walks over the row.
template <typename T, typename P, int kVec>
__global__ void __launch_bounds__(kMaxThreads)
layer_norm_long_kernel(const Forward f) {
  __shared__ float sums[2][32];
  const long long r = blockIdx.x, cols = f.cols;
  const T *x = static_cast<const T *>(f.x) + r * f.ldx;
  T *y = static_cast<T *>(f.y) + r * f.ldy;
  const long long step = static_cast<long long>(blockDim.x) * kVec, first = static_cast<long long>(threadIdx.x) * kVec;
  float sum = 0.0f;
  for (long long c = first; c < cols; c += step) {
    const Pack<T, kVec> p = load_pack<T, kVec>(x, c, cols);
    float part = 0.0f;
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      part += to_float(p.v[i]);
    sum += part;
  }
  const float inv = 1.0f / static_cast<float>(cols);
  const float mean = row_sum<false>(sum, sums[0]) * inv;
  float square = 0.0f;
  for (long long c = first; c < cols; c += step) {
    const Pack<T, kVec> p = load_pack<T, kVec>(x, c, cols);
    float part = 0.0f;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const float d = to_float(p.v[i]) - mean;
      if (c + i < cols)
        part = fmaf(d, d, part);
    }
    square += part;
  }
  const float rstd = rsqrtf(row_sum<false>(square, sums[1]) * inv + f.eps);
  for (long long c = first; c < cols; c += step) {
    const Pack<T, kVec> p = load_pack<T, kVec>(x, c, cols);
    float w[kVec], b[kVec];
    load_params<P, kVec>(w, static_cast<const P *>(f.weight), c, cols, f.params_aligned != 0, 1.0f);
    load_params<P, kVec>(b, static_cast<const P *>(f.bias), c, cols, f.params_aligned != 0, 0.0f);
    Pack<T, kVec> out;
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      out.v[i] = from_float<T>(fmaf((to_float(p.v[i]) - mean) * rstd, w[i], b[i]));
    store_pack<T, kVec>(y, c, cols, out);
  }
  if (threadIdx.x == 0) {
    if (f.mean != nullptr)
      f.mean[r] = mean;
    if (f.rstd != nullptr)
      f.rstd[r] = rstd;
  }
}

// ---------------------------------------------------------------- backward ----------

struct Backward {
  const void *dy, *x, *weight;
  const float *mean, *rstd;
  void *dx;
  float *partials;  // [gridDim.x][2][cols]: dw, then db; null when neither is wanted
  long long rows, cols, lddy, ldx, lddx;
  int params_aligned;
};

// Sums over the threads that own a row, two values at once.
template <bool kWarpRow>
__device__ __forceinline__ float2 row_sum2(float a, float b, float2 *shared) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (kWarpRow)
    return make_float2(a, b);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (blockDim.x + 31) >> 5;
  if (lane == 0)
    shared[warp] = make_float2(a, b);
  __syncthreads();
  const float2 s = lane < warps ? shared[lane] : make_float2(0.0f, 0.0f);
  a = s.x, b = s.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  return make_float2(a, b);
}

template <typename T, typename P, int kVec, int kPacks, bool kWarpRow, int kThreads>
__global__ void __launch_bounds__(kThreads)
layer_norm_backward_kernel(const Backward g) {
  __shared__ float2 sums[2][32];
  extern __shared__ float columns[];  // warp rows only: [warps][2][cols]
  const int step = kWarpRow ? 32 : blockDim.x;
  const int t = kWarpRow ? (threadIdx.x & 31) : threadIdx.x;
  const int worker = kWarpRow ? threadIdx.x >> 5 : 0, workers = kWarpRow ? kThreads / 32 : 1;
  const long long cols = g.cols;
  float dw[kPacks][kVec], db[kPacks][kVec];
#pragma unroll
  for (int j = 0; j < kPacks; ++j)
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      dw[j][i] = db[j][i] = 0.0f;
  const float inv = 1.0f / static_cast<float>(cols);
  const long long stride = static_cast<long long>(gridDim.x) * workers;
  int turn = 0;
  for (long long r = static_cast<long long>(blockIdx.x) * workers + worker; r < g.rows; r += stride, turn ^= 1) {
    const T *x = static_cast<const T *>(g.x) + r * g.ldx;
    const T *dy = static_cast<const T *>(g.dy) + r * g.lddy;
    Pack<T, kVec> px[kPacks], pd[kPacks];
#pragma unroll
    for (int j = 0; j < kPacks; ++j) {
      const long long c = static_cast<long long>(t + j * step) * kVec;
      px[j] = load_pack<T, kVec>(x, c, cols);
      pd[j] = load_pack<T, kVec>(dy, c, cols);
    }
    const float mean = g.mean[r], rstd = g.rstd[r];
    float s = 0.0f, sn = 0.0f;
#pragma unroll
    for (int j = 0; j < kPacks; ++j) {
      const long long c = static_cast<long long>(t + j * step) * kVec;
      if (c >= cols)  // (a row is whole packs; what lies past it is no 0 here: -mean * rstd may be infinite)
        break;
      float w[kVec];
      load_params<P, kVec>(w, static_cast<const P *>(g.weight), c, cols, g.params_aligned != 0, 1.0f);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float n = (to_float(px[j].v[i]) - mean) * rstd, d = to_float(pd[j].v[i]);
        const float a = d * w[i];
        s += a;
        sn = fmaf(a, n, sn);
        dw[j][i] = fmaf(d, n, dw[j][i]);
        db[j][i] += d;
      }
    }
    const float2 total = row_sum2<kWarpRow>(s, sn, sums[turn]);
    const float ms = total.x * inv, msn = total.y * inv;
    T *dx = static_cast<T *>(g.dx) + r * g.lddx;
#pragma unroll
    for (int j = 0; j < kPacks; ++j) {
      const long long c = static_cast<long long>(t + j * step) * kVec;
      if (c >= cols)
        break;
      float w[kVec];
      load_params<P, kVec>(w, static_cast<const P *>(g.weight), c, cols, g.params_aligned != 0, 1.0f);
      Pack<T, kVec> out;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float n = (to_float(px[j].v[i]) - mean) * rstd;
        out.v[i] = from_float<T>((fmaf(to_float(pd[j].v[i]), w[i], -ms) - n * msn) * rstd);
      }
      store_pack<T, kVec>(dx, c, cols, out);
    }
  }
  if (g.partials == nullptr)
    return;
  float *mine = g.partials + static_cast<long long>(blockIdx.x) * 2 * cols;
  if constexpr (!kWarpRow) {
#pragma unroll
    for (int j = 0; j < kPacks; ++j) {
      const long long c = static_cast<long long>(t + j * step) * kVec;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        if (c + i < cols) {
          mine[c + i] = dw[j][i];
          mine[cols + c + i] = db[j][i];
        }
      }
    }
  } else {
    // The warps of the CTA meet in shared memory and are added in their order.
#pragma unroll
    for (int j = 0; j < kPacks; ++j) {
      const int c = (t + j * step) * kVec;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        if (c + i < cols) {
          columns[worker * 2 * cols + c + i] = dw[j][i];
          columns[worker * 2 * cols + cols + c + i] = db[j][i];
        }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * cols; c += kThreads) {
      float sum = 0.0f;
      for (int k = 0; k < workers; ++k)
        sum += columns[k * 2 * cols + c];
      mine[c] = sum;
    }
  }
}

// Rows too long for a CTA's registers: dx in two walks over the row ...
template <typename T, typename P, int kVec>
__global__ void __launch_bounds__(kMaxThreads)
layer_norm_backward_long_kernel(const Backward g) {
  __shared__ float2 sums[32];
  const long long r = blockIdx.x, cols = g.cols;
  const T *x = static_cast<const T *>(g.x) + r * g.ldx;
  const T *dy = static_cast<const T *>(g.dy) + r * g.lddy;
  T *dx = static_cast<T *>(g.dx) + r * g.lddx;
  const float mean = g.mean[r], rstd = g.rstd[r], inv = 1.0f / static_cast<float>(cols);
  const long long step = static_cast<long long>(blockDim.x) * kVec, first = static_cast<long long>(threadIdx.x) * kVec;
  float s = 0.0f, sn = 0.0f;
  for (long long c = first; c < cols; c += step) {
    const Pack<T, kVec> px = load_pack<T, kVec>(x, c, cols), pd = load_pack<T, kVec>(dy, c, cols);
    float w[kVec], part = 0.0f, part_n = 0.0f;
    load_params<P, kVec>(w, static_cast<const P *>(g.weight), c, cols, g.params_aligned != 0, 1.0f);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const float a = to_float(pd.v[i]) * w[i];
      part += a;
      part_n = fmaf(a, (to_float(px.v[i]) - mean) * rstd, part_n);
    }
    s += part;
    sn += part_n;
  }
  const float2 total = row_sum2<false>(s, sn, sums);
  const float ms = total.x * inv, msn = total.y * inv;
  for (long long c = first; c < cols; c += step) {
    const Pack<T, kVec> px = load_pack<T, kVec>(x, c, cols), pd = load_pack<T, kVec>(dy, c, cols);
    float w[kVec];
    load_params<P, kVec>(w, static_cast<const P *>(g.weight), c, cols, g.params_aligned != 0, 1.0f);
    Pack<T, kVec> out;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const float n = (to_float(px.v[i]) - mean) * rstd;
      out.v[i] = from_float<T>((fmaf(to_float(pd.v[i]), w[i], -ms) - n * msn) * rstd);
    }
    store_pack<T, kVec>(dx, c, cols, out);
  }
}

// ... and the sums over rows by threads that keep kVec columns and walk rows blockIdx.y, + gridDim.y, ...
template <typename T, int kVec>
__global__ void __launch_bounds__(256)
layer_norm_columns_kernel(const Backward g) {
  const long long cols = g.cols, c = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) * kVec;
  if (c >= cols)
    return;
  float dw[kVec], db[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    dw[i] = db[i] = 0.0f;
#pragma unroll 4
  for (long long r = blockIdx.y; r < g.rows; r += gridDim.y) {
    const Pack<T, kVec> px = load_pack<T, kVec>(static_cast<const T *>(g.x) + r * g.ldx, c, cols);
    const Pack<T, kVec> pd = load_pack<T, kVec>(static_cast<const T *>(g.dy) + r * g.lddy, c, cols);
    const float mean = g.mean[r], rstd = g.rstd[r];
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const float d = to_float(pd.v[i]);
      dw[i] = fmaf(d, (to_float(px.v[i]) - mean) * rstd, dw[i]);
      db[i] += d;
    }
  }
  float *mine = g.partials + static_cast<long long>(blockIdx.y) * 2 * cols;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    if (c + i < cols) {
      mine[c + i] = dw[i];
      mine[cols + c + i] = db[i];
    }
  }
}

// out[c] = sum over the partial rows, in their order within each of kChains interleaved chains that are then added.
// A warp reads 32 neighbouring columns of a partial row. With 32 chains a column's sum is soon there but an SM holds
// two CTAs only; with 8 all CTAs of wide rows run at once. Backward passes with 8 and 32 chains: 16384 x 1024 bfloat16
// 46.5 and 42.6 us, x 2048 67.5 and 65.9, x 4096 120.9 and 121.0; 4000 x 6144 float16 61.6 and 61.7, x 8192 69.7 and
// 71.0; 2000 x 12288 67.8 and 69.9, 1025 x 16384 49.8 and 53.4: 8 from 8192 columns on.
template <typename P, int kChains>
__global__ void __launch_bounds__(32 * kChains)
layer_norm_partials_kernel(const float *partials, int count, long long cols, P *dweight, P *dbias) {
  __shared__ float part[kChains][33];
  constexpr int kAhead = 8;
  const int lane = threadIdx.x & 31, chain = threadIdx.x >> 5;
  const long long c = static_cast<long long>(blockIdx.x) * 32 + lane;
  const bool bias = blockIdx.y != 0;
  P *out = bias ? dbias : dweight;
  if (out == nullptr)
    return;
  float sum = 0.0f;
  if (c < cols) {
    const float *from = partials + (static_cast<long long>(chain) * 2 + (bias ? 1 : 0)) * cols + c;
    const long long step = 2LL * kChains * cols;
    int left = (count - chain + kChains - 1) / kChains;
    for (; left >= kAhead; left -= kAhead) {
      float v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        v[u] = from[u * step];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        sum += v[u];
      from += kAhead * step;
    }
    for (; left > 0; --left, from += step)
      sum += *from;
  }
  part[chain][lane] = sum;
  __syncthreads();
  if (chain == 0 && c < cols) {
    float total = 0.0f;
#pragma unroll
    for (int k = 0; k < kChains; ++k)
      total += part[k][lane];
    out[c] = from_float<P>(total);
  }
}

// ---------------------------------------------------------------- rows through a ring in shared memory ------
//
// For many rows: a CTA is persistent and its rows arrive by cp.async.bulk a few rows ahead, so that the bytes
// in flight depend neither on registers nor on how far the arithmetic has got.
//
// Rows that do not all start on 16-byte boundaries (an odd number of columns): as long as the matrices agree about
// where between two boundaries a row starts, that place is the same for every kVec-th row, and a CTA keeps to
// rows of one place (kShift). Its packs are the 16-byte pieces as they lie in memory, `lead` elements of the first
// one belonging to what precedes the row; rows are copied from the boundary below their first element to the one
// above their last, though never behind the matrix: the few elements that leaves out are stored one by one.

// How a thread's kPer elements lie: packs of kVec, a pack of every thread after another.
template <int kVec>
__device__ __forceinline__ int element_of(int t, int j, int threads) {
  return (t + j / kVec * threads) * kVec + j % kVec;
}

__device__ __forceinline__ float2 splat(float v) { return make_float2(v, v); }

// A row's copy: where it starts in memory, how many bytes come by the bulk copy.
struct RowCopy {
  uintptr_t low;
  uint32_t bytes;
  __device__ __forceinline__ RowCopy(const void *base, long long row, long long ld, long long cols, long long rows, int size) {
    const uintptr_t first = reinterpret_cast<uintptr_t>(base) + static_cast<uintptr_t>(row * ld * size);
    const uintptr_t end = reinterpret_cast<uintptr_t>(base) + static_cast<uintptr_t>(((rows - 1) * ld + cols) * size);
    low = first & ~uintptr_t{15};
    uintptr_t high = (first + static_cast<uintptr_t>(cols * size) + 15) & ~uintptr_t{15};
    if (high > end)
      high = end & ~uintptr_t{15};
    bytes = high > low ? static_cast<uint32_t>(high - low) : 0u;
  }
};

__device__ __forceinline__ void bulk_load(uint32_t dst, uintptr_t src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               :: "r"(dst), "l"(static_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
               : "memory");
}

// The rows of a CTA: those of one place, ring.step rows apart, in tiles.
struct Ring {
  int stages;
  uint32_t slot;    // bytes of one matrix's row in a stage, a multiple of 16
  int rows, parts;  // backward: rows of a tile, warps that share one (rows x parts warps in all)
  int step;         // 1, or with kShift kVec; the grid is a multiple of it
};

struct Place {
  int first;   // the first row of this CTA's place
  int lead;    // elements between the boundary and a row's start
  __device__ __forceinline__ Place(const void *base, long long ld, int size, int step) {
    first = static_cast<int>(blockIdx.x) % step;
    lead = static_cast<int>((reinterpret_cast<uintptr_t>(base) + static_cast<uintptr_t>(first * ld * size)) & 15) / size;
  }
};

// What the copy of the matrix's last row leaves out (at most 14 bytes), into the slot at `place`.
template <typename T>
__device__ __forceinline__ void store_rest(const RowCopy &copy, const T *row, long long cols, uint8_t *place) {
  const uint8_t *const low = reinterpret_cast<const uint8_t *>(copy.low);
  const int end = static_cast<int>(reinterpret_cast<const uint8_t *>(row + cols) - low);
  for (int at = max(static_cast<int>(copy.bytes), static_cast<int>(reinterpret_cast<const uint8_t *>(row) - low)); at < end;
       at += static_cast<int>(sizeof(T)))
    *reinterpret_cast<T *>(place + at) = *reinterpret_cast<const T *>(low + at);
}

// kVec elements from column c on of a row that lies in the ring at `place`, as floats; zeros beyond its ends.
template <typename T, int kVec, bool kShift>
__device__ __forceinline__ void read_unit(float2 (&out)[kVec / 2], const uint8_t *place, int c, int lead, int cols) {
  const Pack<T, kVec> p = *reinterpret_cast<const Pack<T, kVec> *>(place + (c + lead) * static_cast<int>(sizeof(T)));
  float v[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    v[i] = to_float(p.v[i]);
  if (kShift && (c < 0 || c + kVec > cols)) {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (c + i < 0 || c + i >= cols)
        v[i] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < kVec / 2; ++i)
    out[i] = make_float2(v[2 * i], v[2 * i + 1]);
}

// kVec elements to column c on of a row, nothing beyond its ends.
template <typename T, int kVec, bool kShift>
__device__ __forceinline__ void store_unit(T *row, int c, int cols, const float2 (&v)[kVec / 2]) {
  Pack<T, kVec> p;
#pragma unroll
  for (int i = 0; i < kVec / 2; ++i) {
    p.v[2 * i] = from_float<T>(v[i].x);
    p.v[2 * i + 1] = from_float<T>(v[i].y);
  }
  if (!kShift || (c >= 0 && c + kVec <= cols)) {
    *reinterpret_cast<Pack<T, kVec> *>(row + c) = p;
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (c + i >= 0 && c + i < cols)
        row[c + i] = p.v[i];
  }
}

// A thread's share of a weight or bias vector, kept for all rows as it lies in memory.
template <typename P, int kVec, int kPer>
struct Params {
  Pack<P, kVec> v[kPer / kVec];
  __device__ __forceinline__ Params(const P *p, int cols, int lead, int t, int threads, float fallback) {
#pragma unroll
    for (int q = 0; q < kPer / kVec; ++q) {
      const int c = (t + q * threads) * kVec - lead;
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        v[q].v[i] = p != nullptr && c + i >= 0 && c + i < cols ? p[c + i] : from_float<P>(fallback);
    }
  }
  __device__ __forceinline__ float operator[](int j) const { return to_float(v[j / kVec].v[j % kVec]); }
  __device__ __forceinline__ float2 pair(int j) const { return make_float2((*this)[2 * j], (*this)[2 * j + 1]); }
};

template <typename T, typename P, int kVec, int kPer, int kThreads, int kCtas, bool kShift>
__global__ void __launch_bounds__(kThreads, kCtas)
layer_norm_ring_kernel(const Forward f, const Ring ring, int *status) {
  extern __shared__ __align__(128) uint8_t shared[];
  __shared__ float sums[2][2][32];
  __shared__ uint32_t abort_word;
  volatile uint32_t *abort_flag = &abort_word;
  constexpr int kUnits = kPer / kVec, kPairs = kVec / 2;
  const int t = threadIdx.x, threads = blockDim.x, cols = static_cast<int>(f.cols);
  const uint32_t bars = smem_u32(shared), slots = bars + 128;
  const uint8_t *const slots_gen = shared + 128;
  const T *x = static_cast<const T *>(f.x);
  const Place place(x, f.ldx, sizeof(T), kShift ? ring.step : 1);
  const int lead = kShift ? place.lead : 0;
  // Rows blockIdx.x, blockIdx.x + gridDim.x, ...: all of one place, since the grid is a multiple of ring.step.
  auto load = [&](long long row, int stage) {
    const RowCopy copy(x, row, f.ldx, f.cols, f.rows, sizeof(T));
    if (!HC_CHECK(status, abort_flag, HC_CHECK_RING_STAGE, stage >= 0 && stage < ring.stages && copy.bytes <= ring.slot) ||
        !HC_CHECK(status, abort_flag, HC_CHECK_TILE_COORDINATES, row >= 0 && row < f.rows))
      return;
    if (kShift && row == f.rows - 1)
      store_rest(copy, x + row * f.ldx, f.cols, shared + 128 + stage * ring.slot);
    mbar_arrive_expect_tx(bars + 8u * stage, copy.bytes);
    if (copy.bytes != 0)
      bulk_load(slots + stage * ring.slot, copy.low, copy.bytes, bars + 8u * stage);
  };
  if (t == 0) {
    for (int s = 0; s < ring.stages; ++s)
      mbar_init(bars + 8u * s, 1);
    abort_word = 0;
    mbar_fence_init();
    for (int s = 0; s < ring.stages; ++s)
      if (blockIdx.x + static_cast<long long>(s) * gridDim.x < f.rows)
        load(blockIdx.x + static_cast<long long>(s) * gridDim.x, s);
  }
  const Params<P, kVec, kPer> weight(static_cast<const P *>(f.weight), cols, lead, t, threads, 1.0f);
  const Params<P, kVec, kPer> bias(static_cast<const P *>(f.bias), cols, lead, t, threads, 0.0f);
  __syncthreads();
  const float inv = 1.0f / static_cast<float>(cols);
  int stage = 0, turn = 0;
  uint32_t parity = 0;
  for (long long r = blockIdx.x; r < f.rows; r += gridDim.x, turn ^= 1) {
    float2 v[kUnits][kPairs];
    mbar_wait(bars + 8u * stage, parity, abort_flag);
    float2 two = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int c = element_of<kVec>(t, u * kVec, threads) - lead;
#pragma unroll
      for (int i = 0; i < kPairs; ++i)
        v[u][i] = make_float2(0.0f, 0.0f);
      if (c < cols)
        read_unit<T, kVec, kShift>(v[u], slots_gen + stage * ring.slot, c, lead, cols);
#pragma unroll
      for (int i = 0; i < kPairs; ++i)
        two = __fadd2_rn(two, v[u][i]);
    }
    fence_proxy_async_smem();  // the slot has been read before a bulk copy, another proxy's write, refills it
    const float sum = two.x + two.y;
    const float mean = row_sum<false>(sum, sums[turn][0]) * inv;
    if (t == 0 && r + static_cast<long long>(ring.stages) * gridDim.x < f.rows)
      load(r + static_cast<long long>(ring.stages) * gridDim.x, stage);  // every thread has read the slot
    if (++stage == ring.stages) {
      stage = 0;
      parity ^= 1u;
    }
    two = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int c = element_of<kVec>(t, u * kVec, threads) - lead;
      if (c < cols) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
          v[u][i] = __fadd2_rn(v[u][i], splat(-mean));
        if (kShift && (c < 0 || c + kVec > cols)) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            if (c + 2 * i < 0 || c + 2 * i >= cols)
              v[u][i].x = 0.0f;
            if (c + 2 * i + 1 < 0 || c + 2 * i + 1 >= cols)
              v[u][i].y = 0.0f;
          }
        }
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
          two = __ffma2_rn(v[u][i], v[u][i], two);
      }
    }
    const float square = two.x + two.y;
    const float rstd = rsqrtf(row_sum<false>(square, sums[turn][1]) * inv + f.eps);
    T *y = static_cast<T *>(f.y) + r * f.ldy;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int c = element_of<kVec>(t, u * kVec, threads) - lead;
      if (c < cols) {
        float2 out[kPairs];
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
          out[i] = __ffma2_rn(__fmul2_rn(v[u][i], splat(rstd)), weight.pair(u * kPairs + i), bias.pair(u * kPairs + i));
        store_unit<T, kVec, kShift>(y, c, cols, out);
      }
    }
    if (t == 0) {
      if (f.mean != nullptr)
        f.mean[r] = mean;
      if (f.rstd != nullptr)
        f.rstd[r] = rstd;
    }
  }
  __syncthreads();
  if (t == 0 && abort_word != 0)
    atomicCAS(status, 0, kStatusDeviceWaitTimeout);
}

// Backward: a stage holds a tile of ring.rows rows of x and dy, and a tile is gone through twice. First the warps
// share its rows, ring.parts warps a row, and find the two sums of each; then, with one barrier between, every
// thread takes its own kPer columns of all rows, writes dx and adds to dw and db, which stay in registers. What
// a row costs besides its elements (shuffles, barrier, addresses) is thus paid by few warps or for several
// rows at once. With kShift the weights lie in shared memory behind the ring, as far from a boundary as the rows.
template <typename T, typename P, int kVec, int kPer, int kThreads, bool kShift>
__global__ void __launch_bounds__(kThreads, 1)
layer_norm_backward_ring_kernel(const Backward g, const Ring ring, int *status) {
  extern __shared__ __align__(128) uint8_t shared[];
  __shared__ float4 sums[2][32];  // [row * parts + part]: sum a, sum a n, mean, rstd
  __shared__ uint32_t abort_word;
  volatile uint32_t *abort_flag = &abort_word;
  constexpr int kUnits = kPer / kVec, kPairs = kVec / 2;
  const int t = threadIdx.x, threads = blockDim.x, cols = static_cast<int>(g.cols), lane = t & 31, warp = t >> 5;
  const int rows = ring.rows, parts = ring.parts, step = kShift ? ring.step : 1;
  const uint32_t bars = smem_u32(shared), slots = bars + 128, stage_bytes = 2u * rows * ring.slot;
  const uint8_t *const slots_gen = shared + 128;
  const T *x = static_cast<const T *>(g.x), *dy = static_cast<const T *>(g.dy);
  const Place place(x, g.ldx, sizeof(T), step);
  const int lead = kShift ? place.lead : 0;
  const long long of_place = place.first < g.rows ? (g.rows - place.first + step - 1) / step : 0;  // rows
  const long long tiles = (of_place + rows - 1) / rows;
  const long long first_tile = blockIdx.x / step, tile_step = gridDim.x / step;
  auto row_of = [&](long long tile, int r) { return place.first + step * (tile * rows + r); };
  auto live_of = [&](long long tile) { return static_cast<int>(min(static_cast<long long>(rows), of_place - tile * rows)); };
  auto load = [&](long long tile, int stage) {
    const int live = live_of(tile);
    uint32_t total = 0;
    if (!HC_CHECK(status, abort_flag, HC_CHECK_RING_STAGE, stage >= 0 && stage < ring.stages) ||
        !HC_CHECK(status, abort_flag, HC_CHECK_TILE_COORDINATES,
                  tile >= 0 && tile < tiles && live >= 1 && live <= rows && row_of(tile, live - 1) < g.rows) ||
        !HC_CHECK(status, abort_flag, HC_CHECK_TMA_COORDINATES,
                  RowCopy(x, row_of(tile, 0), g.ldx, g.cols, g.rows, sizeof(T)).bytes <= ring.slot &&
                      RowCopy(dy, row_of(tile, 0), g.lddy, g.cols, g.rows, sizeof(T)).bytes <= ring.slot))
      return;
    if (kShift && row_of(tile, live - 1) == g.rows - 1) {
      uint8_t *const at = shared + 128 + stage * stage_bytes + 2u * (live - 1) * ring.slot;
      store_rest(RowCopy(x, g.rows - 1, g.ldx, g.cols, g.rows, sizeof(T)), x + (g.rows - 1) * g.ldx, g.cols, at);
      store_rest(RowCopy(dy, g.rows - 1, g.lddy, g.cols, g.rows, sizeof(T)), dy + (g.rows - 1) * g.lddy, g.cols, at + ring.slot);
    }
    for (int r = 0; r < live; ++r)
      total += RowCopy(x, row_of(tile, r), g.ldx, g.cols, g.rows, sizeof(T)).bytes +
               RowCopy(dy, row_of(tile, r), g.lddy, g.cols, g.rows, sizeof(T)).bytes;
    mbar_arrive_expect_tx(bars + 8u * stage, total);
    for (int r = 0; r < live; ++r) {
      const RowCopy cx(x, row_of(tile, r), g.ldx, g.cols, g.rows, sizeof(T)),
          cd(dy, row_of(tile, r), g.lddy, g.cols, g.rows, sizeof(T));
      const uint32_t at = slots + stage * stage_bytes + 2u * r * ring.slot;
      if (cx.bytes != 0)
        bulk_load(at, cx.low, cx.bytes, bars + 8u * stage);
      if (cd.bytes != 0)
        bulk_load(at + ring.slot, cd.low, cd.bytes, bars + 8u * stage);
    }
  };
  if (t == 0) {
    for (int s = 0; s < ring.stages; ++s)
      mbar_init(bars + 8u * s, 1);
    abort_word = 0;
    mbar_fence_init();
    for (int s = 0; s < ring.stages; ++s)
      if (first_tile + s * tile_step < tiles)
        load(first_tile + s * tile_step, s);
  }
  const P *const w = static_cast<const P *>(g.weight);
  P *const shifted = reinterpret_cast<P *>(shared + 128 + ring.stages * stage_bytes);
  if constexpr (kShift) {
    const int all = (lead + cols + kVec - 1) / kVec * kVec;
    for (int i = t; i < all; i += threads)
      shifted[i] = w != nullptr && i >= lead && i - lead < cols ? w[i - lead] : from_float<P>(1.0f);
    __syncthreads();
  }
  auto weights = [&](float2 (&out)[kPairs], int c) {
    float v[kVec];
    if constexpr (kShift) {
      const Pack<P, kVec> p = *reinterpret_cast<const Pack<P, kVec> *>(shifted + c + lead);
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        v[i] = to_float(p.v[i]);
    } else {
      load_params<P, kVec>(v, w, c, cols, g.params_aligned != 0, 1.0f);
    }
#pragma unroll
    for (int i = 0; i < kPairs; ++i)
      out[i] = make_float2(v[2 * i], v[2 * i + 1]);
  };
  constexpr bool kKeep = kPer <= 16;  // the weights stay in registers between the rows (else dw and db fill them)
  float2 dw[kUnits][kPairs], db[kUnits][kPairs], weight[kKeep ? kUnits : 1][kPairs];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int c = element_of<kVec>(t, u * kVec, threads) - lead;
#pragma unroll
    for (int i = 0; i < kPairs; ++i)
      dw[u][i] = db[u][i] = make_float2(0.0f, 0.0f);
    if (kKeep && c < cols)
      weights(weight[kKeep ? u : 0], c);
  }
  __syncthreads();
  const float inv = 1.0f / static_cast<float>(cols);
  const int my_row = warp / parts, my_part = warp - my_row * parts;
  float next_mean = 0.0f, next_rstd = 0.0f;  // of this warp's row of the tile to come
  auto fetch_statistics = [&](long long tile) {
    const long long r = row_of(tile, my_row);
    if (r < g.rows) {
      next_mean = g.mean[r];
      next_rstd = g.rstd[r];
    }
  };
  fetch_statistics(first_tile);
  int stage = 0, turn = 0, before = 0;
  uint32_t parity = 0;
  for (long long tile = first_tile; tile < tiles; tile += tile_step, turn ^= 1) {
    const int live = live_of(tile);
    const uint8_t *const tile_at = slots_gen + stage * stage_bytes;
    auto unit = [&](float2 (&out)[kPairs], int r, int which, int c) {
      read_unit<T, kVec, kShift>(out, tile_at + (2u * r + which) * ring.slot, c, lead, cols);
    };
    const float mean = next_mean, rstd = next_rstd;
    fetch_statistics(tile + tile_step);
    mbar_wait(bars + 8u * stage, parity, abort_flag);
    if (my_row < live) {
      // sum of a, and of a (x - mean): rstd is multiplied in once at the end.
      float2 s = make_float2(0.0f, 0.0f), sn = s;
      const float2 minus = splat(-mean);
#pragma unroll 4
      for (int c = (my_part * 32 + lane) * kVec - lead; c < cols; c += parts * 32 * kVec) {
        float2 vx[kPairs], vd[kPairs], vw[kPairs];
        unit(vx, my_row, 0, c);
        unit(vd, my_row, 1, c);
        weights(vw, c);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const float2 a = __fmul2_rn(vd[i], vw[i]);
          s = __fadd2_rn(s, a);
          sn = __ffma2_rn(a, __fadd2_rn(vx[i], minus), sn);
        }
      }
      const float s1 = warp_sum(s.x + s.y), sn1 = warp_sum(sn.x + sn.y) * rstd;
      if (lane == 0)
        sums[turn][warp] = make_float4(s1, sn1, mean, rstd);
    }
    __syncthreads();
    // Every thread is through with the tile before: its stage takes another.
    const long long next = tile + (ring.stages - 1) * tile_step;
    if (t == 0 && tile != first_tile && next < tiles)
      load(next, before);
    for (int r = 0; r < live; ++r) {
      float4 total = sums[turn][r * parts];
      if (parts <= 4) {
        for (int k = 1; k < parts; ++k) {
          total.x += sums[turn][r * parts + k].x;
          total.y += sums[turn][r * parts + k].y;
        }
      } else {
        const float4 v = lane < parts ? sums[turn][r * parts + lane] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        total.x = warp_sum(v.x);
        total.y = warp_sum(v.y);
      }
      const float2 minus_ms = splat(-total.x * inv), minus_msn = splat(-total.y * inv), minus_mean = splat(-total.z),
                   rs = splat(total.w);
      T *dx = static_cast<T *>(g.dx) + row_of(tile, r) * g.lddx;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int c = element_of<kVec>(t, u * kVec, threads) - lead;
        if (c < cols) {
          float2 vx[kPairs], vd[kPairs], vw[kPairs], out[kPairs];
          unit(vx, r, 0, c);
          unit(vd, r, 1, c);
          if constexpr (!kKeep)
            weights(vw, c);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            const float2 n = __fmul2_rn(__fadd2_rn(vx[i], minus_mean), rs), d = vd[i];
            dw[u][i] = __ffma2_rn(d, n, dw[u][i]);
            db[u][i] = __fadd2_rn(db[u][i], d);
            out[i] = __fmul2_rn(__ffma2_rn(n, minus_msn, __ffma2_rn(d, kKeep ? weight[kKeep ? u : 0][i] : vw[i], minus_ms)), rs);
          }
          store_unit<T, kVec, kShift>(dx, c, cols, out);
        }
      }
    }
    fence_proxy_async_smem();  // this thread's reads of the stage come before its refill, after the next barrier
    before = stage;
    if (++stage == ring.stages) {
      stage = 0;
      parity ^= 1u;
    }
  }
  if (g.partials != nullptr) {
    float *mine = g.partials + static_cast<long long>(blockIdx.x) * 2 * cols;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int c = element_of<kVec>(t, u * kVec, threads) - lead;
      if (!kShift && c < cols) {  // four at a time: cols is a multiple of four, and so is every row of partials
#pragma unroll
        for (int i = 0; i < kPairs; i += 2) {
          *reinterpret_cast<float4 *>(mine + c + 2 * i) = make_float4(dw[u][i].x, dw[u][i].y, dw[u][i + 1].x, dw[u][i + 1].y);
          *reinterpret_cast<float4 *>(mine + cols + c + 2 * i) = make_float4(db[u][i].x, db[u][i].y, db[u][i + 1].x, db[u][i + 1].y);
        }
      }
      if (kShift) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          if (c + 2 * i >= 0 && c + 2 * i < cols) {
            mine[c + 2 * i] = dw[u][i].x;
            mine[cols + c + 2 * i] = db[u][i].x;
          }
          if (c + 2 * i + 1 >= 0 && c + 2 * i + 1 < cols) {
            mine[c + 2 * i + 1] = dw[u][i].y;
            mine[cols + c + 2 * i + 1] = db[u][i].y;
          }
        }
      }
    }
  }
  __syncthreads();
  if (t == 0 && abort_word != 0)
    atomicCAS(status, 0, kStatusDeviceWaitTimeout);
}

// ---------------------------------------------------------------- launch ------------

// How a call is laid out; for the kernels and for the scratch they need.
struct Plan {
  enum Kind { kWarpRows, kDirect, kRing, kLong } kind;
  int threads, per;  // per: elements per thread (ring) or packs per thread (direct, warp rows)
  int grid;          // CTAs of the kernel that walks rows; of a long backward pass, the row chunks of dw and db
  Ring ring;
  size_t shared;
};

constexpr long long kMostRingCols = 16 * kMaxThreads;
constexpr int kMostStages = 8;
constexpr int kRingBytes = 200 * 1024;  // dynamic shared memory of an SM that the rings of its CTAs may take

int threads_for(long long cols, int per) { return static_cast<int>((cols + per - 1) / per + 31) / 32 * 32; }

// CTAs that share an SM: as many as its registers hold, at most eight.
int ring_ctas(int threads_per_sm, int threads) {
  const int ctas = threads_per_sm / threads;
  return ctas < 8 ? ctas : 8;
}

// How the matrices of a call lie: 16 / size where every row of every one consists of whole 16-byte pieces, kShifted
// where they agree about where between two boundaries a row starts, else 1.
constexpr int kShifted = 0;

// Forward. What a row costs besides its elements is per warp, so few warps with 32 elements a thread (and the
// registers of 512 threads) suit long rows: 16384 x 2048 bfloat16 takes 33.0 us so and 38.2 us with 8 elements
// a thread; 16384 x 1024 takes 24.9 and 22.7 us. A second warp that is mostly idle spoils it: 4095 x 1031 float32
// takes 16.4 us so, 14.4 us with 8.
bool forward_ring(Plan *plan, long long rows, long long cols, int vec, int size, int sm_count) {
  const int step = vec == kShifted ? 16 / size : 1;
  if (vec == 1 || cols + step - 1 > kMostRingCols)
    return false;
  plan->kind = Plan::kRing;
  plan->per = cols <= 1024 || (cols <= 2048 && threads_for(cols, 32) * 32 > 3 * cols / 2) ? 8 : 32;
  plan->threads = threads_for(cols + step - 1, plan->per);
  plan->ring.slot = static_cast<uint32_t>((cols * size + 15) / 16 * 16 + 16);  // a row at an odd place needs 16 more
  plan->ring.step = step;
  const int most = ring_ctas(plan->per == 8 ? 1024 : 512, plan->threads);
  const long long stages = (kRingBytes / most - 256) / plan->ring.slot;
  if (stages < 2)
    return false;
  plan->ring.stages = static_cast<int>(stages < kMostStages ? stages : kMostStages);
  plan->shared = 128 + static_cast<size_t>(plan->ring.stages) * plan->ring.slot;
  const long long ctas = static_cast<long long>(sm_count) * most / step * step;
  plan->grid = static_cast<int>(rows < ctas ? (rows + step - 1) / step * step : ctas);
  return true;
}

// Backward: 16 elements a thread up to 8192 columns (16384 x 4096 bfloat16 takes 115 us so, with 8 elements
// 143 us, with 32 elements 136 us), 32 beyond, where dw and db of 512 threads fill the registers. Tiles of as
// many rows as leave three stages and give every CTA four tiles, and warps to share them.
bool backward_ring(Plan *plan, long long rows, long long cols, int vec, int size, int param_size, int sm_count) {
  const int step = vec == kShifted ? 16 / size : 1;
  if (vec == 1 || cols + step - 1 > kMostRingCols)
    return false;
  plan->kind = Plan::kRing;
  plan->per = cols + step - 1 <= 8192 ? 16 : 32;
  plan->threads = threads_for(cols + step - 1, plan->per);
  plan->ring.slot = static_cast<uint32_t>((cols * size + 15) / 16 * 16 + 16);
  plan->ring.step = step;
  const int most = ring_ctas(512, plan->threads);
  const long long shifted = step > 1 ? (cols + 2 * step) * param_size : 0;  // the weights
  const long long budget = kRingBytes / most - 256 - shifted, pair = 2LL * plan->ring.slot;
  const int warps = plan->threads / 32;
  int tile = 1;
  while (tile < 8 && warps % (2 * tile) == 0 && 3 * 2 * tile * pair <= budget && rows >= 4LL * tile * most * sm_count)
    tile *= 2;
  const long long stages = budget / (tile * pair);
  if (stages < 2)
    return false;
  plan->ring.rows = tile;
  plan->ring.parts = warps / tile;
  plan->ring.stages = static_cast<int>(stages < kMostStages ? stages : kMostStages);
  plan->shared = 128 + static_cast<size_t>(plan->ring.stages) * tile * pair + shifted;
  const long long ctas = static_cast<long long>(sm_count) * most / step * step;
  const long long tiles = ((rows + step - 1) / step + tile - 1) / tile * step;  // of all places
  plan->grid = static_cast<int>(tiles < ctas ? tiles : ctas);
  return true;
}

Plan forward_plan(long long rows, long long cols, int vec, int size, int sm_count) {
  Plan plan{};
  const long long packs = vec > 1 ? (cols + vec - 1) / vec : cols;  // outside the ring
  // The ring pays for rows of more than 1 KiB (16384 x 512 float32: 18.7 us either way; 65536 x 512 bfloat16
  // 53 us, without it 47 us) in matrices of 4 MiB and more, which give every CTA several rows (592 x 4096
  // bfloat16: 7.5 us, without it 7.9 us; 296 x 4096: 7.6 and 6.9 us).
  // At odd places, where the other kernels take one element at a time, it pays from 256 columns on (20000 x 259
  // bfloat16: 31.0 us, without it 35.1 us; 16384 x 1503 float16 43 and 118 us, 4096 x 4095 bfloat16 32 and 55 us;
  // but 20000 x 131 float32 24.8 and 20.7 us).
  if ((vec == kShifted ? cols > 256 : cols * size > 1024) && rows * cols * size >= 4LL << 20 && forward_ring(&plan, rows, cols, vec, size, sm_count))
    return plan;
  if (packs <= 64) {  // a warp holds a row in at most two packs per lane
    plan.kind = Plan::kWarpRows;
    plan.threads = 32 * kWarpRowWarps;
    plan.per = packs <= 32 ? 1 : 2;
    plan.grid = static_cast<int>((rows + kWarpRowWarps - 1) / kWarpRowWarps);
    return plan;
  }
  plan.grid = static_cast<int>(rows);
  if (packs > 4 * kMaxThreads) {
    plan.kind = Plan::kLong;
    plan.threads = kMaxThreads;
    return plan;
  }
  // As many threads as the row has packs, for the shortest chain of loads.
  plan.kind = Plan::kDirect;
  plan.per = packs <= kMaxThreads ? 1 : packs <= 2 * kMaxThreads ? 2 : 4;
  plan.threads = static_cast<int>(((packs + plan.per - 1) / plan.per + 31) / 32 * 32);
  return plan;
}

Plan backward_plan(long long rows, long long cols, int vec, int size, int param_size, int sm_count) {
  Plan plan{};
  const long long packs = vec > 1 ? (cols + vec - 1) / vec : cols;  // outside the ring
  if (packs <= 32) {
    plan.kind = Plan::kWarpRows;
    plan.threads = 32 * kWarpRowWarps;
    const long long units = (rows + kWarpRowWarps - 1) / kWarpRowWarps;
    plan.grid = static_cast<int>(units < 4LL * sm_count ? units : 4LL * sm_count);
    plan.shared = sizeof(float) * kWarpRowWarps * 2 * static_cast<size_t>(cols);
    return plan;
  }
  // Without the ring a thread holds one pack, which float32 rows of up to 1024 columns do with few enough
  // threads: 16384 x 512 takes 41.1 us, through the ring 45.2 us, 16384 x 1024 51.6 and 53.9 us (bfloat16: 65.7
  // and 43.3 us).
  // At odd places it takes more of a start, and pays for many rows that are not short: 16384 x 1503 float16 takes
  // 80 us, without it 272 us, 2405 x 1503 bfloat16 30 and 49 us, but 200 x 16371 48 and 36 us, 2000 x 515 22 and
  // 17 us, 20000 x 75 45 and 27 us.
  const bool small = vec == kShifted && (cols * size <= 512 || rows * cols * size < 4LL << 20 || rows < 2LL * sm_count);
  if (!(vec == 4 && cols <= 1024) && !small && backward_ring(&plan, rows, cols, vec, size, param_size, sm_count))
    return plan;
  if (packs <= kMaxThreads) {
    plan.kind = Plan::kDirect;
    plan.threads = static_cast<int>((packs + 31) / 32 * 32);
    const long long ctas = static_cast<long long>(sm_count) * (plan.threads > 512 ? 1 : plan.threads > 256 ? 2 : 4);
    plan.grid = static_cast<int>(rows < ctas ? rows : ctas);
    return plan;
  }
  plan.kind = Plan::kLong;
  plan.threads = kMaxThreads;
  // Row chunks of the column kernel: enough CTAs to fill the GPU a few times over.
  const long long column_blocks = (packs + 255) / 256;
  const long long chunks = (8LL * sm_count + column_blocks - 1) / column_blocks;
  plan.grid = static_cast<int>(rows < chunks ? rows : chunks);
  return plan;
}

// The most shared memory a kernel may be launched with belongs to the kernel on its device, not to a launch: it is
// set to what the largest ring takes, always the same number, so that threads whose contexts launch one kernel with
// rings of different sizes cannot lower it for each other.
template <auto kKernel, typename... Args>
cudaError_t launch_ring(const Plan &plan, cudaStream_t stream, const Args &...args) {
  static thread_local int configured_device = -1;
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err == cudaSuccess && configured_device != device) {
    err = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes);
    if (err == cudaSuccess)
      configured_device = device;
  }
  if (err != cudaSuccess)
    return err;
  kKernel<<<plan.grid, plan.threads, plan.shared, stream>>>(args...);
  return cudaGetLastError();
}

template <typename T, typename P, int kVec>
cudaError_t launch_forward(const Forward &f, int vec, int sm_count, int *status, cudaStream_t stream) {
  const Plan plan = forward_plan(f.rows, f.cols, vec, sizeof(T), sm_count);
  constexpr bool kShift = kVec == 1;  // of the ring
  constexpr int kFull = 16 / static_cast<int>(sizeof(T));
  switch (plan.kind) {
  case Plan::kWarpRows:
    if (plan.per == 1)
      layer_norm_kernel<T, P, kVec, 1, true><<<plan.grid, plan.threads, 0, stream>>>(f);
    else
      layer_norm_kernel<T, P, kVec, 2, true><<<plan.grid, plan.threads, 0, stream>>>(f);
    break;
  case Plan::kRing:
    if (plan.per == 8)
      return launch_ring<layer_norm_ring_kernel<T, P, kFull, 8, 256, 4, kShift>>(plan, stream, f, plan.ring, status);
    return launch_ring<layer_norm_ring_kernel<T, P, kFull, 32, 512, 1, kShift>>(plan, stream, f, plan.ring, status);
  case Plan::kDirect:
    if (plan.per == 1)
      layer_norm_kernel<T, P, kVec, 1, false><<<plan.grid, plan.threads, 0, stream>>>(f);
    else if (plan.per == 2)
      layer_norm_kernel<T, P, kVec, 2, false><<<plan.grid, plan.threads, 0, stream>>>(f);
    else
      layer_norm_kernel<T, P, kVec, 4, false><<<plan.grid, plan.threads, 0, stream>>>(f);
    break;
  case Plan::kLong:
    layer_norm_long_kernel<T, P, kVec><<<plan.grid, plan.threads, 0, stream>>>(f);
    break;
  }
  return cudaGetLastError();
}

template <typename T, typename P, int kVec>
cudaError_t launch_backward(const Backward &g, P *dweight, P *dbias, int vec, int sm_count, int *status, cudaStream_t stream) {
  const Plan plan = backward_plan(g.rows, g.cols, vec, sizeof(T), sizeof(P), sm_count);
  constexpr bool kShift = kVec == 1;  // of the ring
  constexpr int kFull = 16 / static_cast<int>(sizeof(T));
  cudaError_t err = cudaSuccess;
  switch (plan.kind) {
  case Plan::kWarpRows:
    layer_norm_backward_kernel<T, P, kVec, 1, true, 32 * kWarpRowWarps>
        <<<plan.grid, plan.threads, g.partials != nullptr ? plan.shared : 0, stream>>>(g);
    err = cudaGetLastError();
    break;
  case Plan::kRing:
    if (plan.per == 16)
      err = launch_ring<layer_norm_backward_ring_kernel<T, P, kFull, 16, 512, kShift>>(plan, stream, g, plan.ring, status);
    else
      err = launch_ring<layer_norm_backward_ring_kernel<T, P, kFull, 32, 512, kShift>>(plan, stream, g, plan.ring, status);
    break;
  case Plan::kDirect:
    // (The ring takes all 16-bit rows of whole packs that fit it, and float32 rows of more than 256 packs.)
    if constexpr (kVec == 8) {
      err = cudaErrorInvalidConfiguration;
    } else {
      if (kVec > 1 || plan.threads <= 512)
        layer_norm_backward_kernel<T, P, kVec, 1, false, 512><<<plan.grid, plan.threads, 0, stream>>>(g);
      else if constexpr (kVec == 1)
        layer_norm_backward_kernel<T, P, kVec, 1, false, kMaxThreads><<<plan.grid, plan.threads, 0, stream>>>(g);
      err = cudaGetLastError();
    }
    break;
  case Plan::kLong:
    if (g.partials != nullptr) {  // before dx, which may be written over dy or x
      const long long packs = (g.cols + kVec - 1) / kVec;
      const dim3 blocks(static_cast<unsigned>((packs + 255) / 256), static_cast<unsigned>(plan.grid));
      layer_norm_columns_kernel<T, kVec><<<blocks, 256, 0, stream>>>(g);
      err = cudaGetLastError();
      if (err != cudaSuccess)
        return err;
    }
    layer_norm_backward_long_kernel<T, P, kVec><<<static_cast<unsigned>(g.rows), kMaxThreads, 0, stream>>>(g);
    err = cudaGetLastError();
    break;
  }
  if (err != cudaSuccess || g.partials == nullptr)
    return err;
  const dim3 blocks(static_cast<unsigned>((g.cols + 31) / 32), 2);
  if (g.cols >= 8192)
    layer_norm_partials_kernel<P, 8><<<blocks, 256, 0, stream>>>(g.partials, plan.grid, g.cols, dweight, dbias);
  else
    layer_norm_partials_kernel<P, 32><<<blocks, 1024, 0, stream>>>(g.partials, plan.grid, g.cols, dweight, dbias);
  return cudaGetLastError();
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace norm

// See norm::kShifted.
int layer_norm_vector(int dtype, long long cols, const void *a, long long lda, const void *b, long long ldb, const void *c,
                      long long ldc) {
  const int size = dtype == kCTypeF32 ? 4 : 2;
  auto place = [](const void *p) { return reinterpret_cast<uintptr_t>(p) & 15; };
  auto pitch = [&](long long ld) { return static_cast<int>((ld * size) & 15); };
  if (place(a) != place(b) || place(a) != place(c) || pitch(lda) != pitch(ldb) || pitch(lda) != pitch(ldc))
    return 1;
  return place(a) == 0 && pitch(lda) == 0 && pitch(cols) == 0 ? 16 / size : norm::kShifted;
}

#define HC_NORM_TYPES(CALL)                                                                          \
  if (dtype == kCTypeF32)                                                                            \
    return vec <= 1 ? CALL(float, float, 1) : CALL(float, float, 4);                                 \
  if (dtype == kCTypeF16) {                                                                          \
    if (param_dtype == kCTypeF32)                                                                    \
      return vec <= 1 ? CALL(__half, float, 1) : CALL(__half, float, 8);                             \
    return vec <= 1 ? CALL(__half, __half, 1) : CALL(__half, __half, 8);                             \
  }                                                                                                  \
  if (param_dtype == kCTypeF32)                                                                      \
    return vec <= 1 ? CALL(__nv_bfloat16, float, 1) : CALL(__nv_bfloat16, float, 8);                 \
  return vec <= 1 ? CALL(__nv_bfloat16, __nv_bfloat16, 1) : CALL(__nv_bfloat16, __nv_bfloat16, 8)

cudaError_t launch_layer_norm(const void *x, long long ldx, const void *weight, const void *bias, void *y,
                              long long ldy, float *mean, float *rstd, long long rows, long long cols, float eps,
                              int dtype, int param_dtype, int sm_count, int *status, cudaStream_t stream) {
  const int vec = layer_norm_vector(dtype, cols, x, ldx, y, ldy, y, ldy);
  norm::Forward f{x, weight, bias, y, mean, rstd, rows, cols, ldx, ldy, eps,
                  norm::aligned16(weight) && norm::aligned16(bias) ? 1 : 0};
#define HC_NORM_FORWARD(T, P, V) norm::launch_forward<T, P, V>(f, vec, sm_count, status, stream)
  HC_NORM_TYPES(HC_NORM_FORWARD);
#undef HC_NORM_FORWARD
}

int layer_norm_backward_launches(long long rows, long long cols, int vec, int dtype, int param_dtype, int sm_count, bool params) {
  const norm::Plan plan =
      norm::backward_plan(rows, cols, vec, dtype == kCTypeF32 ? 4 : 2, param_dtype == kCTypeF32 ? 4 : 2, sm_count);
  return 1 + (params ? (plan.kind == norm::Plan::kLong ? 2 : 1) : 0);
}

size_t layer_norm_backward_scratch(long long rows, long long cols, int vec, int dtype, int param_dtype, int sm_count) {
  const norm::Plan plan =
      norm::backward_plan(rows, cols, vec, dtype == kCTypeF32 ? 4 : 2, param_dtype == kCTypeF32 ? 4 : 2, sm_count);
  return sizeof(float) * 2 * static_cast<size_t>(cols) * static_cast<size_t>(plan.grid);
}

cudaError_t launch_layer_norm_backward(const void *dy, long long lddy, const void *x, long long ldx, const void *weight,
                                       const float *mean, const float *rstd, void *dx, long long lddx, void *dweight,
                                       void *dbias, float *partials, long long rows, long long cols, int dtype,
                                       int param_dtype, int sm_count, int *status, cudaStream_t stream) {
  const int vec = layer_norm_vector(dtype, cols, dy, lddy, x, ldx, dx, lddx);
  norm::Backward g{dy, x, weight, mean, rstd, dx, dweight != nullptr || dbias != nullptr ? partials : nullptr,
                   rows, cols, lddy, ldx, lddx, norm::aligned16(weight) ? 1 : 0};
#define HC_NORM_BACKWARD(T, P, V) \
  norm::launch_backward<T, P, V>(g, static_cast<P *>(dweight), static_cast<P *>(dbias), vec, sm_count, status, stream)
  HC_NORM_TYPES(HC_NORM_BACKWARD);
#undef HC_NORM_BACKWARD
}

}  // namespace sm100
}  // namespace hc

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
#include "gemm_launch.h"

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
  const float rstd = 1.0f / sqrtf(row_sum<kWarpRow>(square, sums[1]) * inv + f.eps);
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
  const float rstd = 1.0f / sqrtf(row_sum<false>(square, sums[1]) * inv + f.eps);
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
      float w[kVec];
      load_params<P, kVec>(w, static_cast<const P *>(g.weight), c, cols, g.params_aligned != 0, 1.0f);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float n = (to_float(px[j].v[i]) - mean) * rstd, d = to_float(pd[j].v[i]);  // (d is 0 past the end)
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

// out[c] = sum over the partial rows, in their order within each of 32 interleaved chains that are then
// added pairwise. A warp reads 32 neighbouring columns of a partial row.
template <typename P>
__global__ void __launch_bounds__(1024)
layer_norm_partials_kernel(const float *partials, int count, long long cols, P *dweight, P *dbias) {
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, chain = threadIdx.x >> 5;
  const long long c = static_cast<long long>(blockIdx.x) * 32 + lane;
  const bool bias = blockIdx.y != 0;
  P *out = bias ? dbias : dweight;
  if (out == nullptr)
    return;
  float sum = 0.0f;
  if (c < cols)
    for (int k = chain; k < count; k += 32)
      sum += partials[(static_cast<long long>(k) * 2 + (bias ? 1 : 0)) * cols + c];
  part[chain][lane] = sum;
  __syncthreads();
  // Warp `chain` now adds the 32 chains of column `chain` of the block.
  const float total = warp_sum(part[lane][chain]);
  const long long column = static_cast<long long>(blockIdx.x) * 32 + chain;
  if (lane == 0 && column < cols)
    out[column] = from_float<P>(total);
}

// ---------------------------------------------------------------- launch ------------

template <typename T, typename P, int kVec>
cudaError_t launch_forward(const Forward &f, int sm_count, cudaStream_t stream) {
  const long long packs = (f.cols + kVec - 1) / kVec;
  if (packs <= 64) {  // a warp holds a row in at most two packs per lane
    const unsigned grid = static_cast<unsigned>((f.rows + kWarpRowWarps - 1) / kWarpRowWarps);
    if (packs <= 32)
      layer_norm_kernel<T, P, kVec, 1, true><<<grid, 32 * kWarpRowWarps, 0, stream>>>(f);
    else
      layer_norm_kernel<T, P, kVec, 2, true><<<grid, 32 * kWarpRowWarps, 0, stream>>>(f);
    return cudaGetLastError();
  }
  if (packs > 4 * kMaxThreads) {
    layer_norm_long_kernel<T, P, kVec><<<static_cast<unsigned>(f.rows), kMaxThreads, 0, stream>>>(f);
    return cudaGetLastError();
  }
  // Few rows: as many threads as the row has packs, for the shortest chain of loads. Many rows: CTAs of
  // at most 256 threads with up to four packs each, so that several CTAs overlap on an SM.
  const int most = f.rows <= sm_count ? kMaxThreads : 256;
  int per = packs <= most ? 1 : packs <= 2 * most ? 2 : 4;
  const int threads = static_cast<int>(((packs + per - 1) / per + 31) / 32 * 32);
  const unsigned grid = static_cast<unsigned>(f.rows);
  if (per == 1)
    layer_norm_kernel<T, P, kVec, 1, false><<<grid, threads, 0, stream>>>(f);
  else if (per == 2)
    layer_norm_kernel<T, P, kVec, 2, false><<<grid, threads, 0, stream>>>(f);
  else
    layer_norm_kernel<T, P, kVec, 4, false><<<grid, threads, 0, stream>>>(f);
  return cudaGetLastError();
}

// CTAs of the backward kernel, which is also the number of partial rows.
int backward_grid(long long rows, long long cols, int vec, int sm_count, bool *long_rows) {
  const long long packs = (cols + vec - 1) / vec;
  *long_rows = packs > kMaxThreads;
  if (*long_rows) {
    // Row chunks of the column kernel: enough CTAs to fill the GPU a few times over.
    const long long column_blocks = (packs + 255) / 256;
    const long long chunks = (8LL * sm_count + column_blocks - 1) / column_blocks;
    return static_cast<int>(rows < chunks ? rows : chunks);
  }
  const bool warp_rows = packs <= 32;
  const long long units = warp_rows ? (rows + kWarpRowWarps - 1) / kWarpRowWarps : rows;
  const int threads = warp_rows ? 32 * kWarpRowWarps : static_cast<int>((packs + 31) / 32 * 32);
  const long long ctas = static_cast<long long>(sm_count) * (threads >= 1024 ? 1 : threads > 512 ? 1 : threads > 256 ? 2 : 4);
  return static_cast<int>(units < ctas ? units : ctas);
}

template <typename T, typename P, int kVec>
cudaError_t launch_backward(const Backward &g, P *dweight, P *dbias, int sm_count, cudaStream_t stream) {
  const long long packs = (g.cols + kVec - 1) / kVec;
  bool long_rows = false;
  const int grid = backward_grid(g.rows, g.cols, kVec, sm_count, &long_rows);
  cudaError_t err = cudaSuccess;
  if (long_rows) {
    if (g.partials != nullptr) {  // before dx, which may be written over dy or x
      const dim3 blocks(static_cast<unsigned>((packs + 255) / 256), static_cast<unsigned>(grid));
      layer_norm_columns_kernel<T, kVec><<<blocks, 256, 0, stream>>>(g);
      err = cudaGetLastError();
      if (err != cudaSuccess)
        return err;
    }
    layer_norm_backward_long_kernel<T, P, kVec><<<static_cast<unsigned>(g.rows), kMaxThreads, 0, stream>>>(g);
  } else if (packs <= 32) {
    const size_t shared = g.partials != nullptr ? sizeof(float) * kWarpRowWarps * 2 * static_cast<size_t>(g.cols) : 0;
    layer_norm_backward_kernel<T, P, kVec, 1, true, 32 * kWarpRowWarps>
        <<<grid, 32 * kWarpRowWarps, shared, stream>>>(g);
  } else {
    const int threads = static_cast<int>((packs + 31) / 32 * 32);
    if (threads <= 512)
      layer_norm_backward_kernel<T, P, kVec, 1, false, 512><<<grid, threads, 0, stream>>>(g);
    else
      layer_norm_backward_kernel<T, P, kVec, 1, false, kMaxThreads><<<grid, threads, 0, stream>>>(g);
  }
  err = cudaGetLastError();
  if (err != cudaSuccess || g.partials == nullptr)
    return err;
  const dim3 blocks(static_cast<unsigned>((g.cols + 31) / 32), 2);
  layer_norm_partials_kernel<P><<<blocks, 1024, 0, stream>>>(g.partials, grid, g.cols, dweight, dbias);
  return cudaGetLastError();
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace norm

// Elements per access: 16 bytes' worth when every row of every matrix starts on a 16-byte boundary.
int layer_norm_vector(int dtype, const void *a, long long lda, const void *b, long long ldb, const void *c,
                      long long ldc) {
  const int size = dtype == kCTypeF32 ? 4 : 2;
  const bool ok = norm::aligned16(a) && norm::aligned16(b) && norm::aligned16(c) && (lda * size) % 16 == 0 &&
                  (ldb * size) % 16 == 0 && (ldc * size) % 16 == 0;
  return ok ? 16 / size : 1;
}

#define HC_NORM_TYPES(CALL)                                                                          \
  if (dtype == kCTypeF32)                                                                            \
    return vec == 1 ? CALL(float, float, 1) : CALL(float, float, 4);                                 \
  if (dtype == kCTypeF16) {                                                                          \
    if (param_dtype == kCTypeF32)                                                                    \
      return vec == 1 ? CALL(__half, float, 1) : CALL(__half, float, 8);                             \
    return vec == 1 ? CALL(__half, __half, 1) : CALL(__half, __half, 8);                             \
  }                                                                                                  \
  if (param_dtype == kCTypeF32)                                                                      \
    return vec == 1 ? CALL(__nv_bfloat16, float, 1) : CALL(__nv_bfloat16, float, 8);                 \
  return vec == 1 ? CALL(__nv_bfloat16, __nv_bfloat16, 1) : CALL(__nv_bfloat16, __nv_bfloat16, 8)

cudaError_t launch_layer_norm(const void *x, long long ldx, const void *weight, const void *bias, void *y,
                              long long ldy, float *mean, float *rstd, long long rows, long long cols, float eps,
                              int dtype, int param_dtype, int sm_count, cudaStream_t stream) {
  const int vec = layer_norm_vector(dtype, x, ldx, y, ldy, y, ldy);
  norm::Forward f{x, weight, bias, y, mean, rstd, rows, cols, ldx, ldy, eps,
                  norm::aligned16(weight) && norm::aligned16(bias) ? 1 : 0};
#define HC_NORM_FORWARD(T, P, V) norm::launch_forward<T, P, V>(f, sm_count, stream)
  HC_NORM_TYPES(HC_NORM_FORWARD);
#undef HC_NORM_FORWARD
}

int layer_norm_backward_launches(long long rows, long long cols, int vec, bool params) {
  bool long_rows = false;
  norm::backward_grid(rows, cols, vec, 1, &long_rows);
  return 1 + (params ? (long_rows ? 2 : 1) : 0);
}

size_t layer_norm_backward_scratch(long long rows, long long cols, int vec, int sm_count) {
  bool long_rows = false;
  return sizeof(float) * 2 * static_cast<size_t>(cols) *
         static_cast<size_t>(norm::backward_grid(rows, cols, vec, sm_count, &long_rows));
}

cudaError_t launch_layer_norm_backward(const void *dy, long long lddy, const void *x, long long ldx, const void *weight,
                                       const float *mean, const float *rstd, void *dx, long long lddx, void *dweight,
                                       void *dbias, float *partials, long long rows, long long cols, int dtype,
                                       int param_dtype, int sm_count, cudaStream_t stream) {
  const int vec = layer_norm_vector(dtype, dy, lddy, x, ldx, dx, lddx);
  norm::Backward g{dy, x, weight, mean, rstd, dx, dweight != nullptr || dbias != nullptr ? partials : nullptr,
                   rows, cols, lddy, ldx, lddx, norm::aligned16(weight) ? 1 : 0};
#define HC_NORM_BACKWARD(T, P, V) \
  norm::launch_backward<T, P, V>(g, static_cast<P *>(dweight), static_cast<P *>(dbias), sm_count, stream)
  HC_NORM_TYPES(HC_NORM_BACKWARD);
#undef HC_NORM_BACKWARD
}

}  // namespace sm100
}  // namespace hc

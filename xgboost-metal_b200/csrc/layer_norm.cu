// Layer norm over rows of n values, forward and backward.
//
//   m = mean x,  q = 1 / sqrt(mean (x - m)^2 + eps),  h = (x - m) q,  y = h w + b
//   g = dy w,  dx = q (g - mean g - h mean(g h)),  dw = sum dy h,  db = sum dy
//
// All arithmetic is float32; the variance is the mean square of the centred
// values, never a difference of two large sums. Results are rounded once.
#include <algorithm>

#include "nn_device.cuh"

namespace xgbb::nn {
namespace {

constexpr int kThreads = 256;

// The sum of one value a thread over the block, in every thread. `part` holds
// one float a warp.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float (*part)[N]) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int m = 16; m; m >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], m);
  __syncthreads();
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) part[warp][i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = lane < warps ? part[lane][i] : 0.0f;
#pragma unroll
    for (int m = 16; m; m >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], m);
  }
}

// A block a row, any length: three passes over the row.
template <class T, class P, int VE>
__global__ void __launch_bounds__(kThreads)
    norm_kernel(const T* __restrict__ x, int64_t x_stride, uint64_t rows, uint32_t dim, const P* __restrict__ w,
                const P* __restrict__ b, float eps, T* __restrict__ y, int64_t y_stride, float* __restrict__ mean,
                float* __restrict__ rstd) {
  __shared__ float part[32][1];
  for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + int64_t(row) * x_stride;
    float sum[1] = {0.0f};
    for (uint32_t c = threadIdx.x * VE; c < dim; c += kThreads * VE) {
      const auto v = load<T, VE>(xr + c);
#pragma unroll
      for (int e = 0; e < VE; ++e) sum[0] += v.f(e);
    }
    block_sum<1>(sum, part);
    const float m = sum[0] / float(dim);
    float square[1] = {0.0f};
    for (uint32_t c = threadIdx.x * VE; c < dim; c += kThreads * VE) {
      const auto v = load<T, VE>(xr + c);
#pragma unroll
      for (int e = 0; e < VE; ++e) square[0] = fmaf(v.f(e) - m, v.f(e) - m, square[0]);
    }
    block_sum<1>(square, part);
    const float q = 1.0f / sqrtf(square[0] / float(dim) + eps);
    if (threadIdx.x == 0) {
      if (mean) mean[row] = m;
      if (rstd) rstd[row] = q;
    }
    for (uint32_t c = threadIdx.x * VE; c < dim; c += kThreads * VE) {
      const auto v = load<T, VE>(xr + c);
      float r[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        r[e] = (v.f(e) - m) * q;
        if (w) r[e] *= to_f32(w[c + e]);
        if (b) r[e] += to_f32(b[c + e]);
      }
      store<T, VE>(y + int64_t(row) * y_stride + c, r);
    }
  }
}

// dx, a block a row, any length.
template <class T, class P, int VE>
__global__ void __launch_bounds__(kThreads)
    norm_dx_kernel(const T* __restrict__ grad, int64_t grad_stride, const T* __restrict__ x, int64_t x_stride,
                   const float* __restrict__ mean, const float* __restrict__ rstd, uint64_t rows, uint32_t dim,
                   const P* __restrict__ w, T* __restrict__ dx, int64_t dx_stride) {
  __shared__ float part[32][2];
  for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + int64_t(row) * x_stride;
    const T* gr = grad + int64_t(row) * grad_stride;
    const float m = mean[row], q = rstd[row];
    float sum[2] = {0.0f, 0.0f};
    for (uint32_t c = threadIdx.x * VE; c < dim; c += kThreads * VE) {
      const auto v = load<T, VE>(xr + c);
      const auto d = load<T, VE>(gr + c);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float g = w ? d.f(e) * to_f32(w[c + e]) : d.f(e);
        sum[0] += g;
        sum[1] = fmaf(g, (v.f(e) - m) * q, sum[1]);
      }
    }
    block_sum<2>(sum, part);
    const float a = sum[0] / float(dim), bb = sum[1] / float(dim);
    for (uint32_t c = threadIdx.x * VE; c < dim; c += kThreads * VE) {
      const auto v = load<T, VE>(xr + c);
      const auto d = load<T, VE>(gr + c);
      float r[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float g = w ? d.f(e) * to_f32(w[c + e]) : d.f(e);
        r[e] = q * (g - a - (v.f(e) - m) * q * bb);
      }
      store<T, VE>(dx + int64_t(row) * dx_stride + c, r);
    }
  }
}

constexpr uint32_t kMaxParts = 296;

uint32_t part_count(uint64_t rows) { return uint32_t(std::min<uint64_t>(kMaxParts, (rows + 15) / 16)); }

// Block (x, y) sums the column tile y over the rows x, x + gridDim.x, ... into
// parts[x][2][dim]: the weight's gradient, then the bias's.
template <class T>
__global__ void __launch_bounds__(kThreads)
    norm_columns_kernel(const T* __restrict__ grad, int64_t grad_stride, const T* __restrict__ x, int64_t x_stride,
                        const float* __restrict__ mean, const float* __restrict__ rstd, uint64_t rows, uint32_t dim,
                        float* __restrict__ parts) {
  const uint32_t c = blockIdx.y * kThreads + threadIdx.x;
  if (c >= dim) return;
  float dw = 0.0f, db = 0.0f;
  for (uint64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float d = to_f32(grad[int64_t(row) * grad_stride + c]);
    dw = fmaf(d, (to_f32(x[int64_t(row) * x_stride + c]) - mean[row]) * rstd[row], dw);
    db += d;
  }
  parts[(uint64_t(blockIdx.x) * 2) * dim + c] = dw;
  parts[(uint64_t(blockIdx.x) * 2 + 1) * dim + c] = db;
}

// The parts' sums, in their order.
template <class P>
__global__ void __launch_bounds__(kThreads)
    norm_parts_kernel(const float* __restrict__ parts, uint32_t count, uint32_t dim, P* __restrict__ dw,
                      P* __restrict__ db) {
  const uint32_t c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= dim) return;
  float a = 0.0f, b = 0.0f;
  for (uint32_t p = 0; p < count; ++p) {
    a += parts[uint64_t(p) * 2 * dim + c];
    b += parts[(uint64_t(p) * 2 + 1) * dim + c];
  }
  if (dw) dw[c] = from_f32<P>(a);
  if (db) db[c] = from_f32<P>(b);
}

}  // namespace

void layer_norm(const Mat& x, uint64_t rows, uint64_t dim, const void* weight, const void* bias, int param_type,
                float eps, const Mat& y, float* mean, float* rstd, cudaStream_t stream) {
  if (!rows) return;
  with_types(x.type, param_type, [&](auto* pt, auto* pp) {
    using T = std::remove_pointer_t<decltype(pt)>;
    using P = std::remove_pointer_t<decltype(pp)>;
    with_width<T>(x, rows, y, rows, dim, [&](auto width) {
      norm_kernel<T, P, decltype(width)::value>
          <<<unsigned(std::min<uint64_t>(rows, 1u << 30)), kThreads, 0, stream>>>(
              static_cast<const T*>(x.data), x.stride, rows, uint32_t(dim), static_cast<const P*>(weight),
              static_cast<const P*>(bias), eps, static_cast<T*>(const_cast<void*>(y.data)), y.stride, mean, rstd);
    });
  });
  XGBB_CUDA(cudaGetLastError());
}

size_t layer_norm_backward_workspace(uint64_t rows, uint64_t dim) { return size_t(part_count(rows)) * 2 * dim * 4; }

void layer_norm_backward(const Mat& grad, const Mat& x, const float* mean, const float* rstd, uint64_t rows,
                         uint64_t dim, const void* weight, int param_type, const Mat& dx, void* dweight,
                         void* dbias, void* workspace, size_t bytes, cudaStream_t stream) {
  require(!(dweight || dbias) || bytes >= layer_norm_backward_workspace(rows, dim),
          "the workspace is smaller than its query says");
  with_types(x.type, param_type, [&](auto* pt, auto* pp) {
    using T = std::remove_pointer_t<decltype(pt)>;
    using P = std::remove_pointer_t<decltype(pp)>;
    const T* g = static_cast<const T*>(grad.data);
    const T* v = static_cast<const T*>(x.data);
    if (rows) {
      // The widths that x and dx allow, and grad too.
      with_width<T>(x, rows, dx, rows, dim, [&](auto wide) {
        constexpr int VE = decltype(wide)::value;
        const auto go = [&](auto width) {
          norm_dx_kernel<T, P, decltype(width)::value>
              <<<unsigned(std::min<uint64_t>(rows, 1u << 30)), kThreads, 0, stream>>>(
                  g, grad.stride, v, x.stride, mean, rstd, rows, uint32_t(dim), static_cast<const P*>(weight),
                  static_cast<T*>(const_cast<void*>(dx.data)), dx.stride);
        };
        if (row_aligned(grad.data, grad.stride, rows, sizeof(T), VE)) go(std::integral_constant<int, VE>());
        else go(std::integral_constant<int, 1>());
      });
    }
    if (!dweight && !dbias) return;
    float* parts = static_cast<float*>(workspace);
    const uint32_t count = part_count(rows);
    if (count)
      norm_columns_kernel<T><<<dim3(count, blocks_for(dim, kThreads)), kThreads, 0, stream>>>(
          g, grad.stride, v, x.stride, mean, rstd, rows, uint32_t(dim), parts);
    norm_parts_kernel<P><<<blocks_for(dim, kThreads), kThreads, 0, stream>>>(
        parts, count, uint32_t(dim), static_cast<P*>(dweight), static_cast<P*>(dbias));
  });
  XGBB_CUDA(cudaGetLastError());
}

}  // namespace xgbb::nn

// Layer norm over the last dimension, forward and backward (layer_norm.h has the formulas).
//
// mean and variance are taken in two passes, the second over the centred values: a variance from the sum of squares
// loses what a mean much larger than the spread leaves of 24 bits.
//
// With g = dy * weight and xhat = (s - mean) * rstd the gradients are
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat)) + dsum,  dweight = sum over rows of dy * xhat,  dbias = sum of dy.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kernels/dependent_launch.cuh"
#include "kernels/layer_norm.h"

using switchml::kernels::LaunchOverlapped;
using switchml::kernels::WaitForEarlierKernels;

namespace {

// As in wgrad_gemm.cu: a failed launch does not leave its error for the next caller of cudaGetLastError().
int Launched(cudaError_t e) {
  if (e == cudaSuccess) return 0;
  cudaGetLastError();
  return -4;
}

__device__ __forceinline__ float ToFloat(float v) { return v; }
__device__ __forceinline__ float ToFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T FromFloat(float v);
template <> __device__ __forceinline__ float FromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 FromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Weight or bias: a pointer to either type, or none.
struct Parameter {
  const void* data;
  int type;
  __device__ __forceinline__ float At(int i, float none) const {
    if (!data) return none;
    return type == SML_NORM_F32 ? static_cast<const float*>(data)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(data)[i]);
  }
};

__device__ __forceinline__ float WarpSum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

constexpr int kAnyThreads = 256;

// The sums of a and b over the block, in every thread. `part` is used again by the next call.
__device__ __forceinline__ float2 BlockSum(float a, float b, float2* part) {
  a = WarpSum(a);
  b = WarpSum(b);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  float2 sum = make_float2(0.f, 0.f);
#pragma unroll
  for (int w = 0; w < kAnyThreads / 32; w++) sum.x += part[w].x, sum.y += part[w].y;
  __syncthreads();
  return sum;
}

// Rows of any length: a block per row, which reads it once for each of the statistics and once more.
template <class T>
__global__ void __launch_bounds__(kAnyThreads)
ForwardAnyKernel(const T* x, const T* residual, Parameter weight, Parameter bias, T* y, T* sum, float* mean_out, float* rstd_out,
                 long long rows, int n, float eps) {
  __shared__ float2 part[kAnyThreads / 32];
  WaitForEarlierKernels();
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* in = x + row * n;
    float total = 0.f;
    if (residual) {
      for (int i = threadIdx.x; i < n; i += kAnyThreads) {
        const T s = FromFloat<T>(ToFloat(in[i]) + ToFloat(residual[row * n + i]));
        sum[row * n + i] = s;
        total += ToFloat(s);
      }
      in = sum + row * n;  // each thread reads what it wrote itself
    } else {
      for (int i = threadIdx.x; i < n; i += kAnyThreads) total += ToFloat(in[i]);
    }
    const float mean = BlockSum(total, 0.f, part).x / n;
    float squares = 0.f;
    for (int i = threadIdx.x; i < n; i += kAnyThreads) {
      const float d = ToFloat(in[i]) - mean;
      squares += d * d;
    }
    const float rstd = 1.f / sqrtf(BlockSum(squares, 0.f, part).x / n + eps);
    for (int i = threadIdx.x; i < n; i += kAnyThreads)
      y[row * n + i] = FromFloat<T>((ToFloat(in[i]) - mean) * rstd * weight.At(i, 1.f) + bias.At(i, 0.f));
    if (threadIdx.x == 0 && mean_out) mean_out[row] = mean, rstd_out[row] = rstd;
  }
}

template <class T>
__global__ void __launch_bounds__(kAnyThreads)
BackwardAnyKernel(const T* dy, const T* dsum, const T* s, Parameter weight, const float* mean_in, const float* rstd_in, T* dx,
                  long long rows, int n) {
  __shared__ float2 part[kAnyThreads / 32];
  WaitForEarlierKernels();
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *g_row = dy + row * n, *s_row = s + row * n;
    const float mean = mean_in[row], rstd = rstd_in[row];
    float a = 0.f, b = 0.f;
    for (int i = threadIdx.x; i < n; i += kAnyThreads) {
      const float g = ToFloat(g_row[i]) * weight.At(i, 1.f);
      a += g;
      b += g * ((ToFloat(s_row[i]) - mean) * rstd);
    }
    const float2 sums = BlockSum(a, b, part);
    const float ca = sums.x / n, cb = sums.y / n;
    for (int i = threadIdx.x; i < n; i += kAnyThreads) {
      const float g = ToFloat(g_row[i]) * weight.At(i, 1.f);
      float d = rstd * (g - ca - (ToFloat(s_row[i]) - mean) * rstd * cb);
      if (dsum) d += ToFloat(dsum[row * n + i]);
      dx[row * n + i] = FromFloat<T>(d);
    }
  }
}

// Sums over rows: a block takes 32 columns and one of gridDim.y shares of the rows; its sums go to the workspace.
template <class T>
__global__ void __launch_bounds__(kAnyThreads)
ColumnsAnyKernel(const T* dy, const T* s, const float* mean, const float* rstd, float* workspace, long long rows, int n) {
  __shared__ float2 part[kAnyThreads / 32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, column = blockIdx.x * 32 + lane;
  const long long first = rows * blockIdx.y / gridDim.y, last = rows * (blockIdx.y + 1) / gridDim.y;
  float dw = 0.f, db = 0.f;
  WaitForEarlierKernels();
  if (column < n) {
#pragma unroll 4
    for (long long row = first + warp; row < last; row += kAnyThreads / 32) {
      const float g = ToFloat(dy[row * n + column]);
      dw += g * ((ToFloat(s[row * n + column]) - mean[row]) * rstd[row]);
      db += g;
    }
  }
  part[warp][lane] = make_float2(dw, db);
  __syncthreads();
  if (warp == 0 && column < n) {
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kAnyThreads / 32; w++) sum.x += part[w][lane].x, sum.y += part[w][lane].y;
    float* out = workspace + static_cast<long long>(blockIdx.y) * 2 * n;
    out[column] = sum.x;
    out[n + column] = sum.y;
  }
}

constexpr int kFinishColumns = 32, kFinishRows = 16;

// The sums of `parts` partial sums, in order.
__global__ void __launch_bounds__(kFinishColumns* kFinishRows)
FinishColumnsKernel(const float* workspace, void* dweight, void* dbias, int parts, int n, int wtype) {
  __shared__ float2 part[kFinishRows][kFinishColumns];
  const int lane = threadIdx.x % kFinishColumns, r = threadIdx.x / kFinishColumns, column = blockIdx.x * kFinishColumns + lane;
  float2 sum = make_float2(0.f, 0.f);
  WaitForEarlierKernels();
  if (column < n) {
#pragma unroll 4
    for (int p = r; p < parts; p += kFinishRows) {
      const float* from = workspace + static_cast<long long>(p) * 2 * n;
      sum.x += from[column];
      sum.y += from[n + column];
    }
  }
  part[r][lane] = sum;
  __syncthreads();
  if (r == 0 && column < n) {
    sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kFinishRows; i++) sum.x += part[i][lane].x, sum.y += part[i][lane].y;
    if (wtype == SML_NORM_F32) {
      if (dweight) static_cast<float*>(dweight)[column] = sum.x;
      if (dbias) static_cast<float*>(dbias)[column] = sum.y;
    } else {
      if (dweight) static_cast<__nv_bfloat16*>(dweight)[column] = __float2bfloat16_rn(sum.x);
      if (dbias) static_cast<__nv_bfloat16*>(dbias)[column] = __float2bfloat16_rn(sum.y);
    }
  }
}

unsigned RowBlocks(long long rows) { return static_cast<unsigned>(rows < (1 << 20) ? rows : (1 << 20)); }

int RowShares(long long rows, int n) {
  const long long columns = (static_cast<long long>(n) + 31) / 32;
  long long shares = (148 * 8 + columns - 1) / columns;
  if (shares > rows / 32 + 1) shares = rows / 32 + 1;
  return static_cast<int>(shares);
}

bool Known(int type) { return type == SML_NORM_F32 || type == SML_NORM_BF16; }

template <class T>
int Forward(const void* x, const void* residual, Parameter weight, Parameter bias, void* y, void* sum, float* mean, float* rstd,
            long long rows, int n, float eps, cudaStream_t stream) {
  return Launched(LaunchOverlapped(ForwardAnyKernel<T>, RowBlocks(rows), kAnyThreads, 0, 1, stream, static_cast<const T*>(x),
                                   static_cast<const T*>(residual), weight, bias, static_cast<T*>(y), static_cast<T*>(sum), mean,
                                   rstd, rows, n, eps));
}

template <class T>
int Backward(const void* dy, const void* dsum, const void* s, Parameter weight, const float* mean, const float* rstd, void* dx,
             void* dweight, void* dbias, float* workspace, long long rows, int n, int wtype, cudaStream_t stream) {
  cudaError_t e = LaunchOverlapped(BackwardAnyKernel<T>, RowBlocks(rows), kAnyThreads, 0, 1, stream, static_cast<const T*>(dy),
                                   static_cast<const T*>(dsum), static_cast<const T*>(s), weight, mean, rstd, static_cast<T*>(dx),
                                   rows, n);
  if (e != cudaSuccess || (!dweight && !dbias)) return Launched(e);
  const int shares = RowShares(rows, n);
  const unsigned columns = static_cast<unsigned>((static_cast<long long>(n) + 31) / 32);
  ColumnsAnyKernel<T><<<dim3(columns, shares), kAnyThreads, 0, stream>>>(static_cast<const T*>(dy), static_cast<const T*>(s), mean,
                                                                          rstd, workspace, rows, n);
  if ((e = cudaGetLastError()) != cudaSuccess) return Launched(e);
  return Launched(LaunchOverlapped(FinishColumnsKernel, (n - 1) / kFinishColumns + 1, kFinishColumns * kFinishRows, 0, 1, stream,
                                   workspace, dweight, dbias, shares, n, wtype));
}

}  // namespace

extern "C" int switchml_layer_norm_forward(const void* x, const void* residual, const void* weight, const void* bias, void* y,
                                           void* sum, float* mean, float* rstd, long long rows, int features, float eps, int type,
                                           int wtype, void* stream) {
  if (!x || !y || (residual && !sum) || !mean != !rstd || rows <= 0 || features <= 0 || !Known(type) || !Known(wtype)) return -1;
  return (type == SML_NORM_F32 ? Forward<float> : Forward<__nv_bfloat16>)(x, residual, Parameter{weight, wtype},
                                                                          Parameter{bias, wtype}, y, sum, mean, rstd, rows, features,
                                                                          eps, static_cast<cudaStream_t>(stream));
}

extern "C" long long switchml_layer_norm_workspace(long long rows, int features, int type) {
  if (rows <= 0 || features <= 0 || !Known(type)) return 0;
  return 2ll * features * RowShares(rows, features);
}

extern "C" int switchml_layer_norm_backward(const void* dy, const void* dsum, const void* s, const void* weight, const float* mean,
                                            const float* rstd, void* dx, void* dweight, void* dbias, float* workspace, long long rows,
                                            int features, int type, int wtype, void* stream) {
  if (!dy || !s || !mean || !rstd || !dx || ((dweight || dbias) && !workspace) || rows <= 0 || features <= 0 || !Known(type) ||
      !Known(wtype))
    return -1;
  return (type == SML_NORM_F32 ? Backward<float> : Backward<__nv_bfloat16>)(dy, dsum, s, Parameter{weight, wtype}, mean, rstd, dx,
                                                                            dweight, dbias, workspace, rows, features, wtype,
                                                                            static_cast<cudaStream_t>(stream));
}

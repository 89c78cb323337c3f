// AdamW over many tensors in one launch, and the norm of all their gradients (adamw.h has the formulas).
//
// A launch takes its tensors' addresses and sizes as kernel parameters: nothing has to be copied to the device, a captured
// launch keeps its own, and two of them share nothing. The parameters' memory is read through the constant cache; a warp
// finds the tensor of its tile by halving.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "kernels/adamw.h"
#include "kernels/dependent_launch.cuh"

using switchml::kernels::LaunchOverlapped;
using switchml::kernels::WaitForEarlierKernels;

namespace {

// As in wgrad_gemm.cu: a failed launch does not leave its error for the next caller of cudaGetLastError().
int Launched(cudaError_t e) {
  if (e == cudaSuccess) return 0;
  cudaGetLastError();
  return -4;
}

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kBlock = SML_ADAMW_ALIGN;  // values that a warp takes at once: 8 per lane
constexpr int kScaled = 32;              // values that share a scale
constexpr long long kMaxNumel = 1ll << 38;  // of a tensor: the number of its tiles fits 31 bits
constexpr int kMaxTensors = SML_ADAMW_TENSORS;

struct StepArgs {
  SmlAdamwTensor tensor[kMaxTensors];
  unsigned first_tile[kMaxTensors + 1];
  int count;
  int tile_blocks;  // kBlock's of a tile
  SmlAdamwState state;
  float lr, beta1, one_minus_beta1, beta2, one_minus_beta2, eps, decay, log_beta1, log_beta2, max_norm;
  const float *lr_tensor, *norm;
};

// The last i with first[i] <= tile.
__device__ __forceinline__ int TensorOfTile(const unsigned* first, int count, unsigned tile) {
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= tile) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A bijection of the 32-bit numbers that leaves no pattern: multiplications by the fractions of the golden ratio and of
// the square root of 2 carry every bit upwards, shifts bring them down again.
__device__ __forceinline__ unsigned Mix(unsigned x) {
  x ^= x >> 16;
  x *= 0x9E3779B1u;
  x ^= x >> 15;
  x *= 0x6A09E667u;
  return x ^ (x >> 16);
}

__device__ __forceinline__ float FromCode(unsigned code) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(code), __NV_E4M3);
  return __half2float(h);
}

// A tensor's factors in this step.
struct Factors {
  float size, rsqrt2, keep;  // lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), 1 - lr * decay
  unsigned key;
};

__device__ __forceinline__ Factors FactorsOf(const StepArgs& a, int t, float lr, unsigned long long value) {
  Factors f;
  // 1 - beta^t = -expm1(t log beta): the logarithm comes from the host in more than fp32, and expm1 keeps what a
  // difference from 1 would lose.
  f.size = lr / -expm1f(t * a.log_beta1);
  f.rsqrt2 = 1.f / sqrtf(-expm1f(t * a.log_beta2));
  f.keep = 1.f - lr * a.decay;
  f.key = Mix(Mix(Mix(a.state.seed) + static_cast<unsigned>(t)) + static_cast<unsigned>(value >> 32));
  return f;
}

// The code (without sign) of a magnitude over its scale.
__device__ __forceinline__ unsigned ToCode(float y, unsigned bits16) {
  const bool small = y < 0.015625f;
  const float t = small ? __fadd_rn(y, 0.015625f) : y;
  return ((__float_as_uint(t) + (bits16 << 4 | 8)) >> 20) - (small ? 968 : 960);
}

// The fp32 value of a parameter, and back.
__device__ __forceinline__ float WithRemainder(__nv_bfloat16 p, short remainder) {
  return __uint_as_float((static_cast<unsigned>(__bfloat16_as_ushort(p)) << 16) + static_cast<unsigned>(static_cast<int>(remainder)));
}
__device__ __forceinline__ unsigned PlusHalf(float p) {  // the parameter is the high half
  return (isnan(p) ? 0x7fc00000u : __float_as_uint(p)) + 0x8000u;
}

template <class T, int kBits>
__global__ void __launch_bounds__(kThreads) AdamwKernel(const __grid_constant__ StepArgs a) {
  WaitForEarlierKernels();
  const int lane = threadIdx.x & 31;
  float clip = 1.f;
  if (a.norm) {
    const float norm = *a.norm;
    if (!(norm <= 3.402823466e38f)) return;  // infinite or NaN, the same for every thread: nothing changes
    clip = fminf(__fdiv_rn(a.max_norm, __fadd_rn(norm, 1e-6f)), 1.f);
  }
  const float lr = a.lr_tensor ? *a.lr_tensor : a.lr;
  const unsigned tile = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (tile < a.first_tile[a.count]) {
    const int i = TensorOfTile(a.first_tile, a.count, tile);
    const SmlAdamwTensor& x = a.tensor[i];
    const long long start = static_cast<long long>(tile - a.first_tile[i]) * a.tile_blocks * kBlock;
    const long long end = min(x.numel, start + static_cast<long long>(a.tile_blocks) * kBlock);
    const int t = a.state.steps[x.step] + 1;
    const long long state = static_cast<long long>(x.place) * kBlock;
    for (long long at = start; at < end; at += kBlock) {
      const unsigned long long first = a.state.first + state + at;
      const Factors f = FactorsOf(a, t, lr, first);
#pragma unroll 1
      for (int j = 0; j < kBlock / 32; j++) {
        const long long k = at + j * 32 + lane;  // 32 values that share a scale: one per lane
        const bool in = k < end;
        float m = 0.f, v = 0.f, g = 0.f, p = 0.f;
        if (in) {
          p = static_cast<float>(static_cast<const T*>(x.param)[k]);
          if constexpr (sizeof(T) == 2) p = WithRemainder(static_cast<const T*>(x.param)[k], a.state.remainder[state + k]);
          g = static_cast<float>(static_cast<const T*>(x.grad)[k]);
          if constexpr (kBits == 32) {
            m = static_cast<const float*>(a.state.exp_avg)[state + k];
            v = static_cast<const float*>(a.state.exp_avg_sq)[state + k];
          } else {
            m = FromCode(static_cast<const unsigned char*>(a.state.exp_avg)[state + k]) *
                __uint_as_float(static_cast<unsigned>(a.state.exp_avg_scale[(state + k) / kScaled]) << 23);
            v = FromCode(static_cast<const unsigned char*>(a.state.exp_avg_sq)[state + k]) *
                __uint_as_float(static_cast<unsigned>(a.state.exp_avg_sq_scale[(state + k) / kScaled]) << 23);
          }
        }
        g = __fmul_rn(g, clip);
        m = __fadd_rn(__fmul_rn(m, a.beta1), __fmul_rn(g, a.one_minus_beta1));
        v = __fadd_rn(__fmul_rn(v, a.beta2), __fmul_rn(__fmul_rn(g, a.one_minus_beta2), g));
        p = p * f.keep - f.size * (m / (sqrtf(v) * f.rsqrt2 + a.eps));
        if (in) {
          if constexpr (sizeof(T) == 2) {
            const unsigned w = PlusHalf(p);
            static_cast<T*>(x.param)[k] = __ushort_as_bfloat16(static_cast<unsigned short>(w >> 16));
            a.state.remainder[state + k] = static_cast<short>(w ^ 0x8000u);  // (w - 0x8000) of its low half
          } else {
            static_cast<T*>(x.param)[k] = p;
          }
        }
        if constexpr (kBits == 32) {
          if (in) {
            static_cast<float*>(a.state.exp_avg)[state + k] = m;
            static_cast<float*>(a.state.exp_avg_sq)[state + k] = v;
          }
        } else {
          const unsigned em = max(__reduce_max_sync(0xffffffffu, __float_as_uint(m) & 0x7fffffffu) >> 23, 8u);
          const unsigned ev = max(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu) >> 23, 8u);
          const unsigned h = Mix(static_cast<unsigned>(first) + j * 32 + lane + f.key);
          unsigned cm = 0x7f, cv = 0x7f;  // NaN
          if (em < 255) cm = ToCode(fabsf(m) * __uint_as_float((261 - em) << 23), h & 0xffff) | (__float_as_uint(m) >> 24 & 0x80);
          if (ev < 255) {
            cv = ToCode(v * __uint_as_float((261 - ev) << 23), h >> 16);
            if (cv == 0 && v > 0.f) cv = 1;
          }
          if (in) {
            static_cast<unsigned char*>(a.state.exp_avg)[state + k] = static_cast<unsigned char>(cm);
            static_cast<unsigned char*>(a.state.exp_avg_sq)[state + k] = static_cast<unsigned char>(cv);
            if (lane == 0) {
              a.state.exp_avg_scale[(state + k) / kScaled] = static_cast<unsigned char>(em < 255 ? em - 7 : 255);
              a.state.exp_avg_sq_scale[(state + k) / kScaled] = static_cast<unsigned char>(ev < 255 ? ev - 7 : 255);
            }
          }
        }
      }
    }
  }
  // The block that ends last counts the step: every block has read the counts by then.
  __syncthreads();
  __shared__ bool last;
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(a.state.ticket, 1) == static_cast<int>(gridDim.x) - 1;
  }
  __syncthreads();
  if (!last) return;
  for (int i = threadIdx.x; i < a.count; i += kThreads) a.state.steps[a.tensor[i].step]++;
  if (threadIdx.x == 0) *a.state.ticket = 0;
}

struct MasterArgs {
  SmlAdamwTensor tensor[kMaxTensors];
  unsigned first_tile[kMaxTensors + 1];
  int count;
  const short* remainder;
  float* out;
};

// A warp per kBlock values.
template <class T>
__global__ void __launch_bounds__(kThreads) MastersKernel(const __grid_constant__ MasterArgs a) {
  WaitForEarlierKernels();
  const unsigned tile = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (tile >= a.first_tile[a.count]) return;
  const int i = TensorOfTile(a.first_tile, a.count, tile);
  const SmlAdamwTensor& x = a.tensor[i];
  const long long start = static_cast<long long>(tile - a.first_tile[i]) * kBlock, state = static_cast<long long>(x.place) * kBlock;
#pragma unroll
  for (int j = 0; j < kBlock / 32; j++) {
    const long long k = start + j * 32 + (threadIdx.x & 31);
    if (k >= x.numel) break;
    const T p = static_cast<const T*>(x.param)[k];
    if constexpr (sizeof(T) == 2) a.out[state + k] = WithRemainder(p, a.remainder[state + k]);
    else a.out[state + k] = p;
  }
}

constexpr int kNormBlocks = 148 * 4;  // partial sums of a launch, at most
constexpr int kNormTile = 4096;       // values that a block takes at once

struct NormArgs {
  SmlNormTensor tensor[kMaxTensors];
  unsigned first_tile[kMaxTensors + 1];
  int count;
  double* partial;
};

__device__ __forceinline__ double BlockSum(double v) {
  __shared__ double part[kWarps];
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int w = 0; w < kWarps; w++) sum += part[w];
  return sum;
}

// Squares are summed in fp64: 2^-53 of a sum over 10^9 values still leaves the result right to its last fp32 bit, and no
// gradient's square overflows or vanishes.
__global__ void __launch_bounds__(kThreads) NormKernel(const __grid_constant__ NormArgs a) {
  WaitForEarlierKernels();
  double sum = 0.0;
  for (unsigned tile = blockIdx.x; tile < a.first_tile[a.count]; tile += gridDim.x) {
    const int i = TensorOfTile(a.first_tile, a.count, tile);
    const SmlNormTensor& x = a.tensor[i];
    const long long start = static_cast<long long>(tile - a.first_tile[i]) * kNormTile;
    const long long end = min(x.numel, start + kNormTile);
    if (x.type == SML_ADAMW_F32) {
      for (long long k = start + threadIdx.x; k < end; k += kThreads) {
        const double g = static_cast<const float*>(x.data)[k];
        sum += g * g;
      }
    } else {
      for (long long k = start + threadIdx.x; k < end; k += kThreads) {
        const double g = __bfloat162float(static_cast<const __nv_bfloat16*>(x.data)[k]);
        sum += g * g;
      }
    }
  }
  sum = BlockSum(sum);
  if (threadIdx.x == 0) a.partial[blockIdx.x] = sum;
}

__global__ void __launch_bounds__(kThreads) FinishNormKernel(const double* partial, int parts, float* out) {
  WaitForEarlierKernels();
  double sum = 0.0;
  for (int i = threadIdx.x; i < parts; i += kThreads) sum += partial[i];
  sum = BlockSum(sum);
  if (threadIdx.x == 0) *out = static_cast<float>(sqrt(sum));
}

// Fills in one launch's share of `tensors` from `*at` on and returns the number of its tiles. Empty tensors take none.
template <class Args, class Tensor>
unsigned TakeTensors(const Tensor* tensors, int count, long long tile, int* at, Args* a) {
  unsigned long long tiles = 0;
  a->count = 0;
  for (; *at < count && a->count < kMaxTensors; ++*at) {
    const unsigned long long more = static_cast<unsigned long long>((tensors[*at].numel + tile - 1) / tile);
    if (tiles + more > 0x7fffffffull && a->count > 0) break;
    a->tensor[a->count] = tensors[*at];
    a->first_tile[a->count++] = static_cast<unsigned>(tiles);
    tiles += more;
  }
  a->first_tile[a->count] = static_cast<unsigned>(tiles);
  return static_cast<unsigned>(tiles);
}

}  // namespace

extern "C" int switchml_adamw_step(const SmlAdamwTensor* tensors, int count, const SmlAdamwState* state, const SmlAdamwStep* step,
                                   int type, void* stream) {
  if (!tensors || count < 0 || !state || !step || (state->bits != 32 && state->bits != 8) || !state->exp_avg || !state->exp_avg_sq ||
      !state->steps || !state->ticket || (state->bits == 8 && (!state->exp_avg_scale || !state->exp_avg_sq_scale)) ||
      (type != SML_ADAMW_F32 && (type != SML_ADAMW_BF16 || !state->remainder)))
    return -1;
  for (int i = 0; i < count; i++)
    if (tensors[i].numel < 0 || tensors[i].numel > kMaxNumel || (tensors[i].numel && (!tensors[i].param || !tensors[i].grad))) return -1;
  StepArgs a;
  a.state = *state;
  a.lr = static_cast<float>(step->lr);
  a.beta1 = static_cast<float>(step->beta1), a.one_minus_beta1 = static_cast<float>(1.0 - step->beta1);
  a.beta2 = static_cast<float>(step->beta2), a.one_minus_beta2 = static_cast<float>(1.0 - step->beta2);
  a.log_beta1 = static_cast<float>(log(step->beta1)), a.log_beta2 = static_cast<float>(log(step->beta2));
  a.eps = static_cast<float>(step->eps), a.decay = static_cast<float>(step->decay);
  a.max_norm = step->max_norm, a.lr_tensor = step->lr_tensor, a.norm = step->norm;
  a.tile_blocks = 4;
  for (int at = 0; at < count;) {
    const unsigned tiles = TakeTensors(tensors, count, static_cast<long long>(a.tile_blocks) * kBlock, &at, &a);
    const unsigned blocks = tiles ? (tiles + kWarps - 1) / kWarps : 1;  // (empty tensors' steps count too)
    void (*kernel)(StepArgs) = type == SML_ADAMW_F32 ? (state->bits == 32 ? AdamwKernel<float, 32> : AdamwKernel<float, 8>)
                                                     : (state->bits == 32 ? AdamwKernel<__nv_bfloat16, 32> : AdamwKernel<__nv_bfloat16, 8>);
    const cudaError_t e = LaunchOverlapped(kernel, blocks, kThreads, 0, 1, static_cast<cudaStream_t>(stream), a);
    if (e != cudaSuccess) return Launched(e);
  }
  return 0;
}

extern "C" int switchml_adamw_masters(const SmlAdamwTensor* tensors, int count, const short* remainder, float* out, int type, void* stream) {
  if (!tensors || count < 0 || !out || (type != SML_ADAMW_F32 && (type != SML_ADAMW_BF16 || !remainder))) return -1;
  for (int i = 0; i < count; i++)
    if (tensors[i].numel < 0 || tensors[i].numel > kMaxNumel || (tensors[i].numel && !tensors[i].param)) return -1;
  MasterArgs a;
  a.remainder = remainder, a.out = out;
  for (int at = 0; at < count;) {
    const unsigned tiles = TakeTensors(tensors, count, kBlock, &at, &a);
    if (!tiles) continue;
    const cudaError_t e = LaunchOverlapped(type == SML_ADAMW_F32 ? MastersKernel<float> : MastersKernel<__nv_bfloat16>,
                                           (tiles + kWarps - 1) / kWarps, kThreads, 0, 1, static_cast<cudaStream_t>(stream), a);
    if (e != cudaSuccess) return Launched(e);
  }
  return 0;
}

extern "C" long long switchml_grad_norm_workspace(int count) {
  return count <= 0 ? 0 : static_cast<long long>((count + kMaxTensors - 1) / kMaxTensors) * kNormBlocks;
}

extern "C" int switchml_grad_norm(const SmlNormTensor* tensors, int count, double* workspace, float* out, void* stream) {
  if (count < 0 || !out || (count && (!tensors || !workspace))) return -1;
  for (int i = 0; i < count; i++)
    if (tensors[i].numel < 0 || tensors[i].numel > kMaxNumel || (tensors[i].numel && !tensors[i].data) ||
        (tensors[i].type != SML_ADAMW_F32 && tensors[i].type != SML_ADAMW_BF16))
      return -1;
  NormArgs a;
  int parts = 0;
  for (int at = 0; at < count;) {
    const unsigned tiles = TakeTensors(tensors, count, kNormTile, &at, &a);
    if (!tiles) continue;
    const unsigned blocks = tiles < kNormBlocks ? tiles : kNormBlocks;
    a.partial = workspace + parts;
    const cudaError_t e = LaunchOverlapped(NormKernel, blocks, kThreads, 0, 1, static_cast<cudaStream_t>(stream), a);
    if (e != cudaSuccess) return Launched(e);
    parts += blocks;
  }
  return Launched(LaunchOverlapped(FinishNormKernel, 1, kThreads, 0, 1, static_cast<cudaStream_t>(stream), workspace, parts, out));
}

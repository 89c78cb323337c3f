// AdamW over many tensors in one launch, and the norm of all their gradients (adamw.h has the formulas).
//
// A launch takes its tensors' addresses and sizes as kernel parameters: nothing has to be copied to the device, and a captured
// launch keeps its own table. (Launches of one optimizer share its counts of steps, its ticket and the norm: they follow each
// other.) The parameters' memory is read through the constant cache; a warp finds the tensor of its tile by halving.
//
// The step is one pass over memory: 28 bytes per value with fp32 parameters and moments, 16.125 with moments in 8 bits (bf16
// parameters: 26 and 14.125). A lane takes 8 neighbours, whole sectors of every array; tiles go to the warps in the order of
// the addresses (blocks that stay and stride over the tiles: 1200 instead of 1096 us). 2^28 values:
//   fp32, moments in 32 bits 1096 us = 6.86 TB/s, in 8 bits 669 us = 6.47 TB/s; bf16 1043 us = 6.69 and 655 us = 5.79 TB/s
// (a plain copy: 6.55 TB/s). With 32 bits memory is the limit. With 8 bits it is nearly so: 53 instructions per value, of
// which hashing takes 9 and each of the two codes 6; one value per lane took 4 times, scalar arithmetic 1.4 times as long. Reading
// the next block ahead gained 1 % there (bf16: 5 %) and lost as much with 32 bits and on a few million values.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "kernels/adamw.h"
#include "kernels/dependent_launch.cuh"
#include "kernels/packed.cuh"

using switchml::kernels::Fma;
using switchml::kernels::LaunchOverlapped;
using switchml::kernels::LetNextKernelStart;
using switchml::kernels::LoadWords;
using switchml::kernels::Packed;
using switchml::kernels::Pair;
using switchml::kernels::StoreWords;
using switchml::kernels::WaitForEarlierKernels;

namespace {

// As in wgrad_gemm.cu: a failed launch does not leave its error for the next caller of cudaGetLastError().
int Launched(cudaError_t e) {
  if (e == cudaSuccess) return 0;
  cudaGetLastError();
  return -4;
}

constexpr int kSms = 148;  // of a B200
constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kBlock = SML_ADAMW_ALIGN;  // values that a warp takes at once: 8 per lane
constexpr int kScaled = 32;              // values that share a scale
constexpr long long kMaxNumel = 1ll << 38;  // of a tensor: the number of its tiles fits 31 bits
constexpr long long kMaxTiles = 0x7fffffff;  // of a launch
constexpr int kMaxTensors = SML_ADAMW_TENSORS;
constexpr int kFewTensors = 32;          // a launch of so few takes kernel parameters of 1 instead of 12 KB

struct StepFactors {
  int count;
  int tile_blocks;  // kBlock's of a tile
  SmlAdamwState state;
  float lr, beta1, one_minus_beta1, beta2, one_minus_beta2, eps, decay, log_beta1, log_beta2, max_norm, minus_zero;
  const float *lr_tensor, *norm;
};
template <int kMax> struct StepArgs {
  StepFactors all;
  SmlAdamwTensor tensor[kMax];
  unsigned first_tile[kMax + 1];
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

// A tensor's factors in this step.
struct Factors {
  float size, rsqrt2, keep;  // lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), 1 - lr * decay
  unsigned key;
};

__device__ __forceinline__ Factors FactorsOf(const StepFactors& a, int t, float lr) {
  Factors f;
  // 1 - beta^t = -expm1(t log beta): the host takes the logarithm in fp64 and rounds it to fp32 once (of a beta that was rounded
  // first, 1 - beta would keep few of its bits), and expm1 keeps what a difference from 1 would lose.
  f.size = lr / -expm1f(t * a.log_beta1);
  f.rsqrt2 = 1.f / sqrtf(-expm1f(t * a.log_beta2));
  f.keep = 1.f - lr * a.decay;
  f.key = Mix(Mix(a.state.seed) + static_cast<unsigned>(t));
  return f;
}

// What is hashed for the value at `place` of the flat buffers; for the next 255 behind a multiple of 256 it counts on.
__device__ __forceinline__ unsigned HashedAt(const StepFactors& a, const Factors& f, long long place) {
  const unsigned long long value = a.state.first + place;
  return static_cast<unsigned>(value) + Mix(f.key + static_cast<unsigned>(value >> 32));
}

// The fp32 values of two parameters with their remainders: parameter << 16 plus the signed remainder, which is the unsigned
// remainder + 0x8000 less 0x8000.
__device__ __forceinline__ Pair WithRemainders(unsigned params, unsigned remainders) {
  remainders ^= 0x80008000u;
  return Pair(__uint_as_float(__byte_perm(params, remainders, 0x1054) - 0x8000u),
              __uint_as_float(__byte_perm(params, remainders, 0x3276) - 0x8000u));
}
// Back: the parameter is the high half of this, the remainder the low half ^ 0x8000. (Arithmetic makes 0x7fffffff of every NaN:
// that one would wrap around.)
__device__ __forceinline__ unsigned PlusHalf(float p) {
  return static_cast<unsigned>(min(static_cast<int>(__float_as_uint(p)), 0x7fff7fff)) + 0x8000u;
}

// The root and the reciprocal of an update come from the SM's approximations (2^-23 and 2^-23 of the result, by the PTX
// manual; correctly rounded ones are sequences of a dozen instructions): they touch p alone, in which the update is a
// small term. Both flush subnormal numbers, so second moments below 2^-126 count as 2^-126.
__device__ __forceinline__ float Root(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float Reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// The larger of two, the largest of three; NaN where one of them is.
__device__ __forceinline__ float Larger(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float Largest(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// One step of two values.
__device__ __forceinline__ void Update(const StepFactors& a, const Factors& f, float clip, Pair g, Pair* p, Pair* m, Pair* v) {
  g = g * Pair(clip);
  // Products that are rounded before they are added: ptxas makes one operation with one rounding of mul.rn.f32x2 and
  // add.rn.f32x2, but not of this, as long as it does not know that what is added is -0.
  const Pair none(a.minus_zero);
  *m = Fma(*m, Pair(a.beta1), none) + Fma(g, Pair(a.one_minus_beta1), none);
  *v = Fma(*v, Pair(a.beta2), none) + Fma(g * Pair(a.one_minus_beta2), g, none);
  const float2 square = v->Both();
  const Pair root(Root(Larger(square.x, 1.17549435e-38f)), Root(Larger(square.y, 1.17549435e-38f)));
  const float2 below = Fma(root, Pair(f.rsqrt2), Pair(a.eps)).Both();
  *p = Fma(*p, Pair(f.keep), *m * Pair(Reciprocal(below.x), Reciprocal(below.y)) * Pair(-f.size));
}

// Scales of a block whose largest magnitude is `largest`: its exponent e (see adamw.h), the byte and the number.
__device__ __forceinline__ unsigned ExponentOf(float largest) { return max(__float_as_uint(largest) >> 23, 8u); }
__device__ __forceinline__ unsigned char ScaleByte(unsigned e) { return static_cast<unsigned char>(e < 255 ? e - 7 : 255); }
__device__ __forceinline__ float ScaleOf(unsigned char byte) { return __uint_as_float(static_cast<unsigned>(byte) << 23); }

// Values, rounded to their codes without the sign: in the top 8 bits of the results. A number over its scale times 2^-120
// has the bits of its e4m3 form in front of 20 more, subnormal numbers too, since both formats then begin at the same
// exponent; the product rounds as the addition of 2^-6 in adamw.h does. `random` is what those 20 bits get added, 4 places up.
__device__ __forceinline__ Pair OverScale(Pair x, unsigned e) {
  return x * Pair(__uint_as_float((261 - e) << 23)) * Pair(7.52316385e-37f);
}
__device__ __forceinline__ unsigned ToCode(float y, unsigned random) { return (__float_as_uint(y) << 4) + random; }
__device__ __forceinline__ unsigned MCode(float y, unsigned hash) {
  return ToCode(y, __byte_perm(hash, 0x80, 0x5104)) | (__float_as_uint(y) & 0x80000000u);
}
__device__ __forceinline__ unsigned VCode(float y, float v, unsigned hash) {
  const unsigned code = ToCode(y, __byte_perm(hash, 0x80, 0x5324));
  return v > 0.f ? max(code, 1u << 24) : code;
}
constexpr unsigned kNanCode = 0x7f;
// A mask of the first n of four bytes (all of them from 4 on, none up to 0).
__device__ __forceinline__ unsigned BytesBelow(int n) { return n >= 4 ? ~0u : n <= 0 ? 0u : (1u << 8 * n) - 1; }

// 8 numbers in e4m3.
struct Packed8 {
  unsigned w[2];
  __device__ __forceinline__ Pair Decoded(int i) const {  // values 2i and 2i + 1 of e4m3
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i / 2] >> (i & 1) * 16), __NV_E4M3);
    const float2 v = __half22float2(h);
    return Pair(v.x, v.y);
  }
};

// 8 neighbours of a tensor: a whole vector, or only the first `valid` of them (the others count as 0) and at any address.
template <bool kWhole, class T> __device__ __forceinline__ void LoadTensor(const T* from, int valid, Packed<T>* to) {
  if constexpr (kWhole) {
    LoadWords(from, to->w);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if constexpr (sizeof(T) == 2) {
        const unsigned v = i < valid ? *reinterpret_cast<const unsigned short*>(from + i) : 0;
        to->w[i / 2] = i & 1 ? to->w[i / 2] | v << 16 : v;
      } else {
        to->w[i] = i < valid ? *reinterpret_cast<const unsigned*>(from + i) : 0;
      }
    }
  }
}
template <bool kWhole, class T> __device__ __forceinline__ void StoreTensor(T* to, int valid, const Packed<T>& from) {
  if constexpr (kWhole) {
    StoreWords(to, from.w);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (i >= valid) continue;
      if constexpr (sizeof(T) == 2) reinterpret_cast<unsigned short*>(to)[i] = static_cast<unsigned short>(from.w[i / 2] >> (i & 1) * 16);
      else reinterpret_cast<unsigned*>(to)[i] = from.w[i];
    }
  }
}

// What is known of a block of kBlock values: whole, at addresses that vectors can be read from or at any other; or a tensor's last.
enum class Block { kVectors, kSingles, kEnd };

// kBlock values of a tensor from k on: 8 neighbours per lane, a scale for 4 lanes. State is there for whole blocks, and what
// lies behind a tensor's end in it stays 0, also where a block of moments becomes NaN: a good state that is loaded into the
// tensor's part of the block would be lost to what shares its scale.
template <class T, int kBits, Block kIs>
__device__ __forceinline__ void StepBlock(const StepFactors& a, const SmlAdamwTensor& x, long long k, long long state, const Factors& f,
                                          float clip, int lane) {
  using M = std::conditional_t<kBits == 32, Packed<float>, Packed8>;
  constexpr int kMoment = kBits / 8;
  constexpr bool kWhole = kIs == Block::kVectors;
  k += lane * 8;
  state += k;
  const int valid = kIs == Block::kEnd ? static_cast<int>(max(min(x.numel - k, 8ll), 0ll)) : 8;
  T* const param = static_cast<T*>(x.param) + k;
  char* const m_at = static_cast<char*>(a.state.exp_avg) + state * kMoment;
  char* const v_at = static_cast<char*>(a.state.exp_avg_sq) + state * kMoment;
  Packed<T> p, g;
  Packed<__nv_bfloat16> r;
  M m, v;
  unsigned char sm = 0, sv = 0;
  LoadTensor<kWhole>(static_cast<const T*>(x.grad) + k, valid, &g);
  LoadTensor<kWhole>(param, valid, &p);
  LoadWords(m_at, m.w);
  LoadWords(v_at, v.w);
  if constexpr (sizeof(T) == 2) LoadWords(a.state.remainder + state, r.w);
  if constexpr (kBits == 8) sm = a.state.exp_avg_scale[state / kScaled], sv = a.state.exp_avg_sq_scale[state / kScaled];
  Pair mf[4], vf[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (kBits == 32) {
      mf[i] = Pair(m.At(2 * i), m.At(2 * i + 1)), vf[i] = Pair(v.At(2 * i), v.At(2 * i + 1));
    } else {
      mf[i] = m.Decoded(i) * Pair(ScaleOf(sm)), vf[i] = v.Decoded(i) * Pair(ScaleOf(sv));
    }
    Pair pf(p.At(2 * i), p.At(2 * i + 1));
    if constexpr (sizeof(T) == 2)
      pf = WithRemainders(p.w[i], r.w[i]);
    Update(a, f, clip, Pair(g.At(2 * i), g.At(2 * i + 1)), &pf, &mf[i], &vf[i]);
    const float2 both = pf.Both();
    if constexpr (sizeof(T) == 2) {
      const unsigned x = PlusHalf(both.x), y = PlusHalf(both.y);
      p.w[i] = __byte_perm(x, y, 0x7632);
      r.w[i] = __byte_perm(x, y, 0x5410) ^ 0x80008000u;
    } else {
      p.w[2 * i] = __float_as_uint(both.x), p.w[2 * i + 1] = __float_as_uint(both.y);
    }
    if constexpr (kBits == 32) {
      const float2 mb = mf[i].Both(), vb = vf[i].Both();
      m.w[2 * i] = __float_as_uint(mb.x), m.w[2 * i + 1] = __float_as_uint(mb.y);
      v.w[2 * i] = __float_as_uint(vb.x), v.w[2 * i + 1] = __float_as_uint(vb.y);
    }
  }
  StoreTensor<kWhole>(param, valid, p);
  if constexpr (sizeof(T) == 2) {
    if constexpr (kIs == Block::kEnd) {
#pragma unroll
      for (int i = 0; i < 4; i++) r.w[i] = valid > 2 * i + 1 ? r.w[i] : valid > 2 * i ? r.w[i] & 0xffffu : 0;
    }
    StoreWords(a.state.remainder + state, r.w);
  }
  if constexpr (kBits == 8) {
    float largest_m = 0.f, largest_v = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 mb = mf[i].Both(), vb = vf[i].Both();
      largest_m = Largest(largest_m, fabsf(mb.x), fabsf(mb.y));
      largest_v = Largest(largest_v, vb.x, vb.y);
    }
#pragma unroll
    for (int o = 1; o < kScaled / 8; o *= 2) {
      largest_m = Larger(largest_m, __shfl_xor_sync(0xffffffffu, largest_m, o));
      largest_v = Larger(largest_v, __shfl_xor_sync(0xffffffffu, largest_v, o));
    }
    const unsigned em = ExponentOf(largest_m), ev = ExponentOf(largest_v);
    const unsigned first = HashedAt(a, f, state);
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      unsigned cm[4], cv[4];
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const float2 vb = vf[i + j / 2].Both(), ym = OverScale(mf[i + j / 2], em).Both(), yv = OverScale(vf[i + j / 2], ev).Both();
        const unsigned hx = Mix(first + i * 2 + j), hy = Mix(first + i * 2 + j + 1);
        cm[j] = MCode(ym.x, hx), cm[j + 1] = MCode(ym.y, hy);
        cv[j] = VCode(yv.x, vb.x, hx), cv[j + 1] = VCode(yv.y, vb.y, hy);
      }
      m.w[i / 2] = __byte_perm(__byte_perm(cm[0], cm[1], 0x73), __byte_perm(cm[2], cm[3], 0x73), 0x5410);
      v.w[i / 2] = __byte_perm(__byte_perm(cv[0], cv[1], 0x73), __byte_perm(cv[2], cv[3], 0x73), 0x5410);
    }
    if (em == 255) m.w[0] = m.w[1] = kNanCode * 0x01010101u;
    if (ev == 255) v.w[0] = v.w[1] = kNanCode * 0x01010101u;
    if constexpr (kIs == Block::kEnd) {
      const unsigned low = BytesBelow(valid), high = BytesBelow(valid - 4);
      m.w[0] &= low, m.w[1] &= high;
      v.w[0] &= low, v.w[1] &= high;
    }
    if (lane % (kScaled / 8) == 0) {
      a.state.exp_avg_scale[state / kScaled] = ScaleByte(em);
      a.state.exp_avg_sq_scale[state / kScaled] = ScaleByte(ev);
    }
  }
  StoreWords(m_at, m.w);
  StoreWords(v_at, v.w);
}

// For tensors at other addresses and for ends: out of the way of the first kind's registers and instructions. (A value per load
// and store: 2^25 values one element behind a multiple of 32 bytes take 172 us in fp32 with 32 bits and 132 with 8, where aligned
// ones take 144 and 93, in bf16 166 and 126 for 139 and 89.)
template <class T, int kBits, Block kIs, int kMax>  // (one for each kernel: ptxas 12.9 falls over one that two share)
__device__ __noinline__ void StepAnyBlock(const StepFactors& a, const SmlAdamwTensor& x, long long k, long long state, Factors f,
                                          float clip, int lane) {
  StepBlock<T, kBits, kIs>(a, x, k, state, f, clip, lane);
}

template <class T, int kBits, int kMax>
__global__ void __launch_bounds__(kThreads, kBits == 8 ? 7 : 8) AdamwKernel(const __grid_constant__ StepArgs<kMax> a) {
  const StepFactors& all = a.all;
  WaitForEarlierKernels();
  const int lane = threadIdx.x & 31;
  float clip = 1.f;
  if (all.norm) {
    const float norm = *all.norm;
    if (!(norm <= 3.402823466e38f)) return;  // infinite or NaN, the same for every thread: nothing changes
    clip = fminf(__fdiv_rn(all.max_norm, __fadd_rn(norm, 1e-6f)), 1.f);
  }
  const float lr = all.lr_tensor ? *all.lr_tensor : all.lr;
  const unsigned tile = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (tile < a.first_tile[all.count]) {
    const int i = TensorOfTile(a.first_tile, all.count, tile);
    const SmlAdamwTensor& x = a.tensor[i];
    const long long start = static_cast<long long>(tile - a.first_tile[i]) * all.tile_blocks * kBlock;
    const long long end = min(x.numel, start + static_cast<long long>(all.tile_blocks) * kBlock);
    const long long state = static_cast<long long>(x.place) * kBlock;
    const Factors f = FactorsOf(all, all.state.steps[x.step] + 1, lr);
    const bool vectors = ((reinterpret_cast<uintptr_t>(x.param) | reinterpret_cast<uintptr_t>(x.grad)) & (8 * sizeof(T) - 1)) == 0;
    for (long long k = start; k < end; k += kBlock) {
      if (k + kBlock > end) StepAnyBlock<T, kBits, Block::kEnd, kMax>(all, x, k, state, f, clip, lane);
      else if (vectors) StepBlock<T, kBits, Block::kVectors>(all, x, k, state, f, clip, lane);
      else StepAnyBlock<T, kBits, Block::kSingles, kMax>(all, x, k, state, f, clip, lane);
    }
  }
  // The block that ends last counts the step: every block has read the counts by then.
  __syncthreads();
  __shared__ bool last;
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(all.state.ticket, 1) == static_cast<int>(gridDim.x) - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();  // (every block's reads of the counts lie before its turn at the ticket)
  for (int i = threadIdx.x; i < all.count; i += kThreads) all.state.steps[a.tensor[i].step]++;
  if (threadIdx.x == 0) *all.state.ticket = 0;
}

template <int kMax> struct MasterArgs {
  SmlAdamwTensor tensor[kMax];
  unsigned first_tile[kMax + 1];
  int count;
  const short* remainder;
  float* out;
};

constexpr int kMasterBlocks = 4;  // kBlock's of a warp

// `out` is written up to the end of a tensor's last block, with zeros there.
template <class T, int kMax>
__global__ void __launch_bounds__(kThreads) MastersKernel(const __grid_constant__ MasterArgs<kMax> a) {
  WaitForEarlierKernels();
  const unsigned tile = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (tile >= a.first_tile[a.count]) return;
  const int i = TensorOfTile(a.first_tile, a.count, tile);
  const SmlAdamwTensor& x = a.tensor[i];
  const long long state = static_cast<long long>(x.place) * kBlock;
  const long long start = static_cast<long long>(tile - a.first_tile[i]) * kMasterBlocks * kBlock;
  const bool vectors = (reinterpret_cast<uintptr_t>(x.param) & (8 * sizeof(T) - 1)) == 0;
#pragma unroll
  for (int j = 0; j < kMasterBlocks; j++) {
    if (start + j * kBlock >= x.numel) break;
    const long long k = start + j * kBlock + (threadIdx.x & 31) * 8;
    Packed<T> p;
    if (vectors && k + 8 <= x.numel) LoadTensor<true>(static_cast<const T*>(x.param) + k, 8, &p);
    else LoadTensor<false>(static_cast<const T*>(x.param) + k, static_cast<int>(max(min(x.numel - k, 8ll), 0ll)), &p);
    Packed<float> out;
    if constexpr (sizeof(T) == 2) {
      Packed<__nv_bfloat16> r;
      LoadWords(a.remainder + state + k, r.w);
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const float2 both = WithRemainders(p.w[u], r.w[u]).Both();
        out.w[2 * u] = __float_as_uint(both.x), out.w[2 * u + 1] = __float_as_uint(both.y);
      }
    } else {
      out = p;
    }
    StoreWords(a.out + state + k, out.w);
  }
}

constexpr int kNormThreads = 256;
// Values that a block takes at once: 4 vectors per thread in flight. Reading needs them, the more the shorter the type: with 2048,
// 4096 and 8192 64 bf16 tensors of 2^20 values took 54, 37 and 30 us (fp32 56, 43 and 43), one of 2^22 4.9, 4.5 and 4.2, one of
// 2^20 fp32 values 3.6, 3.3 and 3.1, 300 of 5000 5.2, 5.1 and 4.9. 2^28 values in one are best with 4096 (162, 150 and 158), tensors
// far below a tile with the smallest (1000 of 1000: 8.6, 9.3 and 11.4).
constexpr int kNormTile = 8192;
constexpr int kNormBlocks = kSms * 5;  // partial sums of a launch, at most: the blocks that the GPU holds

template <int kMax> struct NormArgs {
  SmlNormTensor tensor[kMax];
  unsigned first_tile[kMax + 1];
  int count;
  double* partial;  // one for each block of this launch
  const double* all;  // of all launches: the last one's last block sums them, if there is a ticket
  int parts;
  int* ticket;
  float* out;
};

__device__ __forceinline__ double BlockSum(double v) {
  __shared__ double part[kNormThreads / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int w = 0; w < kNormThreads / 32; w++) sum += part[w];
  __syncthreads();
  return sum;
}

// Over this thread's share of the values from start to end, at most kNormTile.
template <class T>
__device__ __forceinline__ double SquaresOf(const T* x, long long start, long long end) {
  constexpr int kVectors = kNormTile / (kNormThreads * 8);
  const bool vectors = (reinterpret_cast<uintptr_t>(x) & (8 * sizeof(T) - 1)) == 0;
  double sum = 0.0;
  Packed<T> v[kVectors];
#pragma unroll
  for (int u = 0; u < kVectors; u++) {
    const long long k = start + (u * kNormThreads + threadIdx.x) * 8;
    if (vectors && k + 8 <= end) LoadTensor<true>(x + k, 8, &v[u]);
    else LoadTensor<false>(x + k, static_cast<int>(max(min(end - k, 8ll), 0ll)), &v[u]);
  }
#pragma unroll
  for (int u = 0; u < kVectors; u++) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const double g = v[u].At(i);
      sum += g * g;
    }
  }
  return sum;
}

// The root of the sum of all partial sums, in their order.
__device__ __forceinline__ void Finish(const double* partial, int parts, float* out) {
  double sum = 0.0;
#pragma unroll 8
  for (int i = threadIdx.x; i < parts; i += kNormThreads) sum += __ldcg(partial + i);
  sum = BlockSum(sum);
  if (threadIdx.x == 0) *out = static_cast<float>(sqrt(sum));
}

// Squares are summed in fp64: 2^-53 of a sum over 10^9 values still leaves the result right to its last fp32 bit, and no
// gradient's square overflows or vanishes. Converting takes 16 values per cycle and SM, where memory brings 6. Bound by reading:
// 335 M values 205 us = 6.5 TB/s, the 25.6 M of ResNet-50 19.4 us = 5.3 TB/s.
template <int kMax> __global__ void __launch_bounds__(kNormThreads, 5) NormKernel(const __grid_constant__ NormArgs<kMax> a) {
  WaitForEarlierKernels();
  LetNextKernelStart();
  double sum = 0.0;
  for (unsigned tile = blockIdx.x; tile < a.first_tile[a.count]; tile += gridDim.x) {
    const int i = TensorOfTile(a.first_tile, a.count, tile);
    const SmlNormTensor& x = a.tensor[i];
    const long long start = static_cast<long long>(tile - a.first_tile[i]) * kNormTile;
    const long long end = min(x.numel, start + kNormTile);
    sum += x.type == SML_ADAMW_F32 ? SquaresOf(static_cast<const float*>(x.data), start, end)
                                   : SquaresOf(static_cast<const __nv_bfloat16*>(x.data), start, end);
  }
  sum = BlockSum(sum);
  if (threadIdx.x == 0) a.partial[blockIdx.x] = sum;
  if (!a.ticket) return;
  __shared__ bool last;
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(a.ticket, 1) == static_cast<int>(gridDim.x) - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  Finish(a.all, a.parts, a.out);
  if (threadIdx.x == 0) *a.ticket = 0;
}

__global__ void __launch_bounds__(kNormThreads) FinishNormKernel(const double* partial, int parts, float* out) {
  WaitForEarlierKernels();
  Finish(partial, parts, out);
}

// Fills in one launch's share of `tensors` from `*at` on and returns the number of its tiles. Empty tensors take none.
template <class Args, class Tensor>
unsigned TakeTensors(const Tensor* tensors, int count, long long tile, int* at, Args* a, int* taken) {
  constexpr int kMax = sizeof(a->tensor) / sizeof(a->tensor[0]);
  unsigned long long tiles = 0;
  *taken = 0;
  for (; *at < count && *taken < kMax; ++*at) {
    const unsigned long long more = static_cast<unsigned long long>((tensors[*at].numel + tile - 1) / tile);
    if (tiles + more > kMaxTiles && *taken > 0) break;
    a->tensor[*taken] = tensors[*at];
    a->first_tile[(*taken)++] = static_cast<unsigned>(tiles);
    tiles += more;
  }
  a->first_tile[*taken] = static_cast<unsigned>(tiles);
  return static_cast<unsigned>(tiles);
}

// A warp's tile, in kBlock's. What a tile costs by itself (finding its tensor, the factors, a place among the resident
// warps) is shared by its blocks: 2^28 fp32 parameters with moments in 8 bits took 943, 771, 669 and 675 us with tiles
// of 4, 8, 16 and 32 blocks, with fp32 moments 1104, 1120, 1125 and 1131 us (there the memory is the limit, which likes short
// ones). Fewer values make smaller tiles: as many as the GPU holds warps, so that all run at once.
int TileBlocks(const SmlAdamwTensor* tensors, int count, int bits) {
  const int most = bits == 8 ? 16 : 4;
  const long long resident = static_cast<long long>(kSms) * kWarps * (bits == 8 ? 7 : 8);
  long long blocks = 0;
  for (int i = 0; i < count; i++) blocks += (tensors[i].numel + kBlock - 1) / kBlock;
  for (long long tile = (blocks + resident - 1) / resident; tile < most; tile++) {
    if (tile < 1) return 1;
    long long tiles = 0;
    for (int i = 0; i < count; i++) tiles += ((tensors[i].numel + kBlock - 1) / kBlock + tile - 1) / tile;
    if (tiles <= resident || (tile == 1 && blocks < resident)) return static_cast<int>(tile);
  }
  return most;
}

template <int kMax> int Step(const SmlAdamwTensor* tensors, int count, const StepFactors& factors, int type, cudaStream_t stream) {
  StepArgs<kMax> a;
  a.all = factors;
  for (int at = 0; at < count;) {
    const unsigned tiles = TakeTensors(tensors, count, static_cast<long long>(factors.tile_blocks) * kBlock, &at, &a, &a.all.count);
    const unsigned blocks = tiles ? (tiles + kWarps - 1) / kWarps : 1;  // (empty tensors' steps count too)
    void (*kernel)(StepArgs<kMax>) = AdamwKernel<float, 32, kMax>;
    if (type == SML_ADAMW_F32 && factors.state.bits == 8) kernel = AdamwKernel<float, 8, kMax>;
    if (type == SML_ADAMW_BF16) kernel = factors.state.bits == 8 ? AdamwKernel<__nv_bfloat16, 8, kMax> : AdamwKernel<__nv_bfloat16, 32, kMax>;
    const cudaError_t e = LaunchOverlapped(kernel, blocks, kThreads, 0, 1, stream, a);
    if (e != cudaSuccess) return Launched(e);
  }
  return 0;
}

template <int kMax>
int Masters(const SmlAdamwTensor* tensors, int count, const short* remainder, float* out, int type, cudaStream_t stream) {
  MasterArgs<kMax> a;
  a.remainder = remainder, a.out = out;
  for (int at = 0; at < count;) {
    const unsigned tiles = TakeTensors(tensors, count, kMasterBlocks * kBlock, &at, &a, &a.count);
    if (!tiles) continue;
    const cudaError_t e = LaunchOverlapped(type == SML_ADAMW_F32 ? MastersKernel<float, kMax> : MastersKernel<__nv_bfloat16, kMax>,
                                           (tiles + kWarps - 1) / kWarps, kThreads, 0, 1, stream, a);
    if (e != cudaSuccess) return Launched(e);
  }
  return 0;
}

template <int kMax>
int GradNorm(const SmlNormTensor* tensors, int count, double* workspace, int* ticket, float* out, cudaStream_t stream) {
  NormArgs<kMax> a;
  a.all = workspace, a.out = out, a.parts = 0;
  int at = 0;
  do {
    const unsigned tiles = TakeTensors(tensors, count, kNormTile, &at, &a, &a.count);
    if (!tiles && !(ticket && at == count)) continue;
    const unsigned each = (tiles + kNormBlocks - 1) / kNormBlocks;  // tiles of a block: the same number for all but the last
    const unsigned blocks = tiles ? (tiles + each - 1) / each : 1;
    a.partial = workspace + a.parts;
    a.parts += blocks;
    a.ticket = at == count ? ticket : nullptr;
    const cudaError_t e = LaunchOverlapped(NormKernel<kMax>, blocks, kNormThreads, 0, 1, stream, a);
    if (e != cudaSuccess) return Launched(e);
  } while (at < count);
  if (ticket) return 0;
  return Launched(LaunchOverlapped(FinishNormKernel, 1, kNormThreads, 0, 1, stream, a.all, a.parts, out));
}

// (A power of two: a division for every address is seen in a call with hundreds of tensors.)
bool At(const void* p, unsigned multiple) { return (reinterpret_cast<uintptr_t>(p) & (multiple - 1)) == 0; }

unsigned SizeOf(int type) { return type == SML_ADAMW_F32 ? 4 : 2; }

}  // namespace

extern "C" int switchml_adamw_step(const SmlAdamwTensor* tensors, int count, const SmlAdamwState* state, const SmlAdamwStep* step,
                                   int type, void* stream) {
  if (!tensors || count < 0 || !state || !step || (state->bits != 32 && state->bits != 8) || !state->exp_avg || !state->exp_avg_sq ||
      !state->steps || !state->ticket || (state->bits == 8 && (!state->exp_avg_scale || !state->exp_avg_sq_scale)) ||
      (type != SML_ADAMW_F32 && (type != SML_ADAMW_BF16 || !state->remainder)))
    return -1;
  const unsigned vector = state->bits == 32 ? 32 : 8;
  if (!At(state->exp_avg, vector) || !At(state->exp_avg_sq, vector) || !At(state->remainder, 16) || !At(state->steps, 4) ||
      !At(state->ticket, 4) || !At(step->lr_tensor, 4) || !At(step->norm, 4))
    return -1;
  for (int i = 0; i < count; i++)
    if (tensors[i].numel < 0 || tensors[i].numel > kMaxNumel || (tensors[i].numel && (!tensors[i].param || !tensors[i].grad)) ||
        !At(tensors[i].param, SizeOf(type)) || !At(tensors[i].grad, SizeOf(type)))
      return -1;
  StepFactors a;
  a.state = *state;
  a.lr = static_cast<float>(step->lr);
  a.beta1 = static_cast<float>(step->beta1), a.one_minus_beta1 = static_cast<float>(1.0 - step->beta1);
  a.beta2 = static_cast<float>(step->beta2), a.one_minus_beta2 = static_cast<float>(1.0 - step->beta2);
  a.log_beta1 = static_cast<float>(log(step->beta1)), a.log_beta2 = static_cast<float>(log(step->beta2));
  a.eps = static_cast<float>(step->eps), a.decay = static_cast<float>(step->decay);
  a.minus_zero = -0.f;
  a.max_norm = step->max_norm, a.lr_tensor = step->lr_tensor, a.norm = step->norm;
  a.tile_blocks = TileBlocks(tensors, count, state->bits);
  if (count <= kFewTensors) return Step<kFewTensors>(tensors, count, a, type, static_cast<cudaStream_t>(stream));
  return Step<kMaxTensors>(tensors, count, a, type, static_cast<cudaStream_t>(stream));
}

extern "C" int switchml_adamw_masters(const SmlAdamwTensor* tensors, int count, const short* remainder, float* out, int type, void* stream) {
  if (!tensors || count < 0 || !out || (type != SML_ADAMW_F32 && (type != SML_ADAMW_BF16 || !remainder)) || !At(out, 32) || !At(remainder, 16))
    return -1;
  for (int i = 0; i < count; i++)
    if (tensors[i].numel < 0 || tensors[i].numel > kMaxNumel || (tensors[i].numel && !tensors[i].param) || !At(tensors[i].param, SizeOf(type)))
      return -1;
  if (count <= kFewTensors) return Masters<kFewTensors>(tensors, count, remainder, out, type, static_cast<cudaStream_t>(stream));
  return Masters<kMaxTensors>(tensors, count, remainder, out, type, static_cast<cudaStream_t>(stream));
}

extern "C" long long switchml_grad_norm_workspace(int count) {
  return (count <= 0 ? 1ll : static_cast<long long>((count + kMaxTensors - 1) / kMaxTensors)) * kNormBlocks;
}

extern "C" int switchml_grad_norm(const SmlNormTensor* tensors, int count, double* workspace, int* ticket, float* out, void* stream) {
  if (count < 0 || !out || !workspace || (count && !tensors) || !At(out, 4) || !At(workspace, 8) || !At(ticket, 4)) return -1;
  long long tiles = 0;  // (as many as a launch takes: the workspace is for launches that end with their table of tensors)
  for (int i = 0; i < count; i++) {
    if (tensors[i].numel < 0 || tensors[i].numel > kMaxNumel || (tensors[i].numel && !tensors[i].data) ||
        (tensors[i].type != SML_ADAMW_F32 && tensors[i].type != SML_ADAMW_BF16) || !At(tensors[i].data, SizeOf(tensors[i].type)))
      return -1;
    tiles += (tensors[i].numel + kNormTile - 1) / kNormTile;
    if (tiles > kMaxTiles) return -1;
  }
  if (count <= kFewTensors) return GradNorm<kFewTensors>(tensors, count, workspace, ticket, out, static_cast<cudaStream_t>(stream));
  return GradNorm<kMaxTensors>(tensors, count, workspace, ticket, out, static_cast<cudaStream_t>(stream));
}

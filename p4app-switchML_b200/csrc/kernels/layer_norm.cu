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

#include <type_traits>

#include "kernels/dependent_launch.cuh"
#include "kernels/layer_norm.h"
#include "kernels/packed.cuh"

using switchml::kernels::Fma;
using switchml::kernels::LaunchOverlapped;
using switchml::kernels::LetNextKernelStart;
using switchml::kernels::LoadWords;
using switchml::kernels::Pair;
using switchml::kernels::StoreWords;
using switchml::kernels::Sum;
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

// ---- rows that stay in registers ----
//
// A group of threads holds a row: 8 lanes of a warp, 1 to 24 whole warps, or 16 warps of each of 2, 4 or 8 blocks of a cluster. Each
// lane has kHeld values in vectors of kVec neighbours, between which lie kLanes (8 or 32) * kVec values, so that addresses
// differ by constants; warp w has the values from w * 32 * kHeld on. kVec is what the addresses and the length of the rows
// allow: 16 bytes of them, 2, or 1, of which two that are kLanes apart make a vector. Groups go through their rows by
// themselves, and warps of a group meet at a barrier of their own.

// Whether a warp looks if all its columns exist, to leave out the questions where they do. Single values ask twice as often as
// vectors (forward and backward, bf16, with and without: 20000 x 5001 220 and 236, 298 and 311 us; 16384 x 2047 71 and 72, 101 and
// 106; the one loss found is 16384 x 2047 fp32, backward, 110 and 99), and in a cluster's long rows most warps are whole (backward,
// 8192 x 12000 fp32: 416 and 470). Elsewhere the second copy of the code costs more (16384 x 2046 bf16, forward: 61 and 55).
__host__ __device__ constexpr bool WarpAsks(int vec, bool split) { return vec == 1 || split; }

__device__ __forceinline__ uint32_t SharedAddress(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

template <int kLanes, bool kSplit> struct Group {  // kSplit: over the blocks of a cluster
  // number: in the block; warps: of a group in a block; ranks: blocks of a group; lane, warp: in the group
  int number, warps, ranks, lane, warp;
  unsigned mask;
  __device__ __forceinline__ Group(int warps_of_group, int blocks_of_group) : warps(warps_of_group), ranks(kSplit ? blocks_of_group : 1) {
    const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
    lane = l % kLanes;
    mask = kLanes == 32 ? 0xffffffffu : ((1u << kLanes % 32) - 1) << (l - lane);
    number = kLanes == 32 ? w / warps : threadIdx.x / kLanes;
    warp = kLanes == 32 ? w - number * warps + Rank() * warps : 0;
  }
  // Of this block among those of the group.
  __device__ __forceinline__ int Rank() const { return kSplit ? static_cast<int>(blockIdx.x) % ranks : 0; }
  // The first value of this thread's.
  __device__ __forceinline__ int First(int held, int vec) const { return warp * 32 * held + lane * vec; }
  // Whether all values of this warp's exist in a row of n.
  __device__ __forceinline__ bool Whole(int held, int n) const { return kLanes == 32 && (warp + 1) * 32 * held <= n; }
  // Row of the first turn, and the distance to the next.
  __device__ __forceinline__ long long FirstRow(int groups) const {
    return static_cast<long long>(kSplit ? blockIdx.x / ranks : blockIdx.x) * groups + number;
  }
  __device__ __forceinline__ long long Stride(int groups) const {
    return static_cast<long long>(kSplit ? gridDim.x / ranks : gridDim.x) * groups;
  }
  // Before the first Sum: the blocks of a group are there.
  __device__ __forceinline__ void Meet() const {
    if constexpr (kSplit) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  // The sum over the group, in all its threads. Two calls that follow each other take different `part`s (a V for each warp
  // of the block) and `across` (a float2 for each block): between two uses of the same one lies the other's barrier.
  template <class V> __device__ __forceinline__ V Sum(V v, V* part, float2* across) const {
#pragma unroll
    for (int o = kLanes / 2; o; o >>= 1) v = Plus(v, Shuffle(v, o));
    if (kLanes == 32 && warps > 1) {
      const int first = number * warps;
      if (lane == 0) part[threadIdx.x >> 5] = v;
      __syncwarp();  // (bar.sync wants the warp's threads together)
      asm volatile("bar.sync %0, %1;" ::"r"(number + 1), "r"(warps * 32) : "memory");
      v = lane < warps ? part[first + lane] : V{};
      for (int o = warps > 16 ? 16 : warps > 8 ? 8 : warps > 4 ? 4 : warps > 2 ? 2 : 1; o; o >>= 1) v = Plus(v, Shuffle(v, o));
      v = Broadcast(v);
      if constexpr (kSplit) {
        if (threadIdx.x < ranks) {  // thread r tells block r
          const uint32_t mine = SharedAddress(across + Rank());
          const float2 both = Both(v);
          uint32_t to;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(mine), "r"(threadIdx.x));
          asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(both.x), "f"(both.y) : "memory");
        }
        __syncwarp();
        Meet();
        float2 all = make_float2(0.f, 0.f);
        for (int r = 0; r < ranks; r++) all = Plus(all, across[r]);
        Set(all, &v);
      }
    }
    return v;
  }
  __device__ __forceinline__ float Shuffle(float v, int o) const { return __shfl_xor_sync(mask, v, o); }
  __device__ __forceinline__ float2 Shuffle(float2 v, int o) const { return make_float2(Shuffle(v.x, o), Shuffle(v.y, o)); }
  __device__ __forceinline__ float Broadcast(float v) const { return __shfl_sync(mask, v, 0); }
  __device__ __forceinline__ float2 Broadcast(float2 v) const { return make_float2(Broadcast(v.x), Broadcast(v.y)); }
  static __device__ __forceinline__ float Plus(float a, float b) { return a + b; }
  static __device__ __forceinline__ float2 Plus(float2 a, float2 b) { return make_float2(a.x + b.x, a.y + b.y); }
  static __device__ __forceinline__ float2 Both(float v) { return make_float2(v, 0.f); }
  static __device__ __forceinline__ float2 Both(float2 v) { return v; }
  static __device__ __forceinline__ void Set(float2 from, float* to) { *to = from.x; }
  static __device__ __forceinline__ void Set(float2 from, float2* to) { *to = from; }
};

// Values of 16 bytes: what a thread reads at once where addresses and the length of the rows allow it.
template <class T> constexpr int kWide = 16 / sizeof(T);

// Pairs of values of type T in registers, as they lie in memory: kVec neighbours, or with kVec = 1 two values that are kLanes apart.
// `left`: columns from the vector's first one to the end of the row.
template <class T, int kVec, int kLanes> struct Vector {
  static constexpr int kNums = kVec == 1 ? 1 : kVec / 2;        // pairs
  static constexpr int kStep = kLanes * (kVec == 1 ? 2 : kVec);  // columns from one of a thread's vectors to the next
  static constexpr int kWords = kNums * 2 * sizeof(T) / 4;
  unsigned w[kWords];
  __device__ __forceinline__ void Load(const T* from) {
    if constexpr (kVec > 1) LoadWords(from, w);
    else LoadSome(from, 2 * kLanes);
  }
  __device__ __forceinline__ void LoadSome(const T* from, int left) {  // zeros where nothing is there
    if constexpr (kVec > 1) {
      switchml::kernels::LoadWordsIf(left, from, w);
    } else if constexpr (sizeof(T) == 4) {
      unsigned x[1], y[1];
      switchml::kernels::LoadWordsIf(left, from, x);
      switchml::kernels::LoadWordsIf(left - kLanes, from + kLanes, y);
      w[0] = x[0], w[1] = y[0];
    } else {
      asm volatile("{.reg .pred p, q; .reg .b16 x, y; mov.b16 x, 0; mov.b16 y, 0; setp.gt.s32 p, %2, 0; setp.gt.s32 q, %2, %3;"
                   "@p ld.global.b16 x, [%1]; @q ld.global.b16 y, [%1 + %4]; mov.b32 %0, {x, y};}"
                   : "=r"(w[0]) : "l"(from), "r"(left), "n"(kLanes), "n"(kLanes * 2));
    }
  }
  template <bool kWhole> __device__ __forceinline__ void Store(T* to, int left) const {
    if constexpr (kVec > 1) {
      if (kWhole || left > 0) StoreWords(to, w);
    } else {
      if constexpr (sizeof(T) == 4) {
        if (kWhole || left > 0) *reinterpret_cast<unsigned*>(to) = w[0];
        if (kWhole || left > kLanes) *reinterpret_cast<unsigned*>(to + kLanes) = w[1];
      } else {
        if (kWhole || left > 0) *reinterpret_cast<unsigned short*>(to) = static_cast<unsigned short>(w[0]);
        if (kWhole || left > kLanes) *reinterpret_cast<unsigned short*>(to + kLanes) = static_cast<unsigned short>(w[0] >> 16);
      }
    }
  }
  __device__ __forceinline__ void LoadShared(const uint4* from) {  // 16 bytes
    const uint4 v = *from;
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  }
  __device__ __forceinline__ Pair At(int i) const {
    if constexpr (sizeof(T) == 4) return Pair(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else return Pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  __device__ __forceinline__ void Set(int i, Pair v) {
    const float2 both = v.Both();
    if constexpr (sizeof(T) == 4) {
      w[2 * i] = __float_as_uint(both.x), w[2 * i + 1] = __float_as_uint(both.y);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(both.x, both.y);
      w[i] = *reinterpret_cast<const unsigned*>(&h);
    }
  }
  // A pair of which what does not exist is 0.
  template <bool kWhole> static __device__ __forceinline__ Pair There(Pair v, int left) {
    if constexpr (kWhole || kVec > 1) return v;  // (vectors of neighbours exist or do not)
    const float2 both = v.Both();
    return Pair(both.x, left > kLanes ? both.y : 0.f);
  }
};

// Weight or bias of a vector's columns. W: their type where that is known (and both are there), else void. (To find out for every
// vector which of three values it is costs as much as the rest of the forward pass.)
template <int kVec, int kLanes, bool kWhole, class W>
__device__ __forceinline__ void LoadParameter(const Parameter& p, int i, int left, float none, Pair (&out)[Vector<float, kVec, kLanes>::kNums]) {
  constexpr int kNums = Vector<float, kVec, kLanes>::kNums;
  const auto load = [&](auto type) {
    Vector<decltype(type), kVec, kLanes> v;
    const auto* from = static_cast<const decltype(type)*>(p.data) + i;
    if constexpr (kWhole) v.Load(from);
    else v.LoadSome(from, left);
#pragma unroll
    for (int k = 0; k < kNums; k++) out[k] = v.At(k);
  };
  if constexpr (!std::is_void_v<W>) {
    load(W{});
  } else if (!p.data) {
#pragma unroll
    for (int k = 0; k < kNums; k++) out[k] = Pair(none);
  } else if (p.type == SML_NORM_F32) {
    load(float{});
  } else {
    load(__nv_bfloat16{});
  }
}

// One pass: a row is read once, statistics and result come out of registers. Bound by memory: 16384 x 8192 bf16 with a residual,
// 1.07 GB, 162 us = 6.6 TB/s; 8192 x 1024, 67 MB, 13.3 us, where a copy of as many bytes takes 12.2 (most of the difference is
// that 8192 rows make 1.7 times the warps that the GPU holds). Rows at odd addresses take a load per value: 4099 x 1021, 34 MB,
// 12 us, 16384 x 2047, 268 MB, 71 us. Rows of a cluster: 8192 x 12000 fp32 396 us (read three times by a block each: 588).
// 32 bf16 values per lane instead of 16 save half the sums over lanes (8192 x 4096: 45 instead of 57 us); 16 fp32 values are
// as many bytes.
//
// Values that a thread holds. kWhole: the row is exactly what its threads hold.
__host__ __device__ constexpr int ForwardHeld(int vec, int size) { return vec == 8 ? 32 : 16; }

template <class T, int kVec, int kLanes, bool kWhole, bool kSplit, class W>
__device__ __forceinline__ void ForwardRows(const T* x, const T* residual, const Parameter& weight, const Parameter& bias, T* y, T* sum,
                                            float* mean_out, float* rstd_out, long long rows, int n, float eps, int groups,
                                            const Group<kLanes, kSplit>& group, float (*part)[16], float2 (*across)[8]) {
  using V = Vector<T, kVec, kLanes>;
  constexpr int kHeld = ForwardHeld(kVec, sizeof(T)), kNums = V::kNums, kVectors = kHeld / (2 * kNums), kStep = V::kStep;
  const int column = group.First(kHeld, kVec), left = n - column;
  for (long long row = group.FirstRow(groups), stride = group.Stride(groups); row < rows; row += stride) {
    const long long at = row * n + column;
    Pair s[kVectors][kNums];
    {
      V raw[kVectors], more[kVectors];
#pragma unroll
      for (int j = 0; j < kVectors; j++) {
        if constexpr (kWhole) raw[j].Load(x + at + j * kStep);
        else raw[j].LoadSome(x + at + j * kStep, left - j * kStep);
      }
      if (residual) {
#pragma unroll
        for (int j = 0; j < kVectors; j++) {
          if constexpr (kWhole) more[j].Load(residual + at + j * kStep);
          else more[j].LoadSome(residual + at + j * kStep, left - j * kStep);
        }
#pragma unroll
        for (int j = 0; j < kVectors; j++) {
#pragma unroll
          for (int i = 0; i < kNums; i++) raw[j].Set(i, raw[j].At(i) + more[j].At(i));
          raw[j].template Store<kWhole>(sum + at + j * kStep, left - j * kStep);
        }
      }
#pragma unroll
      for (int j = 0; j < kVectors; j++) {
#pragma unroll
        for (int i = 0; i < kNums; i++) s[j][i] = raw[j].At(i);
      }
    }
    Pair total(0.f);
#pragma unroll
    for (int j = 0; j < kVectors; j++) {
#pragma unroll
      for (int i = 0; i < kNums; i++) total = total + s[j][i];
    }
    const float mean = group.Sum(Sum(total), part[0], across[0]) / n;
    Pair squares(0.f);
#pragma unroll
    for (int j = 0; j < kVectors; j++) {
      if (!kWhole && j * kStep >= left) continue;
#pragma unroll
      for (int i = 0; i < kNums; i++) {
        s[j][i] = V::template There<kWhole>(s[j][i] + Pair(-mean), left - j * kStep);
        squares = Fma(s[j][i], s[j][i], squares);
      }
    }
    const float rstd = 1.f / sqrtf(group.Sum(Sum(squares), part[1], across[1]) / n + eps);
#pragma unroll
    for (int j = 0; j < kVectors; j++) {
      if (!kWhole && j * kStep >= left) continue;
      Pair w[kNums], b[kNums];
      LoadParameter<kVec, kLanes, kWhole, W>(weight, column + j * kStep, left - j * kStep, 1.f, w);
      LoadParameter<kVec, kLanes, kWhole, W>(bias, column + j * kStep, left - j * kStep, 0.f, b);
      V out;
#pragma unroll
      for (int i = 0; i < kNums; i++) out.Set(i, Fma(s[j][i] * Pair(rstd), w[i], b[i]));
      out.template Store<kWhole>(y + at + j * kStep, left - j * kStep);
    }
    if (column == 0 && mean_out) mean_out[row] = mean, rstd_out[row] = rstd;
  }
}

template <class T, int kVec, int kLanes, bool kWhole, bool kSplit, class W>
__global__ void __launch_bounds__(512, 2)
ForwardKernel(const T* x, const T* residual, Parameter weight, Parameter bias, T* y, T* sum, float* mean_out, float* rstd_out,
              long long rows, int n, float eps, int groups, int warps, int ranks) {
  __shared__ float part[2][16];
  __shared__ float2 across[2][8];
  const Group<kLanes, kSplit> group(warps, ranks);
  WaitForEarlierKernels();
  group.Meet();
  if (kWhole || (WarpAsks(kVec, kSplit) && group.Whole(ForwardHeld(kVec, sizeof(T)), n)))
    ForwardRows<T, kVec, kLanes, true, kSplit, W>(x, residual, weight, bias, y, sum, mean_out, rstd_out, rows, n, eps, groups, group, part, across);
  else
    ForwardRows<T, kVec, kLanes, false, kSplit, W>(x, residual, weight, bias, y, sum, mean_out, rstd_out, rows, n, eps, groups, group, part, across);
}

// The backward pass of rows that a group holds, and the sums over the rows that each block saw, in the order of the groups.
// A block per SM goes through the rows; a group reads its next rows while it deals with one, so that the sums of weight and
// bias stay in registers and only 148 partial ones meet. Bound by memory: 16384 x 8192 bf16 with the sum's gradient, 1.07 GB,
// 165 us = 6.5 TB/s with the closing sums; on short inputs by its ends (8192 x 1024, 50 MB, 14.8 us: 7 rounds of rows, then 8
// groups' sums). Single values: 16384 x 2047 99 us. Rows of a cluster: 8192 x 12000 255 us (one pass for the input's gradient and
// one for the columns: 539).
// Sums, normalised values, gradients and what is read ahead take 6 to 8 registers per value: 16 bf16 values in vectors fit
// the 128 registers of 16 warps, of the others 8 fit the 85 of 24 warps. (Of 16 of those, for rows that need them, most spill.)
__host__ __device__ constexpr int BackwardThreads(int held) { return held == 16 ? 512 : 768; }
int BackwardHeld(int n, int vec) { return (vec == 8 && n > 256) || n > BackwardThreads(8) * 8 ? 16 : 8; }

// Rows that a thread reads ahead, in vectors: through shared memory, where it alone reads what it has copied itself, so that
// nothing has to be waited for but its own copies. (Registers hold one row: 8192 x 1024 fp32 25.4 us with those.)
__host__ __device__ constexpr int BackwardRowBytes(int held, int size) { return 3 * held * size * BackwardThreads(held); }  // of dy, s and dsum
__host__ __device__ constexpr int BackwardStages(int vec, int held, int size) {
  return vec * size < 16 ? 0 : 216 * 1024 / BackwardRowBytes(held, size) < 4 ? 216 * 1024 / BackwardRowBytes(held, size) : 4;
}

__device__ __forceinline__ void CopyAsync(uint4* to, const void* from, bool there) {  // zeros where nothing is there
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(SharedAddress(to)), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void CommitCopies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void WaitForCopies() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

// The sums over rows that a thread keeps, of its columns.
template <int kPairs> struct ColumnSums {
  Pair dw[kPairs], db[kPairs];
};

template <class T, int kVec, int kLanes, bool kWhole, bool kSplit, int kHeld, class W>
__device__ __forceinline__ void BackwardRows(const T* dy, const T* dsum, const T* s, const Parameter& weight, const float* mean_in,
                                             const float* rstd_in, T* dx, long long rows, int n, int groups, const Group<kLanes, kSplit>& group,
                                             float2 (*part)[BackwardThreads(kHeld) / 32], float2 (*across)[8], uint4* ring,
                                             ColumnSums<kHeld / 2>* sums) {
  using V = Vector<T, kVec, kLanes>;
  constexpr int kNums = V::kNums, kVectors = kHeld / (2 * kNums), kStep = V::kStep;
  const int column = group.First(kHeld, kVec), left = n - column;
  const long long stride = group.Stride(groups);
  // The weight stays in registers where these suffice, else it comes from L1 for every row.
  constexpr bool kKeepWeight = sizeof(T) == 2 && kVec > 1;
  Pair w[kVectors][kNums];
  if constexpr (kKeepWeight) {
#pragma unroll
    for (int j = 0; j < kVectors; j++) {
      if (kWhole || j * kStep < left) LoadParameter<kVec, kLanes, kWhole, W>(weight, column + j * kStep, left - j * kStep, 1.f, w[j]);
    }
  }
  V d[kVectors], v[kVectors], more[kVectors];
  float mean = 0.f, rstd = 0.f;
  const auto load = [&](const T* from, V(&to)[kVectors]) {
#pragma unroll
    for (int j = 0; j < kVectors; j++) {
      if constexpr (kWhole) to[j].Load(from + j * kStep);
      else to[j].LoadSome(from + j * kStep, left - j * kStep);
    }
  };
  // The ring: kStages rows of kVectors vectors of dy, s and, if there is one, dsum for every thread.
  constexpr int kStages = BackwardStages(kVec, kHeld, sizeof(T)), kThreads = BackwardThreads(kHeld);
  const auto copy = [&](long long row, int stage) {
    if (row < rows) {
      const long long at = row * n + column;
      uint4* const to = ring + stage * 3 * kVectors * kThreads;
#pragma unroll
      for (int j = 0; j < kVectors; j++) {
        const bool there = kWhole || j * kStep < left;
        const long long from = there ? at + j * kStep : 0;
        CopyAsync(to + j * kThreads, dy + from, there);
        CopyAsync(to + (kVectors + j) * kThreads, s + from, there);
        if (dsum) CopyAsync(to + (2 * kVectors + j) * kThreads, dsum + from, there);
      }
    }
    CommitCopies();
  };
  // (Groups that do not fit into the block any more have no row.)
  long long row = group.number < groups ? group.FirstRow(groups) : rows;
  if constexpr (kStages > 0) {
#pragma unroll
    for (int i = 0; i < kStages - 1; i++) copy(row + i * stride, i);
  } else if (row < rows) {
    load(dy + row * n + column, d);
    load(s + row * n + column, v);
  }
  if (row < rows) mean = mean_in[row], rstd = rstd_in[row];
  int turn = 0, stage = 0;
  for (; row < rows; row += stride) {
    const long long at = row * n + column;
    const float r = rstd;
    if constexpr (kStages > 0) {
      copy(row + (kStages - 1) * stride, stage ? stage - 1 : kStages - 1);
      WaitForCopies<kStages - 1>();
      const uint4* const from = ring + stage * 3 * kVectors * kThreads;
#pragma unroll
      for (int j = 0; j < kVectors; j++) {
        d[j].LoadShared(from + j * kThreads);
        v[j].LoadShared(from + (kVectors + j) * kThreads);
      }
    }
    Pair c1(0.f), c2(0.f), xhat[kVectors][kNums], g[kVectors][kNums];
#pragma unroll
    for (int j = 0; j < kVectors; j++) {
      if (!kWhole && j * kStep >= left) continue;  // (what is not there has gradients of 0, but 0 times infinity is NaN)
      if constexpr (!kKeepWeight) LoadParameter<kVec, kLanes, kWhole, W>(weight, column + j * kStep, left - j * kStep, 1.f, w[j]);
#pragma unroll
      for (int i = 0; i < kNums; i++) {
        const Pair dyi = d[j].At(i);
        xhat[j][i] = V::template There<kWhole>((v[j].At(i) + Pair(-mean)) * Pair(r), left - j * kStep);
        g[j][i] = dyi * w[j][i];
        c1 = c1 + g[j][i];
        c2 = Fma(g[j][i], xhat[j][i], c2);
        sums->dw[j * kNums + i] = Fma(dyi, xhat[j][i], sums->dw[j * kNums + i]);
        sums->db[j * kNums + i] = sums->db[j * kNums + i] + dyi;
      }
    }
    if constexpr (kStages == 0) {
      if (dsum) load(dsum + at, more);
      if (row + stride < rows) {
        load(dy + at + stride * n, d);
        load(s + at + stride * n, v);
      }
    }
    if (row + stride < rows) mean = mean_in[row + stride], rstd = rstd_in[row + stride];
    const float2 c12 = group.Sum(make_float2(Sum(c1), Sum(c2)), part[turn], across[turn]);
    turn ^= 1;
    const Pair minus_c1(-c12.x / n), minus_c2(-c12.y / n);
    const auto store = [&](auto plus) {
#pragma unroll
      for (int j = 0; j < kVectors; j++) {
        if (!kWhole && j * kStep >= left) continue;
        V out;
#pragma unroll
        for (int i = 0; i < kNums; i++) out.Set(i, plus(Fma(xhat[j][i], minus_c2, g[j][i] + minus_c1) * Pair(r), j, i));
        out.template Store<kWhole>(dx + at + j * kStep, left - j * kStep);
      }
    };
    if (dsum) {
      if constexpr (kStages > 0) {
#pragma unroll
        for (int j = 0; j < kVectors; j++) more[j].LoadShared(ring + (stage * 3 * kVectors + 2 * kVectors + j) * kThreads);
      }
      store([&](Pair e, int j, int i) { return e + more[j].At(i); });
    } else {
      store([](Pair e, int, int) { return e; });
    }
    stage = stage + 1 < kStages ? stage + 1 : 0;
  }
}

template <class T, int kVec, int kLanes, bool kWhole, bool kSplit, int kHeld, class W>
__global__ void __launch_bounds__(BackwardThreads(kHeld), 1)
BackwardKernel(const T* dy, const T* dsum, const T* s, Parameter weight, const float* mean, const float* rstd, T* dx,
               float* workspace, long long rows, int n, int groups, int warps, int ranks) {
  using V = Vector<T, kVec, kLanes>;
  extern __shared__ __align__(16) unsigned char shared[];
  __shared__ float2 part[2][BackwardThreads(kHeld) / 32];
  __shared__ float2 across[2][8];
  const Group<kLanes, kSplit> group(warps, ranks);
  uint4* const ring = reinterpret_cast<uint4*>(shared) + threadIdx.x;
  ColumnSums<kHeld / 2> sums;
#pragma unroll
  for (int i = 0; i < kHeld / 2; i++) sums.dw[i] = sums.db[i] = Pair(0.f);
  WaitForEarlierKernels();
  group.Meet();
  if (kWhole || (WarpAsks(kVec, kSplit) && group.Whole(kHeld, n)))
    BackwardRows<T, kVec, kLanes, true, kSplit, kHeld, W>(dy, dsum, s, weight, mean, rstd, dx, rows, n, groups, group, part, across, ring, &sums);
  else
    BackwardRows<T, kVec, kLanes, false, kSplit, kHeld, W>(dy, dsum, s, weight, mean, rstd, dx, rows, n, groups, group, part, across, ring, &sums);
  if (!workspace) return;
  LetNextKernelStart();  // (what finishes the sums)
  // The upper half of the groups gives its sums to the lower one until one has all. (In the ring's place, after a barrier: no
  // thread has copies under way that are for rows, and what it has of empty ones counts for nothing.)
  Pair* const given = reinterpret_cast<Pair*>(shared);
  const int width = kLanes == 32 ? warps * 32 : kLanes;
  const int t = kLanes == 32 ? static_cast<int>(threadIdx.x) - group.number * width : group.lane;
  for (int there = groups; there > 1;) {
    const int half = (there + 1) / 2;
    __syncthreads();
    if (group.number >= half && group.number < there) {
#pragma unroll
      for (int i = 0; i < kHeld / 2; i++) {
        given[(2 * i * half + group.number - half) * width + t] = sums.dw[i];
        given[((2 * i + 1) * half + group.number - half) * width + t] = sums.db[i];
      }
    }
    __syncthreads();
    if (group.number < there - half) {
#pragma unroll
      for (int i = 0; i < kHeld / 2; i++) {
        sums.dw[i] = sums.dw[i] + given[(2 * i * half + group.number) * width + t];
        sums.db[i] = sums.db[i] + given[((2 * i + 1) * half + group.number) * width + t];
      }
    }
    there = half;
  }
  if (group.number) return;
  const int column = group.First(kHeld, kVec);
  float* const out = workspace + static_cast<long long>(kSplit ? blockIdx.x / ranks : blockIdx.x) * 2 * n;
#pragma unroll
  for (int i = 0; i < kHeld / 2; i++) {
    const int c = column + i / V::kNums * V::kStep + i % V::kNums * 2;
    if constexpr (kVec > 1) {  // (n is even)
      if (c < n) *reinterpret_cast<Pair*>(out + c) = sums.dw[i], *reinterpret_cast<Pair*>(out + n + c) = sums.db[i];
    } else {
      const float2 dw = sums.dw[i].Both(), db = sums.db[i].Both();
      if (c < n) out[c] = dw.x, out[n + c] = db.x;
      if (c + kLanes < n) out[c + kLanes] = dw.y, out[n + c + kLanes] = db.y;
    }
  }
}

// ---- rows of any length ----

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

// Sums over rows: a block takes 32 columns, a warp every 8th row of them. Rows that no cluster holds have more than 65536 values, so
// there are more than 2048 blocks, and shares of the rows would find no SM free. A thread reads four rows before it adds one (4000 x
// 70001, the whole backward pass: 1626 us in fp32 and 1350 in bf16; eight 1668 and 1439, a plain loop that the compiler unrolls 1706
// to 1944 and 1458 to 1714).
template <class T>
__global__ void __launch_bounds__(kAnyThreads)
ColumnsAnyKernel(const T* dy, const T* s, const float* mean, const float* rstd, float* workspace, long long rows, int n) {
  __shared__ float2 part[kAnyThreads / 32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, column = blockIdx.x * 32 + lane;
  float dw = 0.f, db = 0.f;
  WaitForEarlierKernels();
  if (column < n) {
    const auto add = [&](T g, T v, long long row) {
      dw += ToFloat(g) * ((ToFloat(v) - mean[row]) * rstd[row]);
      db += ToFloat(g);
    };
    constexpr int kRows = 4, kStep = kAnyThreads / 32;
    long long row = warp;
    for (; row + (kRows - 1) * kStep < rows; row += kRows * kStep) {
      T g[kRows], v[kRows];
#pragma unroll
      for (int i = 0; i < kRows; i++) g[i] = dy[(row + i * kStep) * n + column], v[i] = s[(row + i * kStep) * n + column];
#pragma unroll
      for (int i = 0; i < kRows; i++) add(g[i], v[i], row + i * kStep);
    }
    for (; row < rows; row += kStep) add(dy[row * n + column], s[row * n + column], row);
  }
  part[warp][lane] = make_float2(dw, db);
  __syncthreads();
  if (warp == 0 && column < n) {
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kAnyThreads / 32; w++) sum.x += part[w][lane].x, sum.y += part[w][lane].y;
    workspace[column] = sum.x;
    workspace[n + column] = sum.y;
  }
}

// The sums of `parts` partial sums, in a fixed order. A block takes 8 columns (a 32-byte sector of each part), a warp 4 parts at
// a time: with 148 parts every thread has all its loads in flight at once.
constexpr int kFinishColumns = 8, kFinishThreads = 256, kFinishParts = kFinishThreads / kFinishColumns;

__global__ void __launch_bounds__(kFinishThreads)
FinishColumnsKernel(const float* workspace, void* dweight, void* dbias, int parts, int n, int wtype) {
  __shared__ float2 part[kFinishThreads / 32][kFinishColumns];
  const int c = threadIdx.x % kFinishColumns, column = blockIdx.x * kFinishColumns + c;
  float2 sum = make_float2(0.f, 0.f);
  WaitForEarlierKernels();
  if (column < n) {
#pragma unroll 5
    for (int p = threadIdx.x / kFinishColumns; p < parts; p += kFinishParts) {
      const float* from = workspace + static_cast<long long>(p) * 2 * n;
      sum.x += from[column];
      sum.y += from[n + column];
    }
  }
#pragma unroll
  for (int o = kFinishColumns; o < 32; o *= 2) {
    sum.x += __shfl_xor_sync(0xffffffffu, sum.x, o);
    sum.y += __shfl_xor_sync(0xffffffffu, sum.y, o);
  }
  if (threadIdx.x % 32 < kFinishColumns) part[threadIdx.x / 32][c] = sum;
  __syncthreads();
  if (threadIdx.x >= kFinishColumns || column >= n) return;
  sum = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kFinishThreads / 32; i++) sum.x += part[i][c].x, sum.y += part[i][c].y;
  if (wtype == SML_NORM_F32) {
    if (dweight) static_cast<float*>(dweight)[column] = sum.x;
    if (dbias) static_cast<float*>(dbias)[column] = sum.y;
  } else {
    if (dweight) static_cast<__nv_bfloat16*>(dweight)[column] = __float2bfloat16_rn(sum.x);
    if (dbias) static_cast<__nv_bfloat16*>(dbias)[column] = __float2bfloat16_rn(sum.y);
  }
}

unsigned RowBlocks(long long rows) { return static_cast<unsigned>(rows < (1 << 20) ? rows : (1 << 20)); }

// Columns are counted in 32 bits, beyond a row's end too.
bool Fits(int features) { return features > 0 && features <= 1 << 30; }

// Whether all of them lie at multiples of their element, a power of two (null does).
template <class... Pointers> bool Aligned(unsigned size, Pointers... p) { return ((reinterpret_cast<uintptr_t>(p) | ...) & (size - 1)) == 0; }
unsigned SizeOf(int type) { return type == SML_NORM_F32 ? 4 : 2; }

bool Known(int type) { return type == SML_NORM_F32 || type == SML_NORM_BF16; }

// Values that are read and written at once: what the length of the rows and all addresses allow.
struct Alignment {
  uintptr_t bits = 0;
  template <class T> void Of(const T* tensor) { bits |= reinterpret_cast<uintptr_t>(tensor) * (4 / sizeof(T)); }  // as if it were fp32
  void Of(const Parameter& p) { bits |= reinterpret_cast<uintptr_t>(p.data) * (p.type == SML_NORM_F32 ? 1 : 2); }
  int Vec(int n, int wide) const { return n % wide == 0 && bits % (4 * wide) == 0 ? wide : n % 2 == 0 && bits % 8 == 0 ? 2 : 1; }
};

// How rows of n values are held by groups of a block of up to `warps` warps, with `held` values per lane.
struct Geometry {
  // lanes = 0: the rows are too long; warps: of a group in a block; groups: of a block; ranks: blocks of a group; parts: blocks / ranks
  int lanes = 0, warps = 0, groups = 0, ranks = 1, parts = 0;
  bool whole = false;
  Geometry(long long rows, int n, int held, int block_warps, int most_warps, int most_blocks) {
    while (n > ranks * most_warps * 32 * held) {
      if (ranks == 8) return;
      ranks *= 2;
    }
    lanes = n <= 8 * held ? 8 : 32;
    warps = lanes == 8 ? 1 : ranks > 1 ? most_warps : (n - 1) / (32 * held) + 1;
    if (block_warps % warps && block_warps < 16) block_warps = 16;  // (a block reserves all barriers: 4 of them to an SM)
    groups = lanes == 8 ? block_warps * 4 : block_warps / warps > 0 ? block_warps / warps : 1;
    whole = n == ranks * warps * 32 * held && lanes == 32;
    const long long wanted = (rows + groups - 1) / groups;
    parts = static_cast<int>(wanted < most_blocks / ranks ? wanted : most_blocks / ranks);
  }
  unsigned Blocks() const { return static_cast<unsigned>(parts) * ranks; }
  int Threads() const { return lanes == 8 ? groups * 8 : groups * warps * 32; }
};

constexpr int kSms = 148;  // of a B200
constexpr int kForwardWarps = 8;  // of a block, where a row does not need more

Geometry BackwardGeometry(long long rows, int n, int held) {
  const int warps = BackwardThreads(held) / 32;
  return Geometry(rows, n, held, warps, warps, kSms);
}

// The type of weight and bias, for kernels that want to know it.
enum class Kind { kF32, kBf16, kNo };
template <class T> Kind TypeOf(const Parameter& a, const Parameter& b) {
  if (!a.data || !b.data || (sizeof(T) == 4 && a.type != SML_NORM_F32)) return Kind::kNo;
  return a.type == SML_NORM_F32 ? Kind::kF32 : Kind::kBf16;
}

template <class T, int kVec, int kLanes, bool kSplit, int kHeld> auto BackwardKernelOf(Kind type) {
  return type == Kind::kF32 ? BackwardKernel<T, kVec, kLanes, false, kSplit, kHeld, float>
                            : BackwardKernel<T, kVec, kLanes, false, kSplit, kHeld, void>;
}
template <class T, int kHeld> auto BackwardKernelOf(const Geometry& g, int vec, Kind type) {
  if constexpr (kHeld == 8) {  // (the others are for longer rows)
    if (g.lanes == 8)
      return vec == 1 ? BackwardKernelOf<T, 1, 8, false, kHeld>(type) : vec == 2 ? BackwardKernelOf<T, 2, 8, false, kHeld>(type)
             : BackwardKernelOf<T, kWide<T>, 8, false, kHeld>(type);
  } else {
    if (g.ranks > 1)
      return vec == 1 ? BackwardKernelOf<T, 1, 32, true, kHeld>(type) : vec == 2 ? BackwardKernelOf<T, 2, 32, true, kHeld>(type)
             : BackwardKernelOf<T, kWide<T>, 32, true, kHeld>(type);
  }
  if (vec <= 2) return vec == 1 ? BackwardKernelOf<T, 1, 32, false, kHeld>(type) : BackwardKernelOf<T, 2, 32, false, kHeld>(type);
  if (!g.whole) return BackwardKernelOf<T, kWide<T>, 32, false, kHeld>(type);
  return type == Kind::kF32 ? BackwardKernel<T, kWide<T>, 32, true, false, kHeld, float>
         : type == Kind::kBf16 ? BackwardKernel<T, kWide<T>, 32, true, false, kHeld, T> : BackwardKernel<T, kWide<T>, 32, true, false, kHeld, void>;
}
template <class T, int kVec, int kLanes, bool kSplit> auto ForwardKernelOf(Kind type) {
  return type == Kind::kF32 ? ForwardKernel<T, kVec, kLanes, false, kSplit, float> : ForwardKernel<T, kVec, kLanes, false, kSplit, void>;
}
template <class T> auto ForwardKernelOf(const Geometry& g, int vec, Kind type) {
  if (g.lanes == 8)
    return vec == 1 ? ForwardKernelOf<T, 1, 8, false>(type) : vec == 2 ? ForwardKernelOf<T, 2, 8, false>(type)
           : ForwardKernelOf<T, kWide<T>, 8, false>(type);
  if (g.ranks > 1)
    return vec == 1 ? ForwardKernelOf<T, 1, 32, true>(type) : vec == 2 ? ForwardKernelOf<T, 2, 32, true>(type)
           : ForwardKernelOf<T, kWide<T>, 32, true>(type);
  if (vec <= 2) return vec == 1 ? ForwardKernelOf<T, 1, 32, false>(type) : ForwardKernelOf<T, 2, 32, false>(type);
  if (!g.whole) return ForwardKernelOf<T, kWide<T>, 32, false>(type);
  return type == Kind::kF32 ? ForwardKernel<T, kWide<T>, 32, true, false, float>
         : type == Kind::kBf16 ? ForwardKernel<T, kWide<T>, 32, true, false, T> : ForwardKernel<T, kWide<T>, 32, true, false, void>;
}

template <class T>
int Forward(const void* x_in, const void* residual_in, Parameter weight, Parameter bias, void* y_in, void* sum_in, float* mean,
            float* rstd, long long rows, int n, float eps, cudaStream_t stream) {
  const T *x = static_cast<const T*>(x_in), *residual = static_cast<const T*>(residual_in);
  T *y = static_cast<T*>(y_in), *sum = static_cast<T*>(sum_in);
  Alignment at;
  at.Of(x), at.Of(residual), at.Of(weight), at.Of(bias), at.Of(y), at.Of(sum);
  const int vec = at.Vec(n, kWide<T>);
  const Geometry g(rows, n, ForwardHeld(vec, sizeof(T)), kForwardWarps, 16, 1 << 30);
  if (!g.lanes)
    return Launched(LaunchOverlapped(ForwardAnyKernel<T>, RowBlocks(rows), kAnyThreads, 0, 1, stream, x, residual, weight, bias, y, sum,
                                     mean, rstd, rows, n, eps));
  return Launched(LaunchOverlapped(ForwardKernelOf<T>(g, vec, TypeOf<T>(weight, bias)), g.Blocks(), g.Threads(), 0, g.ranks, stream,
                                   x, residual, weight, bias, y, sum, mean, rstd, rows, n, eps, g.groups, g.warps, g.ranks));
}

template <class T>
int Backward(const void* dy_in, const void* dsum_in, const void* s_in, Parameter weight, const float* mean, const float* rstd,
             void* dx_in, void* dweight, void* dbias, float* workspace, long long rows, int n, int wtype, cudaStream_t stream) {
  const T *dy = static_cast<const T*>(dy_in), *dsum = static_cast<const T*>(dsum_in), *s = static_cast<const T*>(s_in);
  T* dx = static_cast<T*>(dx_in);
  if (!dweight && !dbias) workspace = nullptr;
  Alignment at;
  at.Of(dy), at.Of(dsum), at.Of(s), at.Of(weight), at.Of(dx), at.Of(workspace);  // (vectors' sums go there in pairs)
  const int vec = at.Vec(n, kWide<T>);
  const int held = BackwardHeld(n, vec);
  const Geometry g = BackwardGeometry(rows, n, held);
  int parts = 0;
  cudaError_t e;
  if (g.lanes) {
    const Kind type = TypeOf<T>(weight, weight);
    const auto kernel = held == 16 ? BackwardKernelOf<T, 16>(g, vec, type) : BackwardKernelOf<T, 8>(g, vec, type);
    const int ring = BackwardStages(vec, held, sizeof(T)) * BackwardRowBytes(held, sizeof(T));
    const int ends = workspace && g.groups > 1 ? (g.groups + 1) / 2 * (g.Threads() / g.groups) * 2 * held * static_cast<int>(sizeof(float)) : 0;
    const int shared = ring > ends ? ring : ends;
    if (shared > 32 << 10) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared);
      if (e != cudaSuccess) return Launched(e);
    }
    parts = g.parts;
    e = LaunchOverlapped(kernel, g.Blocks(), BackwardThreads(held), shared, g.ranks, stream, dy, dsum, s, weight, mean, rstd, dx,
                         workspace, rows, n, g.groups, g.warps, g.ranks);
  } else {
    e = LaunchOverlapped(BackwardAnyKernel<T>, RowBlocks(rows), kAnyThreads, 0, 1, stream, dy, dsum, s, weight, mean, rstd, dx, rows, n);
    if (e == cudaSuccess && workspace) {
      parts = 1;
      ColumnsAnyKernel<T><<<(n - 1) / 32 + 1, kAnyThreads, 0, stream>>>(dy, s, mean, rstd, workspace, rows, n);
      e = cudaGetLastError();
    }
  }
  if (e != cudaSuccess || !workspace) return Launched(e);
  return Launched(LaunchOverlapped(FinishColumnsKernel, (n - 1) / kFinishColumns + 1, kFinishThreads, 0, 1, stream,
                                   workspace, dweight, dbias, parts, n, wtype));
}

}  // namespace

extern "C" int switchml_layer_norm_forward(const void* x, const void* residual, const void* weight, const void* bias, void* y,
                                           void* sum, float* mean, float* rstd, long long rows, int features, float eps, int type,
                                           int wtype, void* stream) {
  if (!x || !y || (residual && !sum) || !mean != !rstd || rows <= 0 || !Fits(features) || !Known(type) || !Known(wtype)) return -1;
  if (!Aligned(SizeOf(type), x, residual, y, sum) || !Aligned(SizeOf(wtype), weight, bias) || !Aligned(4, mean, rstd)) return -1;
  return (type == SML_NORM_F32 ? Forward<float> : Forward<__nv_bfloat16>)(x, residual, Parameter{weight, wtype},
                                                                          Parameter{bias, wtype}, y, sum, mean, rstd, rows, features,
                                                                          eps, static_cast<cudaStream_t>(stream));
}

extern "C" long long switchml_layer_norm_workspace(long long rows, int features, int type) {
  if (rows <= 0 || !Fits(features) || !Known(type)) return 0;
  // (Which it will be depends on the addresses too.)
  const Geometry g = BackwardGeometry(rows, features, 8), h = BackwardGeometry(rows, features, 16);
  const int held = g.parts > h.parts ? g.parts : h.parts;
  return 2ll * features * (h.lanes ? held : 1);
}

extern "C" int switchml_layer_norm_backward(const void* dy, const void* dsum, const void* s, const void* weight, const float* mean,
                                            const float* rstd, void* dx, void* dweight, void* dbias, float* workspace, long long rows,
                                            int features, int type, int wtype, void* stream) {
  if (!dy || !s || !mean || !rstd || !dx || ((dweight || dbias) && !workspace) || rows <= 0 || !Fits(features) || !Known(type) ||
      !Known(wtype))
    return -1;
  if (!Aligned(SizeOf(type), dy, dsum, s, dx) || !Aligned(SizeOf(wtype), weight, dweight, dbias) || !Aligned(4, mean, rstd, workspace)) return -1;
  return (type == SML_NORM_F32 ? Backward<float> : Backward<__nv_bfloat16>)(dy, dsum, s, Parameter{weight, wtype}, mean, rstd, dx,
                                                                            dweight, dbias, workspace, rows, features, wtype,
                                                                            static_cast<cudaStream_t>(stream));
}

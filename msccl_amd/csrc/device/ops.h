// The training-step operators (include/msccl_amd_ops.h): what the host and the kernels share, and
// the kernels' load / store / reduction helpers.
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace msccl {

// ---- shared with the host ------------------------------------------------------------------

constexpr int kOpsThreads = 256;
constexpr int kOpsVec = 8;                              // elements a lane takes at a time
constexpr uint32_t kOpsChunk = kOpsThreads * kOpsVec;   // elements of one tensor a workgroup takes at a time
constexpr int kStateBlock = 256;                        // elements that share a scale in 8-bit states

// rows of the tensor tables; a table is [rows][starts: n + 1 chunk numbers, uint32_t]
struct SumTensor {
  const void* data;
  uint64_t count;
};
struct AdamTensor {
  void* param;
  const void* grad;
  float* master;
  void* m;
  void* v;
  float* mScale;
  float* vScale;
  uint64_t count;
  double decay;
  double lrScale;
};

// what one step's launches share (written by the first, read by the second)
struct AdamControl {
  double lr;
  double rate;       // lr / (1 - beta1^t)
  float invRoot;     // 1 / sqrt(1 - beta2^t)
  float coef;        // on the gradients
  int skip;
  int pad;
};

template <class Row>
struct TensorTable {
  const Row* rows;
  const uint32_t* starts;
  uint32_t n;
  uint32_t chunks;
};

struct AdamStepArgs {
  TensorTable<AdamTensor> tab;
  AdamControl* ctl;
  double lr;
  const float* lrDevice;
  double beta1, beta2;
  double gradScale;
  const double* squareSum;
  double maxNorm;
  int64_t* step;
  float b1, c1, b2, c2, eps;
};

struct BalanceArgs {
  const void* logits;
  int64_t tokens;
  int experts;
  int topK;
  int64_t logitStride;
  const void* index;
  int64_t indexStride;
  const uint8_t* valid;
  // statistics
  int64_t* counts;
  float* probs;
  uint32_t* countPart;   // [grid][experts + 1]
  float* probPart;       // [grid][experts]
  // gradient
  const int64_t* countsIn;
  const float* gradLoss;
  void* grad;
  int64_t gradStride;
  double scale;          // coef * experts / topK
};

// 0: launched; 1: no such variant or a launch error.  Types are ncclDataType_t.
int launchTableWrite(void* dst, const void* host, size_t bytes, void* stream);
int launchGradWrite(AdamTensor* rows, const void* const* grads, size_t n, void* stream);
int launchSquareSum(const TensorTable<SumTensor>& tab, int type, double* out, double* partials, int blocks, void* stream);
int launchAdamW(const AdamStepArgs& a, int paramType, int gradType, bool master, int bits, void* stream);
int balanceBlocks(int64_t tokens, int experts);
int launchBalanceStats(const BalanceArgs& a, int type, bool index64, bool sigmoid, int blocks, void* stream);
int launchBalanceLoss(const int64_t* counts, const float* probs, int experts, double scale, float* loss, void* stream);
int launchBalanceBackward(const BalanceArgs& a, int type, bool sigmoid, bool accumulate, void* stream);
constexpr int kSumBlocks = 2048;        // most workgroups (partial sums) of a square sum
constexpr int kMaxExperts = 1024;

}  // namespace msccl

#ifdef __HIPCC__
#include <hip/hip_runtime.h>

namespace msccl {

#define OPS_GLOBAL __attribute__((address_space(1)))
#define OPS_CONST __attribute__((address_space(4)))

// A tensor's address comes out of a table: without its address space the compiler would take flat
// loads, which wait for LDS too.
template <class T>
__device__ __forceinline__ OPS_GLOBAL T* inGlobal(T* p) { return (OPS_GLOBAL T*)p; }
// A value that no kernel of the launch writes, at an address that is the wave's: a scalar load.
template <class T>
__device__ __forceinline__ T scalarLoad(const T* p) { return *(const OPS_CONST T*)p; }

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t opsU32x2 __attribute__((ext_vector_type(2)));

// Eight contiguous elements.  The vector types carry their element's alignment only: gfx950 loads and
// stores 16 bytes at any address, so tensors that start anywhere take the same path.
template <class T>
struct Vec8;
template <>
struct Vec8<float> {
  typedef float V __attribute__((ext_vector_type(8)));
  typedef float U __attribute__((ext_vector_type(8), aligned(4)));
};
template <>
struct Vec8<__bf16> {
  typedef __bf16 V __attribute__((ext_vector_type(8)));
  typedef __bf16 U __attribute__((ext_vector_type(8), aligned(2)));
};
template <>
struct Vec8<_Float16> {
  typedef _Float16 V __attribute__((ext_vector_type(8)));
  typedef _Float16 U __attribute__((ext_vector_type(8), aligned(2)));
};
typedef opsU32x2 U8x8 __attribute__((aligned(1)));

// n: how many of the eight are there (the rest reads as `fill`)
template <class T>
__device__ __forceinline__ f32x8 load8(const T* p, int n, float fill = 0.f) {
  if (n >= 8) return __builtin_convertvector(*(const OPS_GLOBAL typename Vec8<T>::U*)p, f32x8);
  f32x8 x;
#pragma unroll
  for (int i = 0; i < 8; i++) x[i] = i < n ? (float)inGlobal(p)[i] : fill;
  return x;
}

// rounds to nearest, ties to even
template <class T>
__device__ __forceinline__ void store8(T* p, f32x8 x, int n) {
  if (n >= 8) {
    *(OPS_GLOBAL typename Vec8<T>::U*)p = __builtin_convertvector(x, typename Vec8<T>::V);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (i < n) inGlobal(p)[i] = (T)x[i];
}

__device__ __forceinline__ opsU32x2 loadBytes8(const uint8_t* p, int n) {
  if (n >= 8) return *(const OPS_GLOBAL U8x8*)p;
  opsU32x2 x = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (i < n) x[i / 4] |= (uint32_t)inGlobal(p)[i] << (8 * (i % 4));
  return x;
}

__device__ __forceinline__ void storeBytes8(uint8_t* p, opsU32x2 x, int n) {
  if (n >= 8) {
    *(OPS_GLOBAL U8x8*)p = x;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (i < n) inGlobal(p)[i] = (uint8_t)(x[i / 4] >> (8 * (i % 4)));
}

// The tensor that chunk c of a table lies in: the last row whose first chunk is at most c (empty
// tensors start where the next one does).  All lanes of a wave look at once, 64 rows apart in each
// round: one round for 64 tensors, two for 4096.
__device__ __forceinline__ uint32_t findTensor(const uint32_t* starts, uint32_t n, uint32_t c) {
  uint32_t lo = 0, len = n;
  const uint32_t lane = threadIdx.x & 63;
  while (len > 1) {
    const uint32_t step = (len + 63) / 64;
    const uint32_t i = lane * step;
    const bool below = i < len && inGlobal(starts)[lo + i] <= c;
    const uint32_t k = __builtin_popcountll(__ballot(below)) - 1;
    lo += k * step;
    const uint32_t left = len - k * step;
    len = left < step ? left : step;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

template <class T>
__device__ __forceinline__ T blockSum(T x, T* lds) {   // every thread gets the sum; lds: one T a wave
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  const int waves = blockDim.x / 64;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x / 64] = x;
  __syncthreads();
  T s = lds[0];
  for (int w = 1; w < waves; w++) s += lds[w];
  __syncthreads();
  return s;
}

}  // namespace msccl
#endif

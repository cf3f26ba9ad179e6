// The training-step operators (include/msccl_amd_ops.h): what the host and the kernels share, and
// the kernels' load / store / reduction helpers.
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace msccl {

// ---- shared with the host ------------------------------------------------------------------

constexpr int kOpsThreads = 256;
constexpr int kStateBlock = 256;     // elements that share a scale in 8-bit states
// elements of one tensor that a workgroup takes at a time
// (AdamW: `wide`, where a tensor beside 8-bit states is in 32 bits)
constexpr int adamEach(int bits, bool wide) { return bits == 8 && wide ? 4 : 8; }   // elements a lane
constexpr uint32_t adamChunk(int bits, bool wide) { return kOpsThreads * adamEach(bits, wide); }
constexpr int kSumVecs = 2;          // 16-byte vectors a lane
constexpr uint32_t sumChunk(size_t elemSize) { return kOpsThreads * (16 / elemSize) * kSumVecs; }

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
  int64_t t;         // the step's number
  int skip;
  uint32_t arrived;  // workgroups of a one-launch step that have read the step count; 0 between steps
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
  uint64_t seed;     // of the states' rounding, where that is by chance
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
  double* probPart;      // [grid][experts], 4-byte aligned
  uint32_t* countPart;   // [grid][experts + 1]
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
int launchAdamW(const AdamStepArgs& a, int paramType, int gradType, bool master, int bits, bool dice, void* stream);
int balanceBlocks(int64_t tokens, int experts);   // workgroups of the statistics; one needs no scratch
int launchBalanceStats(const BalanceArgs& a, int type, bool index64, bool sigmoid, int blocks, void* stream);
int launchBalanceLoss(const int64_t* counts, const float* probs, int experts, double scale, float* loss, void* stream);
int launchBalanceBackward(const BalanceArgs& a, int type, bool sigmoid, bool accumulate, void* stream);
constexpr int kSumThreads = 1024;       // a workgroup of a square sum: four groups that take chunks by themselves
constexpr int kSumBlocks = 256;         // most of them, and of the partial sums
// Up to this many chunks one workgroup and one launch: 65536 32-bit values 5.3 us, with the second launch 9.5
// (both the host's time); 131072 would take the workgroup longer than the host.
constexpr uint32_t kSumOne = 32;
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

// N contiguous elements.  The vector types carry their element's alignment only: gfx950 loads and
// stores 16 bytes at any address, so tensors that start anywhere take the same path.
template <class T, int N>
struct VecOf {
  typedef T V __attribute__((ext_vector_type(N)));
  typedef T U __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  typedef float F __attribute__((ext_vector_type(N)));
};

template <int N, class T>
__device__ __forceinline__ typename VecOf<T, N>::V loadVec(const T* p) {
  return *(const OPS_GLOBAL typename VecOf<T, N>::U*)p;
}

// What is read once and written once a step streams past the caches' other contents.
template <int N, class T>
__device__ __forceinline__ typename VecOf<T, N>::V streamVec(const T* p) {
  return __builtin_nontemporal_load((const OPS_GLOBAL typename VecOf<T, N>::U*)p);
}

// n: how many of the N are there (the rest reads as `fill`)
template <int N, class T>
__device__ __forceinline__ typename VecOf<T, N>::F loadN(const T* p, int n, float fill = 0.f) {
  if (n >= N) return __builtin_convertvector(streamVec<N>(p), typename VecOf<T, N>::F);
  typename VecOf<T, N>::F x;
#pragma unroll
  for (int i = 0; i < N; i++) x[i] = fill;
  if (n > 0) {   // the last one again in place of those that are not there: the loads need no branches
    T y[N];
#pragma unroll
    for (int i = 0; i < N; i++) y[i] = inGlobal(p)[i < n ? i : n - 1];
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = i < n ? (float)y[i] : fill;
  }
  return x;
}

// rounds to nearest, ties to even
template <int N, class T>
__device__ __forceinline__ void storeN(T* p, typename VecOf<T, N>::F x, int n) {
  if (n >= N) {
    const typename VecOf<T, N>::U y = __builtin_convertvector(x, typename VecOf<T, N>::V);
    __builtin_nontemporal_store(y, (OPS_GLOBAL typename VecOf<T, N>::U*)p);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; i++)
    if (i < n) inGlobal(p)[i] = (T)x[i];
}

// the same of N bytes, four to a word
template <int N>
struct BytesOf {
  typedef uint32_t V __attribute__((ext_vector_type(N / 4)));
  typedef uint32_t U __attribute__((ext_vector_type(N / 4), aligned(1)));
};

template <int N>
__device__ __forceinline__ typename BytesOf<N>::V loadBytes(const uint8_t* p, int n) {
  if (n >= N) return __builtin_nontemporal_load((const OPS_GLOBAL typename BytesOf<N>::U*)p);
  typename BytesOf<N>::V x = 0;
  if (n > 0) {
    uint8_t y[N];
#pragma unroll
    for (int i = 0; i < N; i++) y[i] = inGlobal(p)[i < n ? i : n - 1];
#pragma unroll
    for (int i = 0; i < N; i++) x[i / 4] |= i < n ? (uint32_t)y[i] << (8 * (i % 4)) : 0;
  }
  return x;
}

template <int N>
__device__ __forceinline__ void storeBytes(uint8_t* p, typename BytesOf<N>::V x, int n) {
  if (n >= N) {
    const typename BytesOf<N>::U y = x;
    __builtin_nontemporal_store(y, (OPS_GLOBAL typename BytesOf<N>::U*)p);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; i++)
    if (i < n) inGlobal(p)[i] = (uint8_t)(x[i / 4] >> (8 * (i % 4)));
}

// ---- exchanges between lanes -------------------------------------------------------------------
// combine(x, of the lane's partner) over groups of 2, 4, ... L lanes; every lane of a group ends with
// the same bits.  All of it in vector instructions (DPP up to 16 lanes, gfx950's row swaps beyond): an
// exchange through LDS takes a hundred cycles, and a row's maximum and sum are five or six in a row.
// (The mirrors pair a lane with one of the other half; within a half all lanes hold the same by then.)
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
template <int L, class F>
__device__ __forceinline__ uint32_t reduceLanes(uint32_t x, F combine) {
  if constexpr (L >= 2) x = combine(x, dpp<0xB1>(x));     // neighbours: quad_perm 1 0 3 2
  if constexpr (L >= 4) x = combine(x, dpp<0x4E>(x));     // pairs: quad_perm 2 3 0 1
  if constexpr (L >= 8) x = combine(x, dpp<0x141>(x));    // mirror of 8
  if constexpr (L >= 16) x = combine(x, dpp<0x140>(x));   // mirror of 16
  if constexpr (L >= 32) {
    const auto y = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = combine(y[0], y[1]);
  }
  if constexpr (L >= 64) {
    const auto y = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = combine(y[0], y[1]);
  }
  return x;
}
template <int L>
__device__ __forceinline__ float maxOver(float x) {
  return __builtin_bit_cast(float, reduceLanes<L>(__builtin_bit_cast(uint32_t, x), [](uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));
  }));
}
template <int L>
__device__ __forceinline__ float sumOver(float x) {
  return __builtin_bit_cast(float, reduceLanes<L>(__builtin_bit_cast(uint32_t, x), [](uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
  }));
}
// the sum of 64-bit values over the wave's lanes whose numbers are the same but for multiples of L, the
// halves exchanged alike (from far to near: what a row rotation by 8, 4, 2 or 1 brings is the lane's partner,
// as all lanes twice as far apart hold the same)
__device__ __forceinline__ double fromHalves(uint32_t hi, uint32_t lo) {
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int L>
__device__ __forceinline__ double sumAcross(double x) {
  const auto hi = [](double y) { return (uint32_t)(__builtin_bit_cast(uint64_t, y) >> 32); };
  const auto lo = [](double y) { return (uint32_t)__builtin_bit_cast(uint64_t, y); };
  if constexpr (L <= 32) {
    const auto h = __builtin_amdgcn_permlane32_swap(hi(x), hi(x), false, false);
    const auto l = __builtin_amdgcn_permlane32_swap(lo(x), lo(x), false, false);
    x = fromHalves(h[0], l[0]) + fromHalves(h[1], l[1]);
  }
  if constexpr (L <= 16) {
    const auto h = __builtin_amdgcn_permlane16_swap(hi(x), hi(x), false, false);
    const auto l = __builtin_amdgcn_permlane16_swap(lo(x), lo(x), false, false);
    x = fromHalves(h[0], l[0]) + fromHalves(h[1], l[1]);
  }
  if constexpr (L <= 8) x += fromHalves(dpp<0x128>(hi(x)), dpp<0x128>(lo(x)));
  if constexpr (L <= 4) x += fromHalves(dpp<0x124>(hi(x)), dpp<0x124>(lo(x)));
  if constexpr (L <= 2) x += fromHalves(dpp<0x122>(hi(x)), dpp<0x122>(lo(x)));
  if constexpr (L <= 1) x += fromHalves(dpp<0x121>(hi(x)), dpp<0x121>(lo(x)));
  return x;
}
// a wave's sum of 64-bit values: the halves exchanged alike
__device__ __forceinline__ double waveSum(double x) {
#define OPS_STEP(CTRL) do { const uint64_t b = __builtin_bit_cast(uint64_t, x); \
    x += fromHalves(dpp<CTRL>((uint32_t)(b >> 32)), dpp<CTRL>((uint32_t)b)); } while (0)
  OPS_STEP(0xB1);
  OPS_STEP(0x4E);
  OPS_STEP(0x141);
  OPS_STEP(0x140);
#undef OPS_STEP
  x += __shfl_xor(x, 16);
  x += __shfl_xor(x, 32);
  return x;
}
template <int L>
__device__ __forceinline__ uint32_t umaxOver(uint32_t x) {
  return reduceLanes<L>(x, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

// The tensor that chunk c of a table lies in: the last row whose first chunk is at most c (empty
// tensors start where the next one does).  All lanes of a wave look at once, 64 rows apart in each
// round: one round for 64 tensors, two for 4096.  What the first round compares is the same for every
// chunk: searchStart, read once.
__device__ __forceinline__ uint32_t searchStart(const uint32_t* starts, uint32_t n) {
  const uint32_t i = (threadIdx.x & 63) * ((n + 63) / 64);
  return i < n ? inGlobal(starts)[i] : 0xffffffffu;
}
__device__ __forceinline__ uint32_t findTensor(const uint32_t* starts, uint32_t n, uint32_t c, uint32_t seen) {
  uint32_t lo = 0, len = n;
  const uint32_t lane = threadIdx.x & 63;
  while (len > 1) {
    const uint32_t step = (len + 63) / 64;
    const uint32_t k = __builtin_popcountll(__ballot(seen <= c)) - 1;
    lo += k * step;
    const uint32_t left = len - k * step;
    len = left < step ? left : step;
    if (len > 1) {
      const uint32_t i = lane * ((len + 63) / 64);
      seen = i < len ? inGlobal(starts)[lo + i] : 0xffffffffu;
    }
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// The workgroup's sum (thread 0's): the wave's by exchanges, the waves' by LDS (lds: one value a wave).
template <int WAVES>
__device__ __forceinline__ double blockSum(double x, double* lds) {
  x = waveSum(x);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x / 64] = x;
  __syncthreads();
  return threadIdx.x < 64 ? waveSum(threadIdx.x < WAVES ? lds[threadIdx.x] : 0.0) : 0.0;
}

}  // namespace msccl
#endif

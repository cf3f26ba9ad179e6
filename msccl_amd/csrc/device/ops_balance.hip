// Balance loss of a router's experts (include/msccl_amd_ops.h): statistics, loss, gradient.
//
// Mathematics: p_t = softmax(x_t) or sigmoid(x_t) over its sum; c_e the valid slots that chose e, P_e the
// sum of p_te over valid tokens, N those; loss = coef E / (k N^2) sum_e c_e P_e, and with
// w_e = coef E / (k N^2) c_e the gradient is p_te (w_e - sum_f w_f p_tf), times 1 - sigmoid(x_te) for sigmoids.
// Both passes are bound by reading the logits once (and writing the gradient once): a row is held in
// the registers of the 1 to 64 lanes that share it, 8 or 16 logits each, so nothing is read twice and
// the sums over a row are lane exchanges.  A lane's columns are the same in every row it takes: the
// sums over rows stay in its registers too, then one exchange through LDS and one partial sum a
// workgroup, which a second launch adds in a fixed order.  They are in 64 bits throughout and rounded once:
// a router that starts from zero weights has equal rows, whose roundings in 32 bits do not average out
// (a 64-bit FMA issues as a 32-bit one does; with the conversions the long batch takes 0.55 us more).
// Counts are integers: their atomics (in LDS) give the same result in any order.  The statistics'
// workgroups are large and few, one a CU, so that there are few partial sums to add (256; with 512 the
// second launch takes 1 us longer than the first gains); the row after the one that is worked on is always
// on its way.  131072 tokens of 256 experts in bfloat16: statistics 19.5 to 20.3 us (68 MiB, bound by
// instruction issue: reading and adding in 32 bits alone take 12.4) and 2.8 to 3.9 for the second launch,
// 21.65 for both and the loss in a stream of them; gradient 23.4 us (128 MiB, 5.7 TB/s).
#include "ops.h"

#include <type_traits>

namespace msccl {

// e^x as 2^(x log2 e); the hardware's 2^t is within a unit of the last place.
constexpr float kLog2e = 1.44269502f;
__device__ __forceinline__ float exp2Of(float t) { return __builtin_amdgcn_exp2f(t); }

// max(a, b), or b where a is not a number; one instruction (the library's makes its operands quiet first)
__device__ __forceinline__ float larger(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, __builtin_inff()); }

// e^(x - top) of a row, by the difference itself: right for any finite top.  A row of -inf alone has no scores.
template <int VPL>
__device__ __forceinline__ void differences(f32x8 (&x)[VPL], float top) {
  const float from = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
  for (int j = 0; j < VPL; j++)
#pragma unroll
    for (int i = 0; i < 8; i++) x[j][i] = exp2Of((x[j][i] - from) * kLog2e);
}

template <int LPR, int VPL>
__device__ __forceinline__ float largest(const f32x8 (&x)[VPL]) {
  float top = -__builtin_inff();
#pragma unroll
  for (int j = 0; j < VPL; j++)
#pragma unroll
    for (int i = 0; i < 8; i++) top = larger(x[j][i], top);
  return maxOver<LPR>(top);
}

template <int LPR, int VPL>
__device__ __forceinline__ float total(const f32x8 (&x)[VPL]) {
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < VPL; j++)
#pragma unroll
    for (int i = 0; i < 8; i++) sum += x[j][i];
  return sumOver<LPR>(sum);
}

// The row's unnormalised scores in place of its logits: e^(x - max) or sigmoid(x) (0 outside the row), or
// what is in proportion to them.  Returns their sum.  SLOPE: also 1 - sigmoid(x), which 1 - s would round
// away near 1.
template <int LPR, int VPL, bool SIG, bool SLOPE>
__device__ __forceinline__ float scores(f32x8 (&x)[VPL], f32x8* slope) {
  if constexpr (SIG) {
    f32x8 logit[VPL];
#pragma unroll
    for (int j = 0; j < VPL; j++) {
      logit[j] = x[j];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        // e = e^-|x|: 1 / (1 + e), or e / (1 + e) left of zero (the reciprocal of 1 to 2: within one unit)
        const float e = exp2Of(-fabsf(x[j][i]) * kLog2e);
        const float r = __builtin_amdgcn_rcpf(1.f + e), er = e * r;
        const bool right = x[j][i] >= 0.f;
        if constexpr (SLOPE) slope[j][i] = right ? er : r;
        x[j][i] = right ? r : er;
      }
    }
    float z = total<LPR, VPL>(x);
    const bool far = z < 0x1p-25f;
    if (__builtin_expect(__ballot(far) != 0, 0)) {
      // Every logit is below -17: 1 + e^x is one, and e^(x - max) in proportion to the scores, which leave 32
      // bits from -87 on.  Above that a score that the exponential flushes is less than 2^-101 of the sum.
      const float top = largest<LPR, VPL>(logit);
      if (far) {
        differences<VPL>(logit, top);
#pragma unroll
        for (int j = 0; j < VPL; j++) x[j] = logit[j];
        z = total<LPR, VPL>(x);
      }
    }
    return z;
  } else {
    const float top = largest<LPR, VPL>(x);
    if (__builtin_expect(__ballot(!(fabsf(top) < 0x1p20f)) != 0, 0)) {
      // Large, masked with a low value throughout, infinite or nothing there.
      differences<VPL>(x, top);
    } else {
      // One FMA: the rounding of top log2(e), at most 2^-4 here, is the same factor of 0.957 to 1.045 on every
      // score of the row (without the bound above it would grow with top until the scores are inf or 0).
      const float from = -top * kLog2e;
#pragma unroll
      for (int j = 0; j < VPL; j++)
#pragma unroll
        for (int i = 0; i < 8; i++) x[j][i] = exp2Of(fmaf(x[j][i], kLog2e, from));
    }
    return total<LPR, VPL>(x);
  }
}

// One over the row's sum; 0 for a row without scores.  A softmax's is 0.95 to 1071, where the hardware's
// reciprocal is within one unit; a sum of sigmoids 2^-25 to 1024.
template <bool SIG>
__device__ __forceinline__ float inverse(float z) {
  if constexpr (SIG) return z == 0.f ? 0.f : 1.f / z;
  else return z == 0.f ? 0.f : __builtin_amdgcn_rcpf(z);
}

// A lane's eight columns of a row: base + i for i from `skip` up to `end`.  Where a row's end leaves
// fewer than eight, the eight before the end, without those that the lane before has: any row of eight
// or more is read in whole vectors that stay inside it.
struct Columns {
  int base, skip, end;
  bool whole;   // of every lane of the row (the wave's: a scalar)
  __device__ __forceinline__ Columns(int experts, int width, int col) {
    base = experts < 8 ? 0 : col < experts - 8 ? col : experts - 8;
    skip = col - base < 8 ? col - base : 8;
    end = experts < 8 ? experts : 8;
    whole = experts % 8 == 0 && experts == width;
  }
  __device__ __forceinline__ bool has(int i) const { return i >= skip && i < end; }
};

// The lane's eight of a row as they stand, and as 32-bit values with `none` in the place of columns that
// are not its own.
template <class T, int LPR>
__device__ __forceinline__ typename VecOf<T, 8>::V loadRow(const T* row, const Columns& c) {
  typename VecOf<T, 8>::V x;
  if (LPR == 1 && c.end < 8) {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = inGlobal(row)[i < c.end ? i : c.end - 1];
  } else {
    x = loadVec<8>(row + c.base);
  }
  return x;
}
template <class V>
__device__ __forceinline__ f32x8 ownColumns(const V& raw, const Columns& c, float none) {
  f32x8 x = __builtin_convertvector(raw, f32x8);
  if (!c.whole) {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = c.has(i) ? x[i] : none;
  }
  return x;
}

constexpr int kStatsThreads = 1024;
typedef double Double4 __attribute__((aligned(4)));   // (the caller's scratch is at a 4-byte boundary)

template <class T, int LPR, int VPL, bool SIG, bool IDX64>
__global__ void __launch_bounds__(kStatsThreads) balanceStatsKernel(BalanceArgs a, int64_t rowsEach) {
  constexpr int rowsPer = kStatsThreads / LPR;
  constexpr int width = LPR * VPL * 8;
  constexpr int waves = kStatsThreads / 64;
  constexpr int copies = width <= 128 ? waves : 1;   // few experts: every wave counts by itself
  __shared__ uint32_t hist[copies][width];
  __shared__ uint32_t tokens;
  constexpr int rooms = width <= 512 ? waves / 2 : waves / 4;   // (32 KiB of sums at most)
  __shared__ double sums[rooms][width];
  const int wave = threadIdx.x / 64;
  const int64_t begin = blockIdx.x * rowsEach;
  const int64_t first = begin < a.tokens ? begin : a.tokens;   // (the last workgroups may have none)
  const int64_t end = a.tokens - first < rowsEach ? a.tokens : first + rowsEach;

  const int lane = threadIdx.x % LPR, own = threadIdx.x / LPR;
  const Columns c0(a.experts, width, lane * 8), c1(a.experts, width, (LPR + lane) * 8);
  const int rows = (int)(end - first);
  const int64_t ahead = (int64_t)rowsPer * a.logitStride;
  const T* at = (const T*)a.logits + (first + own) * a.logitStride;
  const uint8_t* ok = a.valid ? a.valid + first : nullptr;
  // a row is on its way while the one before it, and at first the choices, are worked on
  typename VecOf<T, 8>::V raw[VPL];
  uint32_t valid = 1;   // (as it stands: a comparison here would wait for it)
  if (own < rows) {
    raw[0] = loadRow<T, LPR>(at, c0);
    if constexpr (VPL == 2) raw[1] = loadRow<T, LPR>(at, c1);
    if (ok) valid = inGlobal(ok)[own];
  }

  for (int i = threadIdx.x; i < copies * width; i += kStatsThreads) (&hist[0][0])[i] = 0;
  if (threadIdx.x == 0) tokens = 0;
  __syncthreads();
  const uint32_t slots = (uint32_t)rows * (uint32_t)a.topK;
  const bool packed = !ok && a.indexStride == a.topK;   // slot s of the rows is element s
  typedef typename std::conditional<IDX64, int64_t, int32_t>::type I;
  for (uint32_t s0 = threadIdx.x; s0 < slots; s0 += 4 * kStatsThreads) {
    I e[4];   // four on their way at once, without branches: the last slot again past the end
    uint32_t r[4], here[4] = {1, 1, 1, 1};
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const uint32_t s1 = s0 + k * kStatsThreads, s = s1 < slots ? s1 : slots - 1;
      r[k] = packed ? 0 : s / (uint32_t)a.topK;
      e[k] = inGlobal((const I*)a.index)[(first + r[k]) * a.indexStride + (s - r[k] * (uint32_t)a.topK)];
    }
    if (ok) {
#pragma unroll
      for (int k = 0; k < 4; k++) here[k] = inGlobal(ok)[r[k]];
    }
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (s0 + k * kStatsThreads < slots && here[k] && e[k] >= 0 && e[k] < (I)a.experts)
        atomicAdd(&hist[copies == 1 ? 0 : wave][e[k]], 1u);
  }

  double acc[VPL][8];
#pragma unroll
  for (int j = 0; j < VPL; j++)
#pragma unroll
    for (int i = 0; i < 8; i++) acc[j][i] = 0.0;
  uint32_t here = 0;
  for (int r = own; r < rows; r += rowsPer) {
    f32x8 x[VPL];
    x[0] = ownColumns(raw[0], c0, -__builtin_inff());
    if constexpr (VPL == 2) x[1] = ownColumns(raw[1], c1, -__builtin_inff());
    const bool now = valid != 0;
    if (r + rowsPer < rows) {
      at += ahead;
      raw[0] = loadRow<T, LPR>(at, c0);
      if constexpr (VPL == 2) raw[1] = loadRow<T, LPR>(at, c1);
      if (ok) valid = inGlobal(ok)[r + rowsPer];
    }
    if (!now) continue;   // (whatever the row holds)
    here++;
    const double inv = inverse<SIG>(scores<LPR, VPL, SIG, false>(x, nullptr));
#pragma unroll
    for (int j = 0; j < VPL; j++)
#pragma unroll
      for (int i = 0; i < 8; i++) acc[j][i] = fma((double)x[j][i], inv, acc[j][i]);
  }
  if (here && lane == 0) atomicAdd(&tokens, here);
  // over the wave's rows, then over the waves: some of them first, then the others on top
#pragma unroll
  for (int j = 0; j < VPL; j++)
#pragma unroll
    for (int i = 0; i < 8; i++) acc[j][i] = sumAcross<LPR>(acc[j][i]);
#pragma unroll
  for (int turn = 0; turn < waves / rooms; turn++) {
    if ((threadIdx.x & 63) < LPR && wave / rooms == turn) {
#pragma unroll
      for (int j = 0; j < VPL; j++) {
        const Columns& c = j ? c1 : c0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          if (c.has(i)) {
            double* s = &sums[wave % rooms][c.base + i];
            *s = turn == 0 ? acc[j][i] : *s + acc[j][i];
          }
        }
      }
    }
    __syncthreads();
  }
  const bool only = gridDim.x == 1;
  for (int e = threadIdx.x; e < a.experts; e += kStatsThreads) {
    double s = sums[0][e];
#pragma unroll
    for (int w = 1; w < rooms; w++) s += sums[w][e];
    uint32_t n = hist[0][e];
#pragma unroll
    for (int w = 1; w < copies; w++) n += hist[w][e];
    if (only) {
      a.probs[e] = (float)s;
      a.counts[e] = n;
    } else {
      *(Double4*)(a.probPart + (size_t)blockIdx.x * a.experts + e) = s;
      a.countPart[(size_t)blockIdx.x * (a.experts + 1) + e] = n;
    }
  }
  if (threadIdx.x == 0) {
    if (only) a.counts[a.experts] = tokens;
    else a.countPart[(size_t)blockIdx.x * (a.experts + 1) + a.experts] = tokens;
  }
}

// The partial sums of at most kStatsBlocks workgroups: 16 columns a workgroup, 64 threads down each, all
// loads of a thread under way at once.
constexpr int kStatsBlocks = 256;

__global__ void __launch_bounds__(1024) balanceFinishKernel(BalanceArgs a, int blocks) {
  constexpr int each = kStatsBlocks / 64;
  __shared__ double ps[16][16];
  __shared__ int64_t cs[16][16];
  const int col = threadIdx.x % 16, slice = threadIdx.x / 16;
  const int e = blockIdx.x * 16 + col;
  double p[each];
  uint32_t c[each];
#pragma unroll
  for (int k = 0; k < each; k++) {
    const int b = k * 64 + slice;
    p[k] = b < blocks && e < a.experts ? *(const Double4*)(a.probPart + (size_t)b * a.experts + e) : 0.0;
    c[k] = b < blocks && e <= a.experts ? a.countPart[(size_t)b * (a.experts + 1) + e] : 0;
  }
  double p0 = 0.0;
  int64_t c0 = 0;
#pragma unroll
  for (int k = 0; k < each; k++) {
    p0 += p[k];
    c0 += (int64_t)c[k];
  }
#pragma unroll
  for (int d = 16; d <= 32; d *= 2) {
    p0 += __shfl_xor(p0, d);
    c0 += __shfl_xor((long long)c0, d);
  }
  if ((threadIdx.x & 63) < 16) {
    ps[threadIdx.x / 64][col] = p0;
    cs[threadIdx.x / 64][col] = c0;
  }
  __syncthreads();
  if (threadIdx.x < 16 && e <= a.experts) {
#pragma unroll
    for (int k = 1; k < 16; k++) {
      p0 += ps[k][col];
      c0 += cs[k][col];
    }
    if (e < a.experts) a.probs[e] = (float)p0;
    a.counts[e] = c0;
  }
}

__global__ void __launch_bounds__(kOpsThreads) balanceLossKernel(const int64_t* counts, const float* probs, int experts,
                                                                double scale, float* loss) {
  __shared__ double lds[kOpsThreads / 64];
  double s = 0.0;
  for (int e = threadIdx.x; e < experts; e += kOpsThreads) s += (double)counts[e] * (double)probs[e];
  s = blockSum<kOpsThreads / 64>(s, lds);
  if (threadIdx.x == 0) {
    const double n = (double)counts[experts];
    *loss = n > 0 ? (float)(s * scale / (n * n)) : 0.f;
  }
}

template <class T, int LPR, int VPL, bool SIG, bool ACC>
__global__ void __launch_bounds__(kOpsThreads) balanceBackwardKernel(BalanceArgs a) {
  constexpr int rowsPer = kOpsThreads / LPR;
  const int lane = threadIdx.x % LPR;
  constexpr int width = LPR * VPL * 8;
  const Columns c0(a.experts, width, lane * 8), c1(a.experts, width, (LPR + lane) * 8);
  const int64_t ahead = (int64_t)gridDim.x * rowsPer, first = (int64_t)blockIdx.x * rowsPer + threadIdx.x / LPR;
  const T* in = (const T*)a.logits + first * a.logitStride;
  T* out = (T*)a.grad + first * a.gradStride;
  // as in the statistics, a row is on its way while the one before it is worked on
  typename VecOf<T, 8>::V raw[VPL];
  uint32_t next = 1;
  if (first < a.tokens) {
    raw[0] = loadRow<T, LPR>(in, c0);
    if constexpr (VPL == 2) raw[1] = loadRow<T, LPR>(in, c1);
    if (a.valid) next = inGlobal(a.valid)[first];
  }
  const double n = (double)a.countsIn[a.experts];
  // Every weight less c E / (k N^2) times the mean count of a routing that drops nothing, k N / E: p sums
  // to 1, so the gradient is the same, and with weights that are nearly equal nothing cancels in 32 bits.
  const double mean = n * a.topK / a.experts;
  const double up = n > 0 ? a.scale / (n * n) * (a.gradLoss ? (double)*a.gradLoss : 1.0) : 0.0;
  f32x8 w[VPL];
#pragma unroll
  for (int j = 0; j < VPL; j++) {
    const Columns& c = j ? c1 : c0;
#pragma unroll
    for (int i = 0; i < 8; i++) w[j][i] = c.has(i) ? (float)(((double)a.countsIn[c.base + i] - mean) * up) : 0.f;
  }
  for (int64_t row = first; row < a.tokens; row += ahead, out += ahead * a.gradStride) {
    f32x8 x[VPL], slope[VPL];
    x[0] = ownColumns(raw[0], c0, -__builtin_inff());
    if constexpr (VPL == 2) x[1] = ownColumns(raw[1], c1, -__builtin_inff());
    const bool valid = next != 0;
    if (row + ahead < a.tokens) {
      in += ahead * a.logitStride;
      raw[0] = loadRow<T, LPR>(in, c0);
      if constexpr (VPL == 2) raw[1] = loadRow<T, LPR>(in, c1);
      if (a.valid) next = inGlobal(a.valid)[row + ahead];
    }
    if (ACC && !valid) continue;
    if (valid) {
      const float inv = inverse<SIG>(scores<LPR, VPL, SIG, SIG>(x, slope));
      float dot = 0.f;
      if constexpr (SIG) {
        // A row's scores may be small: the probabilities first, so that their products with the weights are of
        // the weights' size and neither lose their digits nor pass 32 bits.
#pragma unroll
        for (int j = 0; j < VPL; j++)
#pragma unroll
          for (int i = 0; i < 8; i++) {
            x[j][i] *= inv;
            dot = fmaf(x[j][i], w[j][i], dot);
          }
        dot = sumOver<LPR>(dot);
#pragma unroll
        for (int j = 0; j < VPL; j++)
#pragma unroll
          for (int i = 0; i < 8; i++) x[j][i] *= (w[j][i] - dot) * slope[j][i];
      } else {
#pragma unroll
        for (int j = 0; j < VPL; j++)
#pragma unroll
          for (int i = 0; i < 8; i++) dot = fmaf(x[j][i], w[j][i], dot);
        // p (w - sum of w p) = s (w / z - (sum of w s) / z^2): the row's two sums do not wait for one another
        dot = sumOver<LPR>(dot) * inv * inv;
#pragma unroll
        for (int j = 0; j < VPL; j++)
#pragma unroll
          for (int i = 0; i < 8; i++) x[j][i] *= fmaf(w[j][i], inv, -dot);
      }
    } else {
#pragma unroll
      for (int j = 0; j < VPL; j++) x[j] = (f32x8){0, 0, 0, 0, 0, 0, 0, 0};
    }
#pragma unroll
    for (int j = 0; j < VPL; j++) {
      const Columns& c = j ? c1 : c0;
      if constexpr (ACC) x[j] += ownColumns(loadRow<T, LPR>(out, c), c, 0.f);
      if (c.whole || (c.skip == 0 && c.end == 8)) {
        storeN<8>(out + c.base, x[j], 8);
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (c.has(i)) inGlobal(out)[c.base + i] = (T)x[j][i];
      }
    }
  }
}

// ---- variants: the fewest lanes that hold a row, 8 logits each (64 lanes 16 past 512 experts) ----------

static int lanesPerRow(int experts) {
  int l = 1;
  while (l < 64 && l * 8 < experts) l *= 2;
  return l;
}

int balanceBlocks(int64_t tokens, int experts) {
  const int64_t rowsPer = kStatsThreads / lanesPerRow(experts);
  const int64_t passes = (tokens + rowsPer - 1) / rowsPer;
  // One workgroup writes the results itself: 4 passes 8.6 us against 12.9 with the second launch enqueued
  // one by one and 6.4 against 7.0 in a graph (64 experts), 8 passes 8.9 against 13 and 9.1 against 7.3.
  if (passes <= 4) return 1;
  return (int)(passes < kStatsBlocks ? passes : kStatsBlocks);
}

template <template <int, int> class F, class... A>
static int pick(int experts, A... args) {
  if (experts > 512) return F<64, 2>::run(args...);
  switch (lanesPerRow(experts)) {
    case 1: return F<1, 1>::run(args...);
    case 2: return F<2, 1>::run(args...);
    case 4: return F<4, 1>::run(args...);
    case 8: return F<8, 1>::run(args...);
    case 16: return F<16, 1>::run(args...);
    case 32: return F<32, 1>::run(args...);
    default: return F<64, 1>::run(args...);
  }
}

template <class T>
struct Stats {
  template <int LPR, int VPL>
  struct Of {
    static int run(const BalanceArgs* a, bool index64, bool sigmoid, int blocks, hipStream_t s) {
      const dim3 g(blocks), b(kStatsThreads);
      const int64_t each = (a->tokens + blocks - 1) / blocks;
      if (sigmoid) {
        if (index64) hipLaunchKernelGGL((balanceStatsKernel<T, LPR, VPL, true, true>), g, b, 0, s, *a, each);
        else hipLaunchKernelGGL((balanceStatsKernel<T, LPR, VPL, true, false>), g, b, 0, s, *a, each);
      } else {
        if (index64) hipLaunchKernelGGL((balanceStatsKernel<T, LPR, VPL, false, true>), g, b, 0, s, *a, each);
        else hipLaunchKernelGGL((balanceStatsKernel<T, LPR, VPL, false, false>), g, b, 0, s, *a, each);
      }
      return hipGetLastError() == hipSuccess ? 0 : 1;
    }
  };
};

template <class T>
struct Backward {
  template <int LPR, int VPL>
  struct Of {
    static int run(const BalanceArgs* a, bool sigmoid, bool accumulate, hipStream_t s) {
      constexpr int64_t rowsPer = kOpsThreads / LPR;
      const int64_t passes = (a->tokens + rowsPer - 1) / rowsPer;
      const dim3 g((uint32_t)(passes < 1024 ? passes : 1024)), b(kOpsThreads);
      if (sigmoid) {
        if (accumulate) hipLaunchKernelGGL((balanceBackwardKernel<T, LPR, VPL, true, true>), g, b, 0, s, *a);
        else hipLaunchKernelGGL((balanceBackwardKernel<T, LPR, VPL, true, false>), g, b, 0, s, *a);
      } else {
        if (accumulate) hipLaunchKernelGGL((balanceBackwardKernel<T, LPR, VPL, false, true>), g, b, 0, s, *a);
        else hipLaunchKernelGGL((balanceBackwardKernel<T, LPR, VPL, false, false>), g, b, 0, s, *a);
      }
      return hipGetLastError() == hipSuccess ? 0 : 1;
    }
  };
};

int launchBalanceStats(const BalanceArgs& a, int type, bool index64, bool sigmoid, int blocks, void* stream) {
  const hipStream_t s = (hipStream_t)stream;
  int r = 1;
  switch (type) {
    case 6: r = pick<Stats<_Float16>::template Of>(a.experts, &a, index64, sigmoid, blocks, s); break;
    case 7: r = pick<Stats<float>::template Of>(a.experts, &a, index64, sigmoid, blocks, s); break;
    case 9: r = pick<Stats<__bf16>::template Of>(a.experts, &a, index64, sigmoid, blocks, s); break;
  }
  if (r != 0 || blocks == 1) return r;
  hipLaunchKernelGGL(balanceFinishKernel, dim3((a.experts + 1 + 15) / 16), dim3(1024), 0, s, a, blocks);
  return hipGetLastError() == hipSuccess ? 0 : 1;
}

int launchBalanceLoss(const int64_t* counts, const float* probs, int experts, double scale, float* loss, void* stream) {
  hipLaunchKernelGGL(balanceLossKernel, dim3(1), dim3(kOpsThreads), 0, (hipStream_t)stream, counts, probs, experts,
                     scale, loss);
  return hipGetLastError() == hipSuccess ? 0 : 1;
}

int launchBalanceBackward(const BalanceArgs& a, int type, bool sigmoid, bool accumulate, void* stream) {
  const hipStream_t s = (hipStream_t)stream;
  if (a.tokens == 0) return 0;
  switch (type) {
    case 6: return pick<Backward<_Float16>::template Of>(a.experts, &a, sigmoid, accumulate, s);
    case 7: return pick<Backward<float>::template Of>(a.experts, &a, sigmoid, accumulate, s);
    case 9: return pick<Backward<__bf16>::template Of>(a.experts, &a, sigmoid, accumulate, s);
  }
  return 1;
}

}  // namespace msccl

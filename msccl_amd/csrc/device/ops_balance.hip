// Balance loss of a router's experts (include/msccl_amd_ops.h): statistics, loss, gradient.
//
// Mathematics: p_t = softmax(x_t) or sigmoid(x_t) over its sum; c_e the valid slots that chose e, P_e the
// sum of p_te over valid tokens, N those; loss = coef E / (k N^2) sum_e c_e P_e, and with
// w_e = coef E / (k N^2) c_e the gradient is p_te (w_e - sum_f w_f p_tf), times 1 - sigmoid(x_te) for sigmoids.
// Both passes are bound by reading the logits once (and writing the gradient once): a row is held in
// the registers of the 1 to 64 lanes that share it, 8 or 16 logits each, so nothing is read twice and
// the sums over a row are lane exchanges.  A lane's columns are the same in every row it takes: the
// sums over rows stay in its registers too, then one exchange through LDS and one partial sum a
// workgroup, which a second launch adds in a fixed order in 64 bits.  Counts are integers: their
// atomics (in LDS) give the same result in any order.
#include "ops.h"

namespace msccl {

// e^x by 2^x: t = x log2(e) rounded, e = what that rounding and log2(e)'s own left out, e^x = 2^t (1 + e ln 2).
// For x <= 0 within about one unit of the last place; -inf gives 0.
__device__ __forceinline__ float expNeg(float x) {
  constexpr float hi = 1.44269502f, lo = 1.92596303e-8f, ln2 = 0.693147182f;
  const float t = x * hi;
  const float y = __builtin_amdgcn_exp2f(t);
  const float e = fmaf(x, lo, fmaf(x, hi, -t));
  return x < -87.f ? y : fmaf(y, e * ln2, y);   // (also keeps -inf away from the correction)
}

template <int LPR>
__device__ __forceinline__ float rowMax(float x) {
#pragma unroll
  for (int d = LPR / 2; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}
template <int LPR>
__device__ __forceinline__ float rowSum(float x) {
#pragma unroll
  for (int d = LPR / 2; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

// The row's unnormalised scores in place of its logits: e^(x - max) or sigmoid(x) (0 outside the row).
// Returns the lane's part of their sum.  SLOPE: also 1 - sigmoid(x), which 1 - s would round away near 1.
template <int LPR, int VPL, bool SIG, bool SLOPE>
__device__ __forceinline__ float scores(f32x8 (&x)[VPL], f32x8* slope) {
  float sum = 0.f;
  if constexpr (SIG) {
#pragma unroll
    for (int j = 0; j < VPL; j++)
#pragma unroll
      for (int i = 0; i < 8; i++) {
        // e = e^-|x|: 1 / (1 + e), or e / (1 + e) left of zero
        const float e = expNeg(-fabsf(x[j][i]));
        const bool right = x[j][i] >= 0.f;
        if constexpr (SLOPE) slope[j][i] = (right ? e : 1.f) / (1.f + e);
        x[j][i] = (right ? 1.f : e) / (1.f + e);
        sum += x[j][i];
      }
  } else {
    float top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < VPL; j++)
#pragma unroll
      for (int i = 0; i < 8; i++) top = fmaxf(top, x[j][i]);
    top = rowMax<LPR>(top);
    // a row of -inf alone has no scores; its sum stays 0
    const float from = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
    for (int j = 0; j < VPL; j++)
#pragma unroll
      for (int i = 0; i < 8; i++) {
        x[j][i] = expNeg(x[j][i] - from);
        sum += x[j][i];
      }
  }
  return sum;
}

__device__ __forceinline__ int columns(int experts, int col) {   // of the lane's eight, how many are there
  const int n = experts - col;
  return n >= 8 ? 8 : n > 0 ? n : 0;
}

template <class T, int LPR, int VPL, bool SIG, bool IDX64>
__global__ void __launch_bounds__(kOpsThreads) balanceStatsKernel(BalanceArgs a) {
  constexpr int rowsPer = kOpsThreads / LPR;
  constexpr int width = LPR * VPL * 8;
  constexpr int waves = kOpsThreads / 64;
  __shared__ uint32_t hist[width + 1];
  __shared__ float sums[waves][width];
  for (int i = threadIdx.x; i <= width; i += kOpsThreads) hist[i] = 0;
  __syncthreads();

  uint32_t here = 0;
  for (int64_t row = (int64_t)blockIdx.x * kOpsThreads + threadIdx.x; row < a.tokens;
       row += (int64_t)gridDim.x * kOpsThreads) {
    if (a.valid && !a.valid[row]) continue;
    here++;
    for (int j = 0; j < a.topK; j++) {
      const int64_t e = IDX64 ? ((const int64_t*)a.index)[row * a.indexStride + j]
                              : (int64_t)((const int32_t*)a.index)[row * a.indexStride + j];
      if ((uint64_t)e < (uint64_t)a.experts) atomicAdd(&hist[e], 1u);
    }
  }
  if (here) atomicAdd(&hist[width], here);

  const int lane = threadIdx.x % LPR;
  f32x8 acc[VPL];
#pragma unroll
  for (int j = 0; j < VPL; j++) acc[j] = (f32x8){0, 0, 0, 0, 0, 0, 0, 0};
  for (int64_t row = (int64_t)blockIdx.x * rowsPer + threadIdx.x / LPR; row < a.tokens;
       row += (int64_t)gridDim.x * rowsPer) {
    if (a.valid && !a.valid[row]) continue;
    f32x8 x[VPL];
#pragma unroll
    for (int j = 0; j < VPL; j++) {
      const int col = (j * LPR + lane) * 8;
      x[j] = load8((const T*)a.logits + row * a.logitStride + col, columns(a.experts, col), -__builtin_inff());
    }
    const float z = rowSum<LPR>(scores<LPR, VPL, SIG, false>(x, nullptr));
    const float inv = z == 0.f ? 0.f : 1.f / z;
#pragma unroll
    for (int j = 0; j < VPL; j++)
#pragma unroll
      for (int i = 0; i < 8; i++) acc[j][i] += x[j][i] * inv;
  }
  // over the wave's rows, then over the waves
#pragma unroll
  for (int j = 0; j < VPL; j++) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      float s = acc[j][i];
#pragma unroll
      for (int d = 32; d >= LPR; d >>= 1) s += __shfl_xor(s, d);
      if ((threadIdx.x & 63) < LPR) sums[threadIdx.x / 64][(j * LPR + lane) * 8 + i] = s;
    }
  }
  __syncthreads();
  const bool only = gridDim.x == 1;
  for (int e = threadIdx.x; e < a.experts; e += kOpsThreads) {
    float s = sums[0][e];
#pragma unroll
    for (int w = 1; w < waves; w++) s += sums[w][e];
    if (only) {
      a.probs[e] = s;
      a.counts[e] = hist[e];
    } else {
      a.probPart[(size_t)blockIdx.x * a.experts + e] = s;
      a.countPart[(size_t)blockIdx.x * (a.experts + 1) + e] = hist[e];
    }
  }
  if (threadIdx.x == 0) {
    if (only) a.counts[a.experts] = hist[width];
    else a.countPart[(size_t)blockIdx.x * (a.experts + 1) + a.experts] = hist[width];
  }
}

// 16 columns a workgroup, 16 threads down each
__global__ void __launch_bounds__(kOpsThreads) balanceFinishKernel(BalanceArgs a, int blocks) {
  __shared__ double ps[kOpsThreads];
  __shared__ int64_t cs[kOpsThreads];
  const int e = blockIdx.x * 16 + threadIdx.x % 16;
  double p = 0.0;
  int64_t c = 0;
  for (int b = threadIdx.x / 16; b < blocks; b += 16) {
    if (e < a.experts) p += (double)a.probPart[(size_t)b * a.experts + e];
    if (e <= a.experts) c += (int64_t)a.countPart[(size_t)b * (a.experts + 1) + e];
  }
  ps[threadIdx.x] = p;
  cs[threadIdx.x] = c;
  __syncthreads();
  if (threadIdx.x < 16) {
    for (int k = 1; k < 16; k++) {
      p += ps[threadIdx.x + 16 * k];
      c += cs[threadIdx.x + 16 * k];
    }
    if (e < a.experts) a.probs[e] = (float)p;
    if (e <= a.experts) a.counts[e] = c;
  }
}

__global__ void __launch_bounds__(kOpsThreads) balanceLossKernel(const int64_t* counts, const float* probs, int experts,
                                                                double scale, float* loss) {
  __shared__ double lds[kOpsThreads / 64];
  double s = 0.0;
  for (int e = threadIdx.x; e < experts; e += kOpsThreads) s += (double)counts[e] * (double)probs[e];
  s = blockSum(s, lds);
  if (threadIdx.x == 0) {
    const double n = (double)counts[experts];
    *loss = n > 0 ? (float)(s * scale / (n * n)) : 0.f;
  }
}

template <class T, int LPR, int VPL, bool SIG, bool ACC>
__global__ void __launch_bounds__(kOpsThreads) balanceBackwardKernel(BalanceArgs a) {
  constexpr int rowsPer = kOpsThreads / LPR;
  const int lane = threadIdx.x % LPR;
  const double n = (double)a.countsIn[a.experts];
  // Every weight less c E / (k N^2) times the mean count of a routing that drops nothing, k N / E: p sums
  // to 1, so the gradient is the same, and with weights that are nearly equal nothing cancels in 32 bits.
  const double mean = n * a.topK / a.experts;
  const double up = n > 0 ? a.scale / (n * n) * (a.gradLoss ? (double)*a.gradLoss : 1.0) : 0.0;
  f32x8 w[VPL];
#pragma unroll
  for (int j = 0; j < VPL; j++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int e = (j * LPR + lane) * 8 + i;
      w[j][i] = e < a.experts ? (float)(((double)a.countsIn[e] - mean) * up) : 0.f;
    }
  for (int64_t row = (int64_t)blockIdx.x * rowsPer + threadIdx.x / LPR; row < a.tokens;
       row += (int64_t)gridDim.x * rowsPer) {
    const bool valid = !a.valid || a.valid[row];
    if (ACC && !valid) continue;
    f32x8 x[VPL], slope[VPL];
    if (valid) {
#pragma unroll
      for (int j = 0; j < VPL; j++) {
        const int col = (j * LPR + lane) * 8;
        x[j] = load8((const T*)a.logits + row * a.logitStride + col, columns(a.experts, col), -__builtin_inff());
      }
      const float mine = scores<LPR, VPL, SIG, SIG>(x, slope);
      float dot = 0.f;
#pragma unroll
      for (int j = 0; j < VPL; j++)
#pragma unroll
        for (int i = 0; i < 8; i++) dot += x[j][i] * w[j][i];
      const float z = rowSum<LPR>(mine);
      dot = rowSum<LPR>(dot);
      const float inv = z == 0.f ? 0.f : 1.f / z;
      dot *= inv;
#pragma unroll
      for (int j = 0; j < VPL; j++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float s = x[j][i];
          float d = s * inv * (w[j][i] - dot);
          if constexpr (SIG) d *= slope[j][i];
          x[j][i] = d;
        }
    } else {
#pragma unroll
      for (int j = 0; j < VPL; j++) x[j] = (f32x8){0, 0, 0, 0, 0, 0, 0, 0};
    }
#pragma unroll
    for (int j = 0; j < VPL; j++) {
      const int col = (j * LPR + lane) * 8;
      const int k = columns(a.experts, col);
      T* out = (T*)a.grad + row * a.gradStride + col;
      if constexpr (ACC) x[j] += load8(out, k);
      store8(out, x[j], k);
    }
  }
}

// ---- variants: the fewest lanes that hold a row, 8 logits each (two times 8 past 512 experts) --------

static int lanesPerRow(int experts) {
  int l = 1;
  while (l < 64 && l * 8 < experts) l *= 2;
  return l;
}

int balanceBlocks(int64_t tokens, int experts) {
  const int64_t rowsPer = kOpsThreads / lanesPerRow(experts);
  const int64_t passes = (tokens + rowsPer - 1) / rowsPer;
  if (passes <= 4) return 1;
  return (int)(passes < 512 ? passes : 512);
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
      const dim3 g(blocks), b(kOpsThreads);
      if (sigmoid) {
        if (index64) hipLaunchKernelGGL((balanceStatsKernel<T, LPR, VPL, true, true>), g, b, 0, s, *a);
        else hipLaunchKernelGGL((balanceStatsKernel<T, LPR, VPL, true, false>), g, b, 0, s, *a);
      } else {
        if (index64) hipLaunchKernelGGL((balanceStatsKernel<T, LPR, VPL, false, true>), g, b, 0, s, *a);
        else hipLaunchKernelGGL((balanceStatsKernel<T, LPR, VPL, false, false>), g, b, 0, s, *a);
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
      const dim3 g((uint32_t)(passes < 4096 ? passes : 4096)), b(kOpsThreads);
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
  hipLaunchKernelGGL(balanceFinishKernel, dim3((a.experts + 1 + 15) / 16), dim3(kOpsThreads), 0, s, a, blocks);
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

// The AdamW step over many tensors (include/msccl_amd_ops.h: mscclAmdAdamWStep) and the tensor tables.
//
// Mathematics, element by element: m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2,
// p = p (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps).  Nothing is used twice, so
// the step is bound by HBM: 28 bytes an element (32-bit weights, or 16-bit ones with a 32-bit copy, and
// 32-bit moments), 16 or 10 with the moments in a byte each.  One launch takes every tensor: a workgroup
// takes 2048-element chunks, and finds the chunk's tensor in the table with one ballot a round.  A lane
// takes 8 neighbours (16-byte loads of 16-bit types), so that a run of 256 elements that share a scale
// is half a wave and its largest magnitude is five lane exchanges away.
#include "ops.h"

namespace msccl {

// ---- tables: written by kernels from their own arguments --------------------------------------
// (stream-ordered and without a host buffer that would have to outlive the call)

constexpr int kTableBytes = 3840;   // (a launch takes 4096 bytes of arguments)
struct TableArgs {
  uint64_t w[kTableBytes / 8];
};

__global__ void __launch_bounds__(256) tableWriteKernel(uint64_t* dst, int words, TableArgs a) {
  for (int i = threadIdx.x; i < words; i += 256) dst[i] = a.w[i];
}

__global__ void __launch_bounds__(256) gradWriteKernel(AdamTensor* rows, int n, TableArgs a) {
  for (int i = threadIdx.x; i < n; i += 256) rows[i].grad = (const void*)a.w[i];
}

int launchTableWrite(void* dst, const void* host, size_t bytes, void* stream) {
  const size_t words = (bytes + 7) / 8;
  constexpr size_t most = kTableBytes / 8;
  for (size_t at = 0; at < words; at += most) {
    TableArgs a;
    const size_t n = words - at < most ? words - at : most;
    __builtin_memcpy(a.w, (const uint64_t*)host + at, n * 8);
    hipLaunchKernelGGL(tableWriteKernel, dim3(1), dim3(256), 0, (hipStream_t)stream, (uint64_t*)dst + at, (int)n, a);
    if (hipGetLastError() != hipSuccess) return 1;
  }
  return 0;
}

int launchGradWrite(AdamTensor* rows, const void* const* grads, size_t n, void* stream) {
  constexpr size_t most = kTableBytes / 8;
  for (size_t at = 0; at < n; at += most) {
    TableArgs a;
    const size_t k = n - at < most ? n - at : most;
    for (size_t i = 0; i < k; i++) a.w[i] = (uint64_t)grads[at + i];
    hipLaunchKernelGGL(gradWriteKernel, dim3(1), dim3(256), 0, (hipStream_t)stream, rows + at, (int)k, a);
    if (hipGetLastError() != hipSuccess) return 1;
  }
  return 0;
}

// ---- the step ----------------------------------------------------------------------------------

// What every element shares, in 64 bits (1 - b2^t loses its digits in 32 for small t): one thread.
__global__ void adamwBeginKernel(AdamStepArgs a) {
  const double s = a.squareSum ? *a.squareSum : 0.0;
  const bool ok = __builtin_isfinite(s);
  const int64_t t = *a.step + (ok ? 1 : 0);
  double p1 = 1.0, p2 = 1.0, q1 = a.beta1, q2 = a.beta2;
  for (uint64_t e = t > 0 ? (uint64_t)t : 0; e; e >>= 1) {   // beta^t by squaring
    if (e & 1) { p1 *= q1; p2 *= q2; }
    q1 *= q1;
    q2 *= q2;
  }
  double c = a.gradScale;
  if (a.squareSum && a.maxNorm > 0) {
    const double clip = a.maxNorm / (a.gradScale * sqrt(s) + 1e-6);
    if (clip < 1.0) c *= clip;
  }
  const double lr = a.lrDevice ? (double)*a.lrDevice : a.lr;
  a.ctl->lr = lr;
  a.ctl->rate = lr / (1.0 - p1);
  a.ctl->invRoot = (float)(1.0 / sqrt(1.0 - p2));
  a.ctl->coef = (float)c;
  a.ctl->skip = !ok;
  if (ok) *a.step = t;
}

// |x| as an integer orders as |x| does, with infinities and NaN on top: its maximum shows both
__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t halfWaveMax(uint32_t x) {
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const uint32_t y = (uint32_t)__shfl_xor((int)x, d, 32);
    x = x > y ? x : y;
  }
  return x;
}

constexpr float kFp8Max = 448.f;
constexpr float kFp8Min = 0.001953125f;   // 2^-9

__device__ __forceinline__ f32x8 decode8(opsU32x2 w, float scale) {
  f32x8 x;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], true);
    x[4 * h] = lo[0];
    x[4 * h + 1] = lo[1];
    x[4 * h + 2] = hi[0];
    x[4 * h + 3] = hi[1];
  }
#pragma unroll
  for (int i = 0; i < 8; i++) x[i] *= scale;
  return x;
}

// Codes and scale of a run (half a wave, 8 values a lane).  FLOOR: no value above zero gets code zero.
// A rounding to 3 fraction bits is off by at most 2^-4 of the value; values under 2^-10 of the unit
// (scale) become zero.
template <bool FLOOR>
__device__ __forceinline__ opsU32x2 encode8(const f32x8& x, float& scale) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const uint32_t y = magnitude(x[i]);
    top = top > y ? top : y;
  }
  top = halfWaveMax(top);
  const float amax = __builtin_bit_cast(float, top);
  const bool finite = top < 0x7f800000u;
  // (below 2^-118 the reciprocal would overflow: such a run reads back as zeros)
  const float inv = finite && amax >= 0x1p-118f ? 1.f / amax * kFp8Max : 0.f;
  scale = finite ? amax * (1.f / kFp8Max) : __builtin_nanf("");
  f32x8 y;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    y[i] = finite ? x[i] * inv : 0.f;
    if (FLOOR && x[i] > 0.f) y[i] = fmaxf(y[i], kFp8Min);
  }
  opsU32x2 w;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], 0, false);
    w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], c, true);
  }
  return w;
}

// What a chunk's lanes share.
struct AdamChunk {
  void* param;
  const void* grad;
  float* master;
  char* m;
  char* v;
  float* mScale;
  float* vScale;
  float coef, invRoot, keep, rate;
};

// A lane's eight elements from `at` on.  FULL: all are there (so that the loads stand together without
// branches); else n are.
template <class P, class G, bool MASTER, int BITS, bool FULL>
__device__ __forceinline__ void adamwEight(const AdamStepArgs& a, const AdamChunk& t, uint64_t at, int some) {
  const int n = FULL ? 8 : some;
  const uint64_t run = at / kStateBlock;
  P* param = (P*)t.param + at;
  float* master = t.master + at;
  char* mAt = t.m + at * (BITS / 8);
  char* vAt = t.v + at * (BITS / 8);
  const f32x8 g = load8((const G*)t.grad + at, n);
  f32x8 p = MASTER ? load8(master, n) : load8(param, n);
  f32x8 m, v, r;
  if constexpr (BITS == 32) {
    m = load8((const float*)mAt, n);
    v = load8((const float*)vAt, n);
  } else {
    const opsU32x2 mc = loadBytes8((const uint8_t*)mAt, n), vc = loadBytes8((const uint8_t*)vAt, n);
    m = decode8(mc, n ? inGlobal(t.mScale)[run] : 0.f);
    v = decode8(vc, n ? inGlobal(t.vScale)[run] : 0.f);
    v = v * v;
  }
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float gi = g[i] * t.coef;
    m[i] = a.b1 * m[i] + a.c1 * gi;
    v[i] = a.b2 * v[i] + a.c2 * (gi * gi);
    r[i] = sqrtf(v[i]);
    p[i] = p[i] * t.keep - t.rate * (m[i] / (r[i] * t.invRoot + a.eps));
  }
  if (MASTER) store8(master, p, n);
  store8(param, p, n);
  if constexpr (BITS == 32) {
    store8((float*)mAt, m, n);
    store8((float*)vAt, v, n);
  } else {
    if (!FULL) {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (i >= n) m[i] = r[i] = 0.f;   // behind the tensor's end: no part of the run's scale
    }
    float ms, vs;
    const opsU32x2 mc = encode8<false>(m, ms), vc = encode8<true>(r, vs);
    storeBytes8((uint8_t*)mAt, mc, n);
    storeBytes8((uint8_t*)vAt, vc, n);
    if (n && (threadIdx.x & 31) == 0) {
      inGlobal(t.mScale)[run] = ms;
      inGlobal(t.vScale)[run] = vs;
    }
  }
}

template <class P, class G, bool MASTER, int BITS>
__global__ void __launch_bounds__(kOpsThreads) adamwKernel(AdamStepArgs a) {
  if (scalarLoad(&a.ctl->skip)) return;
  const float coef = scalarLoad(&a.ctl->coef), invRoot = scalarLoad(&a.ctl->invRoot);
  const double lr = scalarLoad(&a.ctl->lr), rate = scalarLoad(&a.ctl->rate);
  for (uint32_t c = blockIdx.x; c < a.tab.chunks; c += gridDim.x) {
    const uint32_t ti = findTensor(a.tab.starts, a.tab.n, c);
    const AdamTensor* t = a.tab.rows + ti;
    const uint64_t from = (uint64_t)(c - scalarLoad(a.tab.starts + ti)) * kOpsChunk;
    const uint64_t left = scalarLoad(&t->count) - from;
    const double lrScale = scalarLoad(&t->lrScale);
    const AdamChunk k = {scalarLoad(&t->param), scalarLoad(&t->grad), scalarLoad(&t->master), (char*)scalarLoad(&t->m),
                         (char*)scalarLoad(&t->v), scalarLoad(&t->mScale), scalarLoad(&t->vScale), coef, invRoot,
                         (float)(1.0 - lr * lrScale * scalarLoad(&t->decay)), (float)(rate * lrScale)};
    const uint32_t mine = threadIdx.x * kOpsVec;
    if (left >= kOpsChunk) {
      adamwEight<P, G, MASTER, BITS, true>(a, k, from + mine, 8);
    } else {
      const int n = (int)left - (int)mine;
      adamwEight<P, G, MASTER, BITS, false>(a, k, from + mine, n < 0 ? 0 : n > 8 ? 8 : n);
    }
  }
}

template <class P, class G, bool MASTER, int BITS>
static int launchStep(const AdamStepArgs& a, void* stream) {
  constexpr uint32_t most = 1u << 20;   // a launch's threads are counted in 32 bits
  const uint32_t grid = a.tab.chunks < most ? a.tab.chunks : most;
  hipLaunchKernelGGL(adamwBeginKernel, dim3(1), dim3(1), 0, (hipStream_t)stream, a);
  if (hipGetLastError() != hipSuccess) return 1;
  if (grid == 0) return 0;
  hipLaunchKernelGGL((adamwKernel<P, G, MASTER, BITS>), dim3(grid), dim3(kOpsThreads), 0, (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? 0 : 1;
}

template <class P, class G>
static int launchState(const AdamStepArgs& a, bool master, int bits, void* stream) {
  if constexpr (__is_same(P, float)) {
    if (master) return 1;
  } else {
    if (master) return bits == 32 ? launchStep<P, G, true, 32>(a, stream) : launchStep<P, G, true, 8>(a, stream);
  }
  return bits == 32 ? launchStep<P, G, false, 32>(a, stream) : launchStep<P, G, false, 8>(a, stream);
}

template <class P>
static int launchGrad(const AdamStepArgs& a, int gradType, bool master, int bits, void* stream) {
  switch (gradType) {
    case 6: return launchState<P, _Float16>(a, master, bits, stream);
    case 7: return launchState<P, float>(a, master, bits, stream);
    case 9: return launchState<P, __bf16>(a, master, bits, stream);
  }
  return 1;
}

int launchAdamW(const AdamStepArgs& a, int paramType, int gradType, bool master, int bits, void* stream) {
  switch (paramType) {
    case 6: return launchGrad<_Float16>(a, gradType, master, bits, stream);
    case 7: return launchGrad<float>(a, gradType, master, bits, stream);
    case 9: return launchGrad<__bf16>(a, gradType, master, bits, stream);
  }
  return 1;
}

}  // namespace msccl

// The AdamW step over many tensors (include/msccl_amd_ops.h: mscclAmdAdamWStep) and the tensor tables.
//
// Mathematics, element by element: m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2,
// p = p (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps).  Nothing is used twice, so
// the step is bound by HBM: 28 bytes an element (32-bit weights, or 16-bit ones with a 32-bit copy, and
// 32-bit moments), 16 or 10 with the moments in a byte each.  One launch takes every tensor: a workgroup
// takes a chunk, and finds the chunk's tensor in the table with one ballot a round.  A lane takes 4
// neighbours at a time, so that a wave's 32-bit loads and stores are whole lines one after the other:
// twice with 32-bit states (67M weights: 318 us, once 341), once with 8-bit states beside 32-bit tensors
// (134M: 350 us, twice 369).  Where 8-bit states stand beside 16-bit tensors alone it takes 8 neighbours,
// 16 bytes of those (46M: 80 us, twice 4 82, once 4 89).  256 elements that share a scale are then one or
// half a wave's.  That is 5.8 to 6.15 TB/s; loads that do not stream past the caches make it 5.3.
// 8-bit states rounded by chance take 20 more instructions an element, hidden behind the loads where there are
// 32-bit tensors (134M with a 32-bit copy: 348 -> 356 us; 46M 32-bit weights 120 -> 124), not where all are
// narrow (46M bfloat16: 80 -> 95).
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

// What every element shares, in 64 bits (1 - b2^t loses its digits in 32 for small t), from the step
// count that *a.step + 1 makes t (or *a.step, where the step is left out).
__device__ __forceinline__ AdamControl adamwControl(const AdamStepArgs& a, int64_t taken) {
  const double s = a.squareSum ? *a.squareSum : 0.0;
  const bool ok = __builtin_isfinite(s);
  const int64_t t = taken + 1;
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
  AdamControl r;
  r.lr = a.lrDevice ? (double)*a.lrDevice : a.lr;
  r.rate = r.lr / (1.0 - p1);
  r.invRoot = (float)(1.0 / sqrt(1.0 - p2));
  r.coef = (float)c;
  r.t = t;
  r.skip = !ok;
  r.arrived = 0;
  return r;
}

__global__ void adamwBeginKernel(AdamStepArgs a) {
  const int64_t taken = *a.step;
  const AdamControl r = adamwControl(a, taken);
  a.ctl->lr = r.lr;
  a.ctl->rate = r.rate;
  a.ctl->invRoot = r.invRoot;
  a.ctl->coef = r.coef;
  a.ctl->t = r.t;
  a.ctl->skip = r.skip;
  if (!r.skip) *a.step = taken + 1;
}

// |x| as an integer orders as |x| does, with infinities and NaN on top: its maximum shows both
__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

constexpr float kFp8Max = 448.f;
constexpr float kFp8Min = 0.001953125f;   // 2^-9

template <int N>
__device__ __forceinline__ typename VecOf<float, N>::F decode(typename BytesOf<N>::V w, float scale) {
  typename VecOf<float, N>::F x;
#pragma unroll
  for (int h = 0; h < N / 4; h++) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], true);
    x[4 * h] = lo[0] * scale;
    x[4 * h + 1] = lo[1] * scale;
    x[4 * h + 2] = hi[0] * scale;
    x[4 * h + 3] = hi[1] * scale;
  }
  return x;
}

// ---- rounding by chance -------------------------------------------------------------------------
// A step moves an average by less than half a code's step, so that rounded to nearest it would never arrive.
// Numbers that look random, the same again for the same seed, step and place: multiplications by odd
// constants of linear congruential generators, with the high half folded onto the low one between them.

// what a chunk's elements share
__device__ __forceinline__ uint64_t diceOf(uint64_t seed, uint64_t t, uint32_t chunk) {
  constexpr uint64_t a = 6364136223846793005ull, b = 0x9e3779b97f4a7c15ull;
  uint64_t k = seed + t * b;
  k = (k ^ k >> 32) * a;
  k = ((k ^ k >> 29) + chunk) * b;
  k = (k ^ k >> 32) * a;
  return k ^ k >> 32;
}

// the lane's number for its elements from `first` of the chunk on, and the i-th element's
__device__ __forceinline__ uint32_t diceAt(uint64_t key, uint32_t first) {
  uint32_t x = (uint32_t)key + first * 0x9e3779b1u;
  x = (x ^ x >> 16) * 747796405u;
  x = ((x ^ x >> 15) + (uint32_t)(key >> 32)) * 2891336453u;
  return x ^ x >> 16;
}
__device__ __forceinline__ uint32_t throwOf(uint32_t lane, int i) {
  constexpr uint32_t odd[8] = {0x9e3779b1u, 0x7f4a7c15u, 0x2c9277b5u, 0xac564b05u, 0xd3a2646du, 0x58b47f4du, 0xe9846af9u, 0x6c8e9cf5u};
  return lane * odd[i];
}

// y >= 0, at most 448, as one of the two e4m3 values next to it, such that the square is right in the mean:
// the one that is nearest, q, or the other, o, with probability (y^2 - q^2) / (o^2 - q^2).
__device__ __forceinline__ float squareByChance(float y, uint32_t dice) {
  uint32_t e = __builtin_bit_cast(uint32_t, y) & 0x7f800000u;
  e = e > 0x3c800000u ? e : 0x3c800000u;   // under 2^-6 the codes are as far apart as above
  const float m = __builtin_bit_cast(float, e + (20u << 23));   // its unit is the codes' step
  const float q = (y + m) - m, d = y - q;
  const float step = copysignf(__builtin_bit_cast(float, e - (3u << 23)), d), o = q + step;
  return (float)dice * fabsf(step * (o + q)) < fabsf(d * (y + q)) * 0x1p32f ? o : q;
}

// Codes and scale of a run (256 / N lanes, N values each).  SQUARE: the roots of second moments, none above
// zero with code zero.  Without DICE a rounding to 3 fraction bits is off by at most 2^-4 of the value, and
// values under 2^-10 of the unit (scale) become zero; with it, by at most twice that, and in the mean by
// nothing.  Where a value is not finite the scale is NaN, and the codes say nothing.
template <int N, bool SQUARE, bool DICE>
__device__ __forceinline__ typename BytesOf<N>::V encode(const typename VecOf<float, N>::F& x, float& scale, uint32_t dice) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < N; i++) {
    const uint32_t y = magnitude(x[i]);
    top = top > y ? top : y;
  }
  top = umaxOver<kStateBlock / N>(top);
  const float amax = __builtin_bit_cast(float, top);
  // (below 2^-118 the reciprocal would overflow: such a run reads back as zeros)
  const float inv = amax >= 0x1p-118f ? 1.f / amax * kFp8Max : 0.f;
  scale = top < 0x7f800000u ? amax * (1.f / kFp8Max) : __builtin_nanf("");
  float y[N];
#pragma unroll
  for (int i = 0; i < N; i++) {
    y[i] = x[i] * inv;
    if (SQUARE) y[i] = fmaxf(y[i], x[i] > 0.f ? kFp8Min : 0.f);
    // (the two roundings of inv may leave the largest a unit above 448; nearest takes that back)
    if (DICE) y[i] = __builtin_amdgcn_fmed3f(y[i], -kFp8Max, kFp8Max);
    if (DICE && SQUARE) y[i] = squareByChance(y[i], throwOf(dice, i));
  }
  typename BytesOf<N>::V w;
#pragma unroll
  for (int h = 0; h < N / 4; h++) {
    int c = 0;
    if constexpr (DICE && !SQUARE) {
      // the hardware's: it adds the number's upper 20 bits below the last fraction bit and cuts off
      c = __builtin_amdgcn_cvt_sr_fp8_f32(y[4 * h], throwOf(dice, 4 * h) << 13, c, 0);
      c = __builtin_amdgcn_cvt_sr_fp8_f32(y[4 * h + 1], throwOf(dice, 4 * h + 1) << 13, c, 1);
      c = __builtin_amdgcn_cvt_sr_fp8_f32(y[4 * h + 2], throwOf(dice, 4 * h + 2) << 13, c, 2);
      c = __builtin_amdgcn_cvt_sr_fp8_f32(y[4 * h + 3], throwOf(dice, 4 * h + 3) << 13, c, 3);
    } else {
      c = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], c, false);
      c = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], c, true);
    }
    w[h] = (uint32_t)c;
  }
  return w;
}

// Square roots of N values >= 0: one Newton step behind the hardware's estimate, s + (v - s^2) / (2 s), the
// residual exact by FMA, which leaves the rounding of the last addition.  Where a value of the wave is
// below 2^-96 (the residual would lose its digits) or not finite, the library's.
template <int N>
__device__ __forceinline__ typename VecOf<float, N>::F roots(const typename VecOf<float, N>::F& v) {
  constexpr uint32_t low = 0x0f800000u, span = 0x7f800000u - low;
  uint32_t far = 0;
#pragma unroll
  for (int i = 0; i < N; i++) {
    const uint32_t u = __builtin_bit_cast(uint32_t, (float)v[i]) - low;
    far = far > u ? far : u;
  }
  typename VecOf<float, N>::F r;
  if (__builtin_expect(__ballot(far >= span) != 0, 0)) {
#pragma unroll
    for (int i = 0; i < N; i++) r[i] = sqrtf(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float y = __builtin_amdgcn_rsqf(v[i]);
      const float s = v[i] * y;
      r[i] = fmaf(fmaf(-s, s, v[i]), 0.5f * y, s);
    }
  }
  return r;
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
  uint64_t dice;
};

// A lane's elements of a chunk that begins at `from`.  FULL: the whole chunk is there (so that the loads
// stand together without branches); else `left` elements are.
template <class P, class G, bool MASTER, int BITS, bool DICE, bool FULL>
__device__ __forceinline__ void adamwChunk(const AdamStepArgs& a, const AdamChunk& t, uint64_t from, int left) {
  constexpr bool wide = MASTER || sizeof(P) == 4 || sizeof(G) == 4;
  constexpr int N = BITS == 8 && !wide ? 8 : 4;
  constexpr int J = adamEach(BITS, wide) / N;
  constexpr int runLanes = kStateBlock / N;
  typedef typename VecOf<float, N>::F F;
  F g[J], p[J], m[J], v[J];
  typename BytesOf<N>::V mc[J], vc[J];
  float ms[J], vs[J];
#pragma unroll
  for (int j = 0; j < J; j++) {
    const uint32_t mine = (j * kOpsThreads + threadIdx.x) * N;
    const uint64_t at = from + mine;
    const int n = FULL ? N : left - (int)mine;
    g[j] = loadN<N>((const G*)t.grad + at, n);
    if constexpr (MASTER) p[j] = loadN<N>(t.master + at, n);
    else p[j] = loadN<N>((const P*)t.param + at, n);
    if constexpr (BITS == 32) {
      m[j] = loadN<N>((const float*)t.m + at, n);
      v[j] = loadN<N>((const float*)t.v + at, n);
    } else {
      mc[j] = loadBytes<N>((const uint8_t*)t.m + at, n);
      vc[j] = loadBytes<N>((const uint8_t*)t.v + at, n);
      ms[j] = FULL || n > 0 ? inGlobal(t.mScale)[at / kStateBlock] : 0.f;
      vs[j] = FULL || n > 0 ? inGlobal(t.vScale)[at / kStateBlock] : 0.f;
    }
  }
#pragma unroll
  for (int j = 0; j < J; j++) {
    const uint32_t mine = (j * kOpsThreads + threadIdx.x) * N;
    const uint64_t at = from + mine;
    const int n = FULL ? N : left - (int)mine;
    if constexpr (BITS == 8) {
      m[j] = decode<N>(mc[j], ms[j]);
      v[j] = decode<N>(vc[j], vs[j]);
      v[j] = v[j] * v[j];
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float gi = g[j][i] * t.coef;
      m[j][i] = a.b1 * m[j][i] + a.c1 * gi;
      v[j][i] = a.b2 * v[j][i] + a.c2 * (gi * gi);
    }
    F r = roots<N>(v[j]);
#pragma unroll
    for (int i = 0; i < N; i++) {
      // (the reciprocal is within one unit; the denominator is zero or at least 2^-75)
      const float step = m[j][i] * __builtin_amdgcn_rcpf(fmaf(r[i], t.invRoot, a.eps));
      p[j][i] = fmaf(-t.rate, step, p[j][i] * t.keep);
    }
    if constexpr (MASTER) storeN<N>(t.master + at, p[j], n);
    storeN<N>((P*)t.param + at, p[j], n);
    if constexpr (BITS == 32) {
      storeN<N>((float*)t.m + at, m[j], n);
      storeN<N>((float*)t.v + at, v[j], n);
    } else {
      if (!FULL) {
#pragma unroll
        for (int i = 0; i < N; i++)
          if (i >= n) m[j][i] = r[i] = 0.f;   // behind the tensor's end: no part of the run's scale
      }
      const uint32_t dice = DICE ? diceAt(t.dice, mine) : 0;
      const auto mw = encode<N, false, DICE>(m[j], ms[j], dice);
      const auto vw = encode<N, true, DICE>(r, vs[j], dice);
      storeBytes<N>((uint8_t*)t.m + at, mw, n);
      storeBytes<N>((uint8_t*)t.v + at, vw, n);
      if ((FULL || n > 0) && threadIdx.x % runLanes == 0) {
        inGlobal(t.mScale)[at / kStateBlock] = ms[j];
        inGlobal(t.vScale)[at / kStateBlock] = vs[j];
      }
    }
  }
}

// ONE: the step in one launch, every workgroup making what all share by itself.  The last of them to
// have read the step count advances it.
template <class P, class G, bool MASTER, int BITS, bool DICE, bool ONE>
__global__ void __launch_bounds__(kOpsThreads) adamwKernel(AdamStepArgs a) {
  AdamControl ctl;
  if constexpr (ONE) {
    const int64_t taken = __hip_atomic_load(a.step, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // the count has arrived in this lane before the workgroup says so
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::"v"((uint32_t)taken), "v"((uint32_t)(taken >> 32)) : "memory");
    __syncthreads();
    ctl = adamwControl(a, taken);
    if (threadIdx.x == 0 &&
        __hip_atomic_fetch_add(&a.ctl->arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1) {
      __hip_atomic_store(&a.ctl->arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (!ctl.skip) __hip_atomic_store(a.step, taken + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  } else {
    ctl.skip = scalarLoad(&a.ctl->skip);
    ctl.coef = scalarLoad(&a.ctl->coef);
    ctl.invRoot = scalarLoad(&a.ctl->invRoot);
    ctl.lr = scalarLoad(&a.ctl->lr);
    ctl.rate = scalarLoad(&a.ctl->rate);
    if constexpr (DICE) ctl.t = scalarLoad(&a.ctl->t);
  }
  if (ctl.skip) return;
  constexpr uint32_t chunk = adamChunk(BITS, MASTER || sizeof(P) == 4 || sizeof(G) == 4);
  const uint32_t seen = searchStart(a.tab.starts, a.tab.n);
  for (uint32_t c = blockIdx.x; c < a.tab.chunks; c += gridDim.x) {
    const uint32_t ti = findTensor(a.tab.starts, a.tab.n, c, seen);
    const AdamTensor* t = a.tab.rows + ti;
    const uint64_t from = (uint64_t)(c - scalarLoad(a.tab.starts + ti)) * chunk;
    const uint64_t left = scalarLoad(&t->count) - from;
    const double lrScale = scalarLoad(&t->lrScale);
    const AdamChunk k = {scalarLoad(&t->param), scalarLoad(&t->grad), scalarLoad(&t->master), (char*)scalarLoad(&t->m),
                         (char*)scalarLoad(&t->v), scalarLoad(&t->mScale), scalarLoad(&t->vScale), ctl.coef, ctl.invRoot,
                         (float)(1.0 - ctl.lr * lrScale * scalarLoad(&t->decay)), (float)(ctl.rate * lrScale),
                         DICE ? diceOf(a.seed, (uint64_t)ctl.t, c) : 0};
    if (left >= chunk) adamwChunk<P, G, MASTER, BITS, DICE, true>(a, k, from, 0);
    else adamwChunk<P, G, MASTER, BITS, DICE, false>(a, k, from, (int)left);
  }
}

// Up to this many workgroups one launch.  It saves the first launch (3.4 us of the host's time), and costs
// each workgroup the shared values' arithmetic and one atomic on one address, for which they queue at
// 50 ns each: 16 workgroups 4.7 us against 7.6 enqueued one by one and 4.8 against 4.7 in a graph, 64
// 6.3 against 7.6 and 6.5 against 4.8, 512 29 against 7.
constexpr uint32_t kOneLaunch = 32;

template <class P, class G, bool MASTER, int BITS, bool DICE>
static int launchStep(const AdamStepArgs& a, void* stream) {
  constexpr uint32_t most = 1u << 20;   // a launch's threads are counted in 32 bits
  const uint32_t grid = a.tab.chunks < most ? a.tab.chunks : most;
  if (grid && grid <= kOneLaunch) {
    hipLaunchKernelGGL((adamwKernel<P, G, MASTER, BITS, DICE, true>), dim3(grid), dim3(kOpsThreads), 0, (hipStream_t)stream, a);
    return hipGetLastError() == hipSuccess ? 0 : 1;
  }
  hipLaunchKernelGGL(adamwBeginKernel, dim3(1), dim3(1), 0, (hipStream_t)stream, a);
  if (hipGetLastError() != hipSuccess) return 1;
  if (grid == 0) return 0;
  hipLaunchKernelGGL((adamwKernel<P, G, MASTER, BITS, DICE, false>), dim3(grid), dim3(kOpsThreads), 0, (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? 0 : 1;
}

template <class P, class G, bool MASTER>
static int launchBits(const AdamStepArgs& a, int bits, bool dice, void* stream) {
  if (bits == 32) return launchStep<P, G, MASTER, 32, false>(a, stream);
  return dice ? launchStep<P, G, MASTER, 8, true>(a, stream) : launchStep<P, G, MASTER, 8, false>(a, stream);
}

template <class P, class G>
static int launchState(const AdamStepArgs& a, bool master, int bits, bool dice, void* stream) {
  if constexpr (__is_same(P, float)) {
    if (master) return 1;
  } else {
    if (master) return launchBits<P, G, true>(a, bits, dice, stream);
  }
  return launchBits<P, G, false>(a, bits, dice, stream);
}

template <class P>
static int launchGrad(const AdamStepArgs& a, int gradType, bool master, int bits, bool dice, void* stream) {
  switch (gradType) {
    case 6: return launchState<P, _Float16>(a, master, bits, dice, stream);
    case 7: return launchState<P, float>(a, master, bits, dice, stream);
    case 9: return launchState<P, __bf16>(a, master, bits, dice, stream);
  }
  return 1;
}

int launchAdamW(const AdamStepArgs& a, int paramType, int gradType, bool master, int bits, bool dice, void* stream) {
  switch (paramType) {
    case 6: return launchGrad<_Float16>(a, gradType, master, bits, dice, stream);
    case 7: return launchGrad<float>(a, gradType, master, bits, dice, stream);
    case 9: return launchGrad<__bf16>(a, gradType, master, bits, dice, stream);
  }
  return 1;
}

}  // namespace msccl

// The sum of squares of many tensors (include/msccl_amd_ops.h: mscclAmdSquareSum).
//
// Bound by reading each element once.  Products and sums are in 64 bits: the square of a 32-bit value
// is exact there and cannot overflow, and gfx950's 64-bit FMA rate is several times what the loads can
// feed: 67M 32-bit values take 41.5 us (6.5 TB/s), 46M bfloat16 ones in 32 tensors 17.5 with the second
// launch's 3.  Workgroups add up strided chunks into one partial sum each; a second launch of one workgroup
// adds the partial sums in a fixed order, so the result does not depend on timing.
#include "ops.h"

namespace msccl {

template <class T>
__global__ void __launch_bounds__(kSumThreads) squareSumKernel(TensorTable<SumTensor> tab, double* partials) {
  __shared__ double lds[kSumThreads / 64];
  constexpr uint32_t groups = kSumThreads / kOpsThreads;
  const uint32_t group = __builtin_amdgcn_readfirstlane(threadIdx.x / kOpsThreads), lane = threadIdx.x % kOpsThreads;
  constexpr int N = 16 / sizeof(T);
  constexpr uint32_t chunk = sumChunk(sizeof(T));
  double s = 0.0;
  const uint32_t seen = searchStart(tab.starts, tab.n);
  for (uint32_t c = blockIdx.x * groups + group; c < tab.chunks; c += gridDim.x * groups) {
    const uint32_t ti = findTensor(tab.starts, tab.n, c, seen);
    const uint64_t from = (uint64_t)(c - scalarLoad(tab.starts + ti)) * chunk;
    const uint64_t left = scalarLoad(&tab.rows[ti].count) - from;
    const T* data = (const T*)scalarLoad(&tab.rows[ti].data) + from;
    typename VecOf<T, N>::F x[kSumVecs];
    if (left >= chunk) {
#pragma unroll
      for (int j = 0; j < kSumVecs; j++) x[j] = loadN<N>(data + (j * kOpsThreads + lane) * N, N);
    } else {
#pragma unroll
      for (int j = 0; j < kSumVecs; j++) {
        const uint32_t mine = (j * kOpsThreads + lane) * N;
        x[j] = loadN<N>(data + mine, (int)left - (int)mine);
      }
    }
#pragma unroll
    for (int j = 0; j < kSumVecs; j++)
#pragma unroll
      for (int i = 0; i < N; i++) s = fma((double)x[j][i], (double)x[j][i], s);
  }
  s = blockSum<kSumThreads / 64>(s, lds);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

__global__ void __launch_bounds__(kSumBlocks) sumPartialsKernel(const double* partials, int n, double* out) {
  __shared__ double lds[kSumBlocks / 64];
  const double s = blockSum<kSumBlocks / 64>((int)threadIdx.x < n ? partials[threadIdx.x] : 0.0, lds);
  if (threadIdx.x == 0) *out = s;
}

template <class T>
static int launchSum(const TensorTable<SumTensor>& tab, double* out, double* partials, int blocks, void* stream) {
  // one workgroup's partial sum is the sum
  hipLaunchKernelGGL(squareSumKernel<T>, dim3(blocks), dim3(kSumThreads), 0, (hipStream_t)stream, tab,
                     blocks == 1 ? out : partials);
  if (hipGetLastError() != hipSuccess) return 1;
  if (blocks == 1) return 0;
  hipLaunchKernelGGL(sumPartialsKernel, dim3(1), dim3(kSumBlocks), 0, (hipStream_t)stream, partials, blocks, out);
  return hipGetLastError() == hipSuccess ? 0 : 1;
}

int launchSquareSum(const TensorTable<SumTensor>& tab, int type, double* out, double* partials, int blocks, void* stream) {
  switch (type) {
    case 6: return launchSum<_Float16>(tab, out, partials, blocks, stream);
    case 7: return launchSum<float>(tab, out, partials, blocks, stream);
    case 9: return launchSum<__bf16>(tab, out, partials, blocks, stream);
  }
  return 1;
}

}  // namespace msccl

// Training-step operators: argument checks, plans and launches (include/msccl_amd_ops.h).
#include <string.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <new>
#include <utility>
#include <vector>

#include <hip/hip_runtime.h>

#include "../../include/msccl_amd_ops.h"
#include "debug.h"
#include "device/ops.h"

using namespace msccl;

namespace {

constexpr uint64_t kSumMagic = 0x6d73636c53756d31ull, kAdamMagic = 0x6d73636c41646d31ull;

size_t elemSize(int type) {
  switch (type) {
    case ncclFloat32: return 4;
    case ncclFloat16:
    case ncclBfloat16: return 2;
  }
  return 0;
}

bool aligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

#define REFUSE(...) do { WARN(__VA_ARGS__); return ncclInvalidArgument; } while (0)

// [rows][starts], 8-byte multiples
template <class Row>
size_t tableBytes(size_t n) {
  return n * sizeof(Row) + ((n + 1) * sizeof(uint32_t) + 7) / 8 * 8;
}

// the host image of a table; false: more chunks than 32 bits count
template <class Row>
bool makeTable(std::vector<uint64_t>* image, const Row* rows, size_t n, uint32_t chunk, uint32_t* chunks) {
  image->assign(tableBytes<Row>(n) / 8, 0);
  char* at = (char*)image->data();
  if (n) memcpy(at, rows, n * sizeof(Row));
  uint32_t* starts = (uint32_t*)(at + n * sizeof(Row));
  uint64_t c = 0;
  for (size_t i = 0; i < n; i++) {
    starts[i] = (uint32_t)c;
    c += rows[i].count / chunk + (rows[i].count % chunk != 0);
    if (c > 0x7fffffffull) return false;
  }
  starts[n] = (uint32_t)c;
  *chunks = (uint32_t)c;
  return true;
}

template <class Row>
TensorTable<Row> tableAt(void* device, size_t n, uint32_t chunks) {
  return TensorTable<Row>{(const Row*)device, (const uint32_t*)((const char*)device + n * sizeof(Row)), (uint32_t)n, chunks};
}

constexpr size_t kMostTensors = 1u << 20;

typedef std::pair<uintptr_t, uintptr_t> Range;   // first address, and the one behind the last

void addRange(std::vector<Range>* to, const void* p, size_t bytes) {
  if (p && bytes) to->push_back(Range((uintptr_t)p, (uintptr_t)p + bytes));
}

// whether r meets one of these (sorted, apart from each other)
bool meets(const std::vector<Range>& sorted, const Range& r) {
  const auto after = std::lower_bound(sorted.begin(), sorted.end(), Range(r.second, 0));
  return after != sorted.begin() && (after - 1)->second > r.first;
}

}  // namespace

struct mscclAmdSquareSumPlan {
  uint64_t magic;
  int type;
  int blocks;
  TensorTable<SumTensor> tab;
};

struct mscclAmdAdamWPlan {
  uint64_t magic;
  int paramType, gradType, bits;
  bool master;
  int64_t* step;
  AdamControl* ctl;
  AdamTensor* rows;
  TensorTable<AdamTensor> tab;
  std::vector<size_t> counts;
  std::vector<Range> written;   // sorted
  bool dice = false;            // states of 8 bits rounded by chance
  uint64_t seed = 0;
};

extern "C" {

// ---- square sum ------------------------------------------------------------------------------

size_t mscclAmdSquareSumBytes(size_t n) { return n <= kMostTensors ? tableBytes<SumTensor>(n) : 0; }

ncclResult_t mscclAmdSquareSumCreate(mscclAmdSquareSum_t* plan, const void* const* data, const size_t* counts, size_t n,
                                     ncclDataType_t type, void* device, size_t deviceBytes, hipStream_t stream) {
  const char* name = "mscclAmdSquareSumCreate";
  if (!plan) REFUSE("%s : plan argument is NULL", name);
  *plan = nullptr;
  const size_t es = elemSize(type);
  if (!es) REFUSE("%s : invalid type %d", name, (int)type);
  if (n > kMostTensors) REFUSE("%s : %zu tensors, at most %zu", name, n, kMostTensors);
  if (n && (!data || !counts)) REFUSE("%s : tensor list is NULL", name);
  if (!device || !aligned(device, 8) || deviceBytes < tableBytes<SumTensor>(n))
    REFUSE("%s : needs %zu device bytes at an 8-byte boundary", name, tableBytes<SumTensor>(n));
  try {
    std::vector<SumTensor> rows(n);
    for (size_t i = 0; i < n; i++) {
      if (counts[i] && !data[i]) REFUSE("%s : tensor %zu is NULL", name, i);
      if (!aligned(data[i], es)) REFUSE("%s : tensor %zu is not aligned to its elements", name, i);
      rows[i] = SumTensor{data[i], counts[i]};
    }
    std::vector<uint64_t> image;
    uint32_t chunks;
    if (!makeTable(&image, rows.data(), n, sumChunk(es), &chunks)) REFUSE("%s : too many elements", name);
    if (launchTableWrite(device, image.data(), image.size() * 8, stream)) {
      WARN("%s : launch failed", name);
      return ncclUnhandledCudaError;
    }
    constexpr uint32_t groups = kSumThreads / kOpsThreads;
    const uint32_t wanted = chunks <= kSumOne ? 1 : (chunks + groups - 1) / groups;
    const int blocks = wanted < (uint32_t)kSumBlocks ? (int)wanted : kSumBlocks;
    *plan = new mscclAmdSquareSumPlan{kSumMagic, (int)type, blocks, tableAt<SumTensor>(device, n, chunks)};
  } catch (const std::bad_alloc&) {
    WARN("%s : out of host memory", name);
    return ncclSystemError;
  }
  return ncclSuccess;
}

static size_t sumScratch(const mscclAmdSquareSumPlan* plan) { return plan->blocks == 1 ? 0 : plan->blocks * sizeof(double); }

size_t mscclAmdSquareSumWorkspace(mscclAmdSquareSum_t plan) {
  return plan && plan->magic == kSumMagic ? sumScratch(plan) : 0;
}

ncclResult_t mscclAmdSquareSum(mscclAmdSquareSum_t plan, double* out, void* workspace, size_t workspaceBytes,
                               hipStream_t stream) {
  const char* name = "mscclAmdSquareSum";
  if (!plan || plan->magic != kSumMagic) REFUSE("%s : invalid plan", name);
  if (!out || !aligned(out, 8)) REFUSE("%s : out is NULL or not aligned", name);
  if (sumScratch(plan) && (!workspace || !aligned(workspace, 8) || workspaceBytes < sumScratch(plan)))
    REFUSE("%s : needs %zu bytes of workspace at an 8-byte boundary", name, sumScratch(plan));
  if (launchSquareSum(plan->tab, plan->type, out, (double*)workspace, plan->blocks, stream)) {
    WARN("%s : launch failed", name);
    return ncclUnhandledCudaError;
  }
  return ncclSuccess;
}

ncclResult_t mscclAmdSquareSumDestroy(mscclAmdSquareSum_t plan) {
  if (!plan) return ncclSuccess;
  if (plan->magic != kSumMagic) REFUSE("mscclAmdSquareSumDestroy : invalid plan");
  plan->magic = 0;
  delete plan;
  return ncclSuccess;
}

// ---- AdamW -----------------------------------------------------------------------------------

size_t mscclAmdAdamWBytes(size_t n) {
  return n <= kMostTensors ? sizeof(AdamControl) + tableBytes<AdamTensor>(n) : 0;
}

ncclResult_t mscclAmdAdamWCreate(mscclAmdAdamW_t* plan, const mscclAmdAdamWTensor_t* tensors, size_t n,
                                 ncclDataType_t paramType, ncclDataType_t gradType, int stateBits, int64_t* step,
                                 void* device, size_t deviceBytes, hipStream_t stream) {
  const char* name = "mscclAmdAdamWCreate";
  if (!plan) REFUSE("%s : plan argument is NULL", name);
  *plan = nullptr;
  const size_t ps = elemSize(paramType), gs = elemSize(gradType);
  if (!ps || !gs) REFUSE("%s : invalid type %d", name, (int)(ps ? gradType : paramType));
  if (stateBits != 32 && stateBits != 8) REFUSE("%s : states of %d bits (32 or 8)", name, stateBits);
  if (n > kMostTensors) REFUSE("%s : %zu tensors, at most %zu", name, n, kMostTensors);
  if (n && !tensors) REFUSE("%s : tensor list is NULL", name);
  if (!step || !aligned(step, 8)) REFUSE("%s : step is NULL or not aligned", name);
  const size_t need = sizeof(AdamControl) + tableBytes<AdamTensor>(n);
  if (!device || !aligned(device, 8) || deviceBytes < need)
    REFUSE("%s : needs %zu device bytes at an 8-byte boundary", name, need);
  try {
    std::vector<AdamTensor> rows(n);
    std::vector<size_t> counts(n);
    bool master = false, seen = false;
    for (size_t i = 0; i < n; i++) {
      const mscclAmdAdamWTensor_t& t = tensors[i];
      counts[i] = t.count;
      if (t.count) {
        if (!t.param || !t.grad || !t.expAvg || !t.expAvgSq) REFUSE("%s : tensor %zu has a NULL buffer", name, i);
        if (stateBits == 8 && (!t.expAvgScale || !t.expAvgSqScale)) REFUSE("%s : tensor %zu has no scales", name, i);
        if (stateBits == 32 && (t.expAvgScale || t.expAvgSqScale)) REFUSE("%s : tensor %zu has scales for 32-bit states", name, i);
        if (seen && master != (t.master != nullptr)) REFUSE("%s : only some tensors have 32-bit copies", name);
        master = t.master != nullptr;
        seen = true;
        if (master && paramType == ncclFloat32) REFUSE("%s : a 32-bit copy of 32-bit weights", name);
      }
      if (!aligned(t.param, ps) || !aligned(t.grad, gs) || !aligned(t.master, 4) || !aligned(t.expAvgScale, 4) ||
          !aligned(t.expAvgSqScale, 4) || (stateBits == 32 && (!aligned(t.expAvg, 4) || !aligned(t.expAvgSq, 4))))
        REFUSE("%s : tensor %zu is not aligned to its elements", name, i);
      if (!std::isfinite(t.weightDecay) || !std::isfinite(t.lrScale)) REFUSE("%s : tensor %zu: decay or lrScale is not finite", name, i);
      rows[i] = AdamTensor{t.param, t.grad, t.master, t.expAvg, t.expAvgSq, t.expAvgScale, t.expAvgSqScale, t.count, t.weightDecay, t.lrScale};
    }
    // what a step writes lies apart, from itself and from the gradients
    std::vector<Range> written;
    written.reserve(6 * n + 1);
    addRange(&written, step, 8);
    for (const AdamTensor& t : rows) {
      if (t.count > (size_t)1 << 60) REFUSE("%s : too many elements", name);
      const size_t runs = (t.count + kStateBlock - 1) / kStateBlock;
      addRange(&written, t.param, t.count * ps);
      addRange(&written, t.master, t.count * 4);
      addRange(&written, t.m, t.count * (stateBits / 8));
      addRange(&written, t.v, t.count * (stateBits / 8));
      addRange(&written, t.mScale, runs * 4);
      addRange(&written, t.vScale, runs * 4);
    }
    std::sort(written.begin(), written.end());
    for (size_t i = 1; i < written.size(); i++)
      if (written[i - 1].second > written[i].first) REFUSE("%s : buffers overlap (a tensor twice?)", name);
    for (size_t i = 0; i < n; i++)
      if (rows[i].count && meets(written, Range((uintptr_t)rows[i].grad, (uintptr_t)rows[i].grad + rows[i].count * gs)))
        REFUSE("%s : gradient %zu overlaps what the step writes", name, i);
    std::vector<uint64_t> image;
    uint32_t chunks;
    if (!makeTable(&image, rows.data(), n, adamChunk(stateBits, master || ps == 4 || gs == 4), &chunks)) REFUSE("%s : too many elements", name);
    // the control block (zeros) and the table
    image.insert(image.begin(), sizeof(AdamControl) / 8, 0);
    char* table = (char*)device + sizeof(AdamControl);
    if (launchTableWrite(device, image.data(), image.size() * 8, stream)) {
      WARN("%s : launch failed", name);
      return ncclUnhandledCudaError;
    }
    *plan = new mscclAmdAdamWPlan{kAdamMagic, (int)paramType, (int)gradType, stateBits, master, step, (AdamControl*)device,
                              (AdamTensor*)table, tableAt<AdamTensor>(table, n, chunks), std::move(counts), std::move(written)};
  } catch (const std::bad_alloc&) {
    WARN("%s : out of host memory", name);
    return ncclSystemError;
  }
  return ncclSuccess;
}

ncclResult_t mscclAmdAdamWSetRounding(mscclAmdAdamW_t plan, mscclAmdRounding_t rounding, uint64_t seed) {
  const char* name = "mscclAmdAdamWSetRounding";
  if (!plan || plan->magic != kAdamMagic) REFUSE("%s : invalid plan", name);
  if (rounding != mscclAmdNearest && rounding != mscclAmdStochastic) REFUSE("%s : invalid rounding %d", name, (int)rounding);
  if (rounding == mscclAmdStochastic && plan->bits != 8) REFUSE("%s : states of %d bits are rounded to nearest", name, plan->bits);
  plan->dice = rounding == mscclAmdStochastic;
  plan->seed = seed;
  return ncclSuccess;
}

ncclResult_t mscclAmdAdamWSetGrads(mscclAmdAdamW_t plan, const void* const* grads, size_t n, hipStream_t stream) {
  const char* name = "mscclAmdAdamWSetGrads";
  if (!plan || plan->magic != kAdamMagic) REFUSE("%s : invalid plan", name);
  if (n != plan->counts.size()) REFUSE("%s : %zu gradients for %zu tensors", name, n, plan->counts.size());
  if (n && !grads) REFUSE("%s : gradient list is NULL", name);
  for (size_t i = 0; i < n; i++) {
    if (plan->counts[i] && !grads[i]) REFUSE("%s : gradient %zu is NULL", name, i);
    const size_t gs = elemSize(plan->gradType);
    if (!aligned(grads[i], gs)) REFUSE("%s : gradient %zu is not aligned to its elements", name, i);
    if (plan->counts[i] && meets(plan->written, Range((uintptr_t)grads[i], (uintptr_t)grads[i] + plan->counts[i] * gs)))
      REFUSE("%s : gradient %zu overlaps what the step writes", name, i);
  }
  if (launchGradWrite(plan->rows, grads, n, stream)) {
    WARN("%s : launch failed", name);
    return ncclUnhandledCudaError;
  }
  return ncclSuccess;
}

static ncclResult_t checkNumbers(const char* name, double lr, double beta1, double beta2, double eps, double gradScale, double maxNorm) {
  if (!std::isfinite(lr)) REFUSE("%s : lr is not finite", name);
  if (!(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1)) REFUSE("%s : betas (%g, %g) outside [0, 1)", name, beta1, beta2);
  // (a moment that rounds to one times itself would only ever grow)
  if ((float)beta1 == 1.f || (float)beta2 == 1.f) REFUSE("%s : betas (%.17g, %.17g) that are one in 32 bits", name, beta1, beta2);
  if (!(eps == 0 || (eps >= FLT_MIN && eps <= FLT_MAX))) REFUSE("%s : eps %g (0, or a normal 32-bit value)", name, eps);
  if (!(gradScale >= FLT_MIN && gradScale <= FLT_MAX)) REFUSE("%s : gradScale %g (a normal 32-bit value above zero)", name, gradScale);
  if (!(maxNorm >= 0)) REFUSE("%s : maxNorm %g", name, maxNorm);
  return ncclSuccess;
}

ncclResult_t mscclAmdAdamWCheck(double lr, double beta1, double beta2, double eps, double gradScale, double maxNorm) {
  return checkNumbers("mscclAmdAdamWCheck", lr, beta1, beta2, eps, gradScale, maxNorm);
}

ncclResult_t mscclAmdAdamWStep(mscclAmdAdamW_t plan, double lr, const float* lrDevice, double beta1, double beta2,
                               double eps, double gradScale, const double* gradSquareSum, double maxNorm,
                               hipStream_t stream) {
  const char* name = "mscclAmdAdamWStep";
  if (!plan || plan->magic != kAdamMagic) REFUSE("%s : invalid plan", name);
  NCCLCHECK(checkNumbers(name, lr, beta1, beta2, eps, gradScale, maxNorm));
  if (maxNorm > 0 && !gradSquareSum) REFUSE("%s : maxNorm without a square sum", name);
  if (!aligned(gradSquareSum, 8) || !aligned(lrDevice, 4)) REFUSE("%s : gradSquareSum or lrDevice is not aligned", name);
  AdamStepArgs a;
  a.tab = plan->tab;
  a.ctl = plan->ctl;
  a.lr = lr;
  a.lrDevice = lrDevice;
  a.beta1 = beta1;
  a.beta2 = beta2;
  a.gradScale = gradScale;
  a.squareSum = gradSquareSum;
  a.maxNorm = maxNorm;
  a.step = plan->step;
  a.b1 = (float)beta1;
  a.c1 = (float)(1.0 - beta1);   // (1 - 0.999 has no digits to lose in 32 bits)
  a.b2 = (float)beta2;
  a.c2 = (float)(1.0 - beta2);
  a.eps = (float)eps;
  a.seed = plan->seed;
  if (launchAdamW(a, plan->paramType, plan->gradType, plan->master, plan->bits, plan->dice, stream)) {
    WARN("%s : launch failed", name);
    return ncclUnhandledCudaError;
  }
  return ncclSuccess;
}

ncclResult_t mscclAmdAdamWDestroy(mscclAmdAdamW_t plan) {
  if (!plan) return ncclSuccess;
  if (plan->magic != kAdamMagic) REFUSE("mscclAmdAdamWDestroy : invalid plan");
  plan->magic = 0;
  delete plan;
  return ncclSuccess;
}

// ---- balance loss ----------------------------------------------------------------------------

static ncclResult_t checkRouter(const char* name, const mscclAmdRouter_t* r, bool index, BalanceArgs* a) {
  if (!r) REFUSE("%s : router argument is NULL", name);
  const size_t es = elemSize(r->type);
  if (!es) REFUSE("%s : invalid type %d", name, (int)r->type);
  if (r->score != mscclAmdSoftmax && r->score != mscclAmdSigmoid) REFUSE("%s : invalid score %d", name, (int)r->score);
  if (r->experts < 1 || r->experts > (size_t)kMaxExperts) REFUSE("%s : %zu experts (1 to %d)", name, r->experts, kMaxExperts);
  if (r->topK < 1 || r->topK > r->experts) REFUSE("%s : topK %zu of %zu experts", name, r->topK, r->experts);
  if (r->tokens > (size_t)1 << 30) REFUSE("%s : %zu tokens, at most 2^30", name, r->tokens);
  if (r->tokens * r->topK > (size_t)1 << 39) REFUSE("%s : %zu slots, at most 2^39", name, r->tokens * r->topK);
  if (r->logitStride < r->experts || r->logitStride > (size_t)1 << 30) REFUSE("%s : logitStride %zu", name, r->logitStride);
  if (r->tokens && !r->logits) REFUSE("%s : logits is NULL", name);
  if (!aligned(r->logits, es)) REFUSE("%s : logits is not aligned to its elements", name);
  if (index) {
    if (r->indexType != ncclInt32 && r->indexType != ncclInt64) REFUSE("%s : invalid index type %d", name, (int)r->indexType);
    if (r->indexStride < r->topK || r->indexStride > (size_t)1 << 30) REFUSE("%s : indexStride %zu", name, r->indexStride);
    if (r->tokens && !r->index) REFUSE("%s : index is NULL", name);
    if (!aligned(r->index, r->indexType == ncclInt64 ? 8 : 4)) REFUSE("%s : index is not aligned to its elements", name);
  }
  memset(a, 0, sizeof(*a));
  a->logits = r->logits;
  a->tokens = (int64_t)r->tokens;
  a->experts = (int)r->experts;
  a->topK = (int)r->topK;
  a->logitStride = (int64_t)r->logitStride;
  a->index = r->index;
  a->indexStride = (int64_t)r->indexStride;
  a->valid = r->valid;
  return ncclSuccess;
}

size_t mscclAmdBalanceWorkspace(size_t tokens, size_t experts) {
  if (tokens > (size_t)1 << 30 || experts < 1 || experts > (size_t)kMaxExperts) return 0;
  const size_t blocks = (size_t)balanceBlocks((int64_t)tokens, (int)experts);
  return blocks == 1 ? 0 : blocks * (experts * 8 + (experts + 1) * 4);
}

ncclResult_t mscclAmdBalanceStats(const mscclAmdRouter_t* router, int64_t* counts, float* probs, void* workspace,
                                  size_t workspaceBytes, hipStream_t stream) {
  const char* name = "mscclAmdBalanceStats";
  BalanceArgs a;
  NCCLCHECK(checkRouter(name, router, true, &a));
  if (!counts || !probs || !aligned(counts, 8) || !aligned(probs, 4)) REFUSE("%s : counts or probs is NULL or not aligned", name);
  const size_t need = mscclAmdBalanceWorkspace(router->tokens, router->experts);
  if (need && (!workspace || !aligned(workspace, 4) || workspaceBytes < need))
    REFUSE("%s : needs %zu bytes of workspace at a 4-byte boundary", name, need);
  const int blocks = balanceBlocks(a.tokens, a.experts);
  a.counts = counts;
  a.probs = probs;
  a.probPart = (double*)workspace;
  a.countPart = (uint32_t*)workspace + (size_t)blocks * a.experts * 2;
  if (launchBalanceStats(a, router->type, router->indexType == ncclInt64, router->score == mscclAmdSigmoid, blocks, stream)) {
    WARN("%s : launch failed", name);
    return ncclUnhandledCudaError;
  }
  return ncclSuccess;
}

ncclResult_t mscclAmdBalanceLoss(const int64_t* counts, const float* probs, size_t experts, size_t topK, double coef,
                                 float* loss, hipStream_t stream) {
  const char* name = "mscclAmdBalanceLoss";
  if (!counts || !probs || !loss || !aligned(counts, 8) || !aligned(probs, 4) || !aligned(loss, 4))
    REFUSE("%s : an argument is NULL or not aligned", name);
  if (experts < 1 || experts > (size_t)kMaxExperts) REFUSE("%s : %zu experts (1 to %d)", name, experts, kMaxExperts);
  if (topK < 1 || topK > experts) REFUSE("%s : topK %zu of %zu experts", name, topK, experts);
  if (!std::isfinite(coef)) REFUSE("%s : coef is not finite", name);
  if (launchBalanceLoss(counts, probs, (int)experts, coef * (double)experts / (double)topK, loss, stream)) {
    WARN("%s : launch failed", name);
    return ncclUnhandledCudaError;
  }
  return ncclSuccess;
}

ncclResult_t mscclAmdBalanceBackward(const mscclAmdRouter_t* router, const int64_t* counts, double coef,
                                     const float* gradLoss, void* grad, size_t gradStride, int accumulate,
                                     hipStream_t stream) {
  const char* name = "mscclAmdBalanceBackward";
  BalanceArgs a;
  NCCLCHECK(checkRouter(name, router, false, &a));
  if (!counts || !aligned(counts, 8)) REFUSE("%s : counts is NULL or not aligned", name);
  if (!aligned(gradLoss, 4)) REFUSE("%s : gradLoss is not aligned", name);
  if ((a.tokens && !grad) || !aligned(grad, elemSize(router->type))) REFUSE("%s : grad is NULL or not aligned", name);
  if (gradStride < router->experts || gradStride > (size_t)1 << 30) REFUSE("%s : gradStride %zu", name, gradStride);
  if (!std::isfinite(coef)) REFUSE("%s : coef is not finite", name);
  if (grad == router->logits && a.tokens && (accumulate || gradStride != router->logitStride))
    REFUSE("%s : grad is logits, with accumulate or another stride", name);
  a.countsIn = counts;
  a.gradLoss = gradLoss;
  a.grad = grad;
  a.gradStride = (int64_t)gradStride;
  a.scale = coef * (double)a.experts / (double)a.topK;
  if (launchBalanceBackward(a, router->type, router->score == mscclAmdSigmoid, accumulate != 0, stream)) {
    WARN("%s : launch failed", name);
    return ncclUnhandledCudaError;
  }
  return ncclSuccess;
}

}  // extern "C"

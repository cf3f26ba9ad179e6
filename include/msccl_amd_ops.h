/*
 * msccl-amd — operators of a training step that stand beside the collectives.
 *
 * Between ReduceScatter (a rank's gradient shard) and AllGather (its weights): the sum of squares
 * that gradient clipping needs, summed over the ranks by ncclAllReduce in ncclFloat64, and the AdamW
 * step over all of the rank's tensors in one launch, with its states in 32 or in 8 bits.  Beside
 * ncclAllToAll: the counts of the tokens each expert gets and the balance loss of the experts, whose
 * statistics ncclAllReduce sums over the ranks, and its gradient.
 *
 * Every pointer below is a device address of the current device unless it says "host".  Calls return
 * after enqueueing on `stream` and may be captured into a graph; no call allocates or frees device
 * memory, copies between host and device, or waits.  The current device must be the stream's.
 * Results do not depend on timing: the same inputs give the same bits.  Types: ncclFloat32,
 * ncclFloat16, ncclBfloat16.  Tensors need the alignment of their elements only.
 */
#ifndef MSCCL_AMD_OPS_H_
#define MSCCL_AMD_OPS_H_

#include <stddef.h>
#include <stdint.h>
#include "nccl.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- sum of squares of many tensors --------------------------------------------------------- */

typedef struct mscclAmdSquareSumPlan* mscclAmdSquareSum_t;

/* Device bytes a plan over n tensors needs (8-byte aligned), kept by the caller while the plan is used. */
size_t mscclAmdSquareSumBytes(size_t n);

/* A plan over n tensors of one type (data[i]: counts[i] elements; host arrays, read now).  The tensor
 * table is written into `device` on `stream`; later calls on other streams must be ordered after it. */
ncclResult_t mscclAmdSquareSumCreate(mscclAmdSquareSum_t* plan, const void* const* data, const size_t* counts, size_t n,
                                     ncclDataType_t type, void* device, size_t deviceBytes, hipStream_t stream);

/* Device bytes of scratch that one call needs (8-byte aligned; not shared by calls that may overlap);
 * 0 for a few elements, and the workspace is not looked at. */
size_t mscclAmdSquareSumWorkspace(mscclAmdSquareSum_t plan);

/* *out = the sum over all tensors of x * x, every product and sum in 64 bits (a bfloat16 or 32-bit
 * square can pass 32 bits' range).  An infinity or NaN in a tensor shows in the sum. */
ncclResult_t mscclAmdSquareSum(mscclAmdSquareSum_t plan, double* out, void* workspace, size_t workspaceBytes,
                               hipStream_t stream);

/* Frees the host side of the plan (no device call).  NULL is ignored. */
ncclResult_t mscclAmdSquareSumDestroy(mscclAmdSquareSum_t plan);

/* ---- AdamW over many tensors ---------------------------------------------------------------- */

typedef struct mscclAmdAdamWPlan* mscclAmdAdamW_t;

/* One tensor of the step, all pointers to `count` contiguous elements:
 *   param     the weights, paramType; written
 *   grad      the gradient, gradType; read
 *   master    NULL, or the weights in 32 bits: read in place of param, both written (param: rounded)
 *   expAvg, expAvgSq            the moments: 32-bit values, or one byte each (stateBits 8)
 *   expAvgScale, expAvgSqScale  stateBits 8: one 32-bit scale for each run of 256 elements of the
 *                               tensor, (count + 255) / 256 of them; NULL with stateBits 32
 *   weightDecay, lrScale        this tensor's decay, and a factor on its learning rate */
typedef struct {
  void* param;
  const void* grad;
  float* master;
  void* expAvg;
  void* expAvgSq;
  float* expAvgScale;
  float* expAvgSqScale;
  size_t count;
  double weightDecay;
  double lrScale;
} mscclAmdAdamWTensor_t;

size_t mscclAmdAdamWBytes(size_t n);

/* A plan over n tensors (host array, read now; a tensor may be empty).  step: one int64 on the device,
 * the steps taken so far (0 at first), advanced by every step: it and the moments are the optimizer's
 * state, to be saved and loaded with the weights (each plan has its own).  Table and stream as above.
 * Buffers that overlap are refused: a weight that two layers share is listed once.
 * With states in 8 bits expAvg holds e4m3 codes (1 sign, 4 exponent, 3 fraction bits, largest 448) of
 * m / scale, and expAvgSq of sqrt(v) / scale, scale = the run's largest magnitude / 448; a second
 * moment above zero never gets the zero code (its step would be m / eps).  Codes and scales of zero
 * are the state before the first step.  A run that holds an infinity or NaN reads back as NaN.
 * Codes are rounded to nearest unless mscclAmdAdamWSetRounding says otherwise. */
ncclResult_t mscclAmdAdamWCreate(mscclAmdAdamW_t* plan, const mscclAmdAdamWTensor_t* tensors, size_t n,
                                 ncclDataType_t paramType, ncclDataType_t gradType, int stateBits, int64_t* step,
                                 void* device, size_t deviceBytes, hipStream_t stream);

typedef enum { mscclAmdNearest = 0, mscclAmdStochastic = 1 } mscclAmdRounding_t;

/* How the steps enqueued from now on round states of 8 bits (a plan begins with mscclAmdNearest; no
 * device call).  To follow averages over many steps they need mscclAmdStochastic: a code becomes one of
 * the two next to its value, so that m and v (not its root) are right in the mean, step after step.  Which
 * one follows from seed, step count and the element's place in the plan: the same inputs give the same
 * bits again.  One element's root of v is then within about a sixth (beta2 0.999) of the 32-bit state's.
 * mscclAmdNearest is exact to half a code's step (3.1 to 6.3 % of the value) within a step, and loses what
 * changes by less in every step: a decay of the root of v by 1 - sqrt(beta2), 2.5 % at 0.95 and 0.05 % at
 * 0.999, never lowers a code, and an element whose code stays follows its run's scale, so that second
 * moments beside a growing one grow with it for good.  It suits beta2 up to 0.93. */
ncclResult_t mscclAmdAdamWSetRounding(mscclAmdAdamW_t plan, mscclAmdRounding_t rounding, uint64_t seed);

/* Other gradient buffers for all n tensors (host array of device addresses, read now), from `stream`'s
 * next step on.  Captured into a graph it changes them when the graph runs: until then steps read the
 * buffers from before, and every replay sets these again, so both have to live as long. */
ncclResult_t mscclAmdAdamWSetGrads(mscclAmdAdamW_t plan, const void* const* grads, size_t n, hipStream_t stream);

/* One step, with t the advanced step count and g = c * grad:
 *   p = p * (1 - lr * weightDecay), m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2,
 *   p = p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps),  lr times the tensor's lrScale;
 *   c = gradScale, and with a square sum and maxNorm > 0 times min(1, maxNorm / (norm + 1e-6)),
 *   norm = gradScale * sqrt(*gradSquareSum).
 * A square sum that is not finite leaves everything as it was, step included.
 * eps and gradScale are normal 32-bit values (eps may be 0), the betas in [0, 1) in 32
 * bits too.
 *   lrDevice       NULL, or a 32-bit learning rate on the device in place of lr (a captured step
 *                  follows a schedule through it)
 *   gradSquareSum  NULL, or the square sum of the gradients as they are, over all ranks
 * Calls on one plan must be ordered after each other, as calls on one communicator are. */
ncclResult_t mscclAmdAdamWStep(mscclAmdAdamW_t plan, double lr, const float* lrDevice, double beta1, double beta2,
                               double eps, double gradScale, const double* gradSquareSum, double maxNorm,
                               hipStream_t stream);

/* What mscclAmdAdamWStep says to these numbers, without a step: for callers that have to know before they
 * join a collective. */
ncclResult_t mscclAmdAdamWCheck(double lr, double beta1, double beta2, double eps, double gradScale, double maxNorm);

ncclResult_t mscclAmdAdamWDestroy(mscclAmdAdamW_t plan);

/* ---- balance loss of a router's experts ----------------------------------------------------- */

typedef enum { mscclAmdSoftmax = 0, mscclAmdSigmoid = 1 } mscclAmdScore_t;

/* What the router gave for `tokens` tokens over `experts` experts (1 to 1024).  Strides are in
 * elements, from one row to the next. */
typedef struct {
  const void* logits;          /* [tokens][experts] */
  ncclDataType_t type;
  size_t tokens, experts;
  size_t logitStride;          /* at least `experts` */
  const void* index;           /* [tokens][topK]: the chosen experts; one that is not in [0, experts) is a dropped slot */
  ncclDataType_t indexType;    /* ncclInt32 or ncclInt64 */
  size_t topK, indexStride;    /* topK 1 to `experts`; indexStride at least topK */
  const uint8_t* valid;        /* NULL, or one byte a token: zero for padding, whose row is not looked at */
  mscclAmdScore_t score;       /* p = softmax(x), or sigmoid(x) over its sum */
} mscclAmdRouter_t;

/* Scratch bytes of mscclAmdBalanceStats (4-byte aligned; not shared by calls that may overlap); 0 for
 * a few tokens, and the workspace is not looked at. */
size_t mscclAmdBalanceWorkspace(size_t tokens, size_t experts);

/* counts[0..experts): the slots of valid tokens that chose the expert; counts[experts]: the valid
 * tokens.  probs[0..experts): the sum over valid tokens of p, of any finite logits (a p below 2^-100 may
 * be taken as zero), added up in 64 bits and rounded once.  A row whose logits are all -inf adds nothing to probs; one with a NaN logit adds
 * NaN, and under softmax one with a logit of +inf.
 * Summed over the ranks (ncclAllReduce in ncclInt64 and ncclFloat32) they are the whole batch's. */
ncclResult_t mscclAmdBalanceStats(const mscclAmdRouter_t* router, int64_t* counts, float* probs, void* workspace,
                                  size_t workspaceBytes, hipStream_t stream);

/* *loss = coef * experts / (topK * N^2) * sum of counts[e] * probs[e], N = counts[experts]; 0 if N is 0. */
ncclResult_t mscclAmdBalanceLoss(const int64_t* counts, const float* probs, size_t experts, size_t topK, double coef,
                                 float* loss, hipStream_t stream);

/* The loss's gradient at these logits, counts being constants (of all ranks, like the loss's):
 * grad[t][e] = gradLoss * dloss / dx, zero in padded rows (type and shape as logits).
 *   gradLoss    NULL (1), or one 32-bit value
 *   accumulate  nonzero: added to what grad holds, in 32 bits, and rounded once; padded rows stay
 * router->index, indexType, indexStride are not used.  grad may be logits itself without accumulate;
 * otherwise no element of the two is the same. */
ncclResult_t mscclAmdBalanceBackward(const mscclAmdRouter_t* router, const int64_t* counts, double coef,
                                     const float* gradLoss, void* grad, size_t gradStride, int accumulate,
                                     hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif

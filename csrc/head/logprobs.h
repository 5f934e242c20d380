// Launchers of the operators on the logits of a language-model head: log-probabilities of given tokens with the
// entropy and the most likely alternatives, their gradient, and distillation from a teacher's top logits.
// Raw pointers and a stream; every row may start at any address, columns are contiguous.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../common/status.h"

namespace zx {

enum LogitType : int { LOGIT_BF16 = 0, LOGIT_FP16 = 1, LOGIT_FP32 = 2 };

constexpr int kHeadMaxTop = 128;          // most alternatives of a row
constexpr int kHeadMaxVocab = 400000;     // most columns: a row of fp32 fits the shared memory of eight blocks, 200 KB each

// Token numbers, 32 or 64 bits wide; what lies outside [0, V) is absent.
struct IdArray {
  const void* p = nullptr;
  bool wide = true;
};

struct LogprobsArgs {
  const void* logits = nullptr;
  int type = LOGIT_BF16;
  int rows = 0, V = 0;
  int64_t ld = 0;              // elements between two rows
  float temperature = 1.f;
  IdArray targets;             // [rows] or null: no row is left out, no log-probability of a token
  float* logprobs = nullptr;   // [rows] or null
  float* entropy = nullptr;    // [rows]
  float* stats = nullptr;      // [rows, 2] or null in the forward: maximum and sum of the exponentials; 0 sum: no gradient
  int top_k = 0;
  float* top_logprobs = nullptr;   // [rows, top_k]
  int64_t* top_ids = nullptr;      // [rows, top_k]
  // backward
  const float* d_logprobs = nullptr;   // [rows] or null
  const float* d_entropy = nullptr;    // [rows] or null
  const float* d_top = nullptr;        // [rows, top_k] or null
  void* d_logits = nullptr;
  int64_t d_ld = 0;
  int sm_count = 0;
  cudaStream_t stream = nullptr;
};
void launch_token_logprobs_fwd(const LogprobsArgs& a);
void launch_token_logprobs_bwd(const LogprobsArgs& a);

struct DistillArgs {
  const void* logits = nullptr;
  int type = LOGIT_BF16;
  int rows = 0, V = 0;
  int64_t ld = 0;
  float temperature = 1.f;
  const void* values = nullptr;   // [rows, K] teacher log-probabilities (or logits, without the bucket)
  int value_type = LOGIT_FP32;
  IdArray ids;                    // [rows, K]
  int K = 0;
  bool bucket = false;
  float grad_scale = 1.f;
  float* loss = nullptr;          // [rows]
  float* stats = nullptr;         // [rows, 4], written by the forward, read by the backward
  const float* d_loss = nullptr;  // [rows] (backward)
  void* d_logits = nullptr;       // may be the logits themselves
  int64_t d_ld = 0;
  Status* status = nullptr;
  int sm_count = 0;
  cudaStream_t stream = nullptr;
};
void launch_distill_fwd(const DistillArgs& a);       // loss and stats
void launch_distill_bwd(const DistillArgs& a);       // gradient from stats and d_loss
void launch_distill_fwd_bwd(const DistillArgs& a);   // loss and grad_scale * gradient

}  // namespace zx

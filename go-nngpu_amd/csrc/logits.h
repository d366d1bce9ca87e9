// logits.h — host entry points of logits.hip: log-probabilities of given tokens and distillation.
#pragma once

#include "common.h"

namespace gn {

constexpr int kTopMax = 64;       // alternatives to a row
constexpr int kTeacherMax = 256;  // entries of a teacher's row

struct LogitsDesc {
  int dtype;
  const void *x;
  long rows, cols, ld;
  float temperature;
};
struct LogprobsDesc {
  LogitsDesc in;
  const int64_t *targets;
  float *logprob, *lse, *entropy;
  int k;
  int64_t *top_ids;
  float *top_logprobs;
  void *workspace;
  size_t workspace_bytes;
};
struct LogprobsGradDesc {
  LogitsDesc in;
  const int64_t *targets;
  const float *lse, *entropy, *grad_logprob, *grad_entropy;
  void *grad;
  long ldg;
};
struct DistillDesc {
  LogitsDesc in;
  const int64_t *ids;
  const float *teacher;
  int k;
  float *loss, *lse;  // forward
  void *workspace;
  size_t workspace_bytes;
  const float *lse_in, *grad_loss;  // backward
  void *grad;
  long ldg;
};

size_t logits_workspace(long rows, long cols, int k);
// The checks need no device; the launchers expect arguments that passed them.
int check_token_logprobs(const LogprobsDesc &d, CError *err);
int launch_token_logprobs(const LogprobsDesc &d, hipStream_t s, CError *err);
int check_token_logprobs_backward(const LogprobsGradDesc &d, CError *err);
int launch_token_logprobs_backward(const LogprobsGradDesc &d, hipStream_t s, CError *err);
int check_distill_forward(const DistillDesc &d, CError *err);
int launch_distill_forward(const DistillDesc &d, hipStream_t s, CError *err);
int check_distill_backward(const DistillDesc &d, CError *err);
int launch_distill_backward(const DistillDesc &d, hipStream_t s, CError *err);

}  // namespace gn

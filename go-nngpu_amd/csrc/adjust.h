// adjust.h — host entry points of adjust.hip: what is done to logits before they are sampled from, and its gradient.
#pragma once

#include "common.h"

namespace gn {

struct AdjustDesc {
  int dtype;
  const void *x;
  long rows, cols, ld;
  const int64_t *history;
  long h;  // entries of history to a row
  const int64_t *prompt;
  const float *repetition, *frequency, *presence;
  const int64_t *bias_ids;
  const float *bias;
  int biases;
  const uint32_t *mask;
  long ldmask;
  void *out;
  long ldo;
};
struct AdjustGradDesc {
  int dtype;
  const void *x;  // the logits before
  long rows, cols, ld;
  const void *grad_out;
  long ldg;
  const int64_t *history;
  long h;
  const float *repetition;
  const uint32_t *mask;
  long ldmask;
  void *grad;
  long ldo;
};

// The checks need no device; the launchers expect arguments that passed them.
int check_adjust(const AdjustDesc &d, CError *err);
int launch_adjust(const AdjustDesc &d, hipStream_t s, CError *err);
int check_adjust_backward(const AdjustGradDesc &d, CError *err);
int launch_adjust_backward(const AdjustGradDesc &d, hipStream_t s, CError *err);

}  // namespace gn

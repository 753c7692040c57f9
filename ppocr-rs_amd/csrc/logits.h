// Parameter blocks and launchers of the operators on rows of class logits:
// rules (logit_rules.hip), top classes (top_logits.hip), distillation
// (distill.hip).  All pointers are device memory; the C entry points
// (operators.cpp) have checked the shapes.
#pragma once

#include <hip/hip_runtime.h>
#include <cstddef>
#include <cstdint>

#include "kernels.h"

namespace ppocr {

// Largest number of classes of a row (the marks of a row take 32 KB of LDS) and
// largest k (an entry a lane of a wave).
constexpr int kMaxLogitClasses = 1 << 18;
constexpr int kMaxTop = 64;

// Rows of `classes` logits, `stride` elements apart, in storage type `dt`.
struct LogitRows {
  const void* x;
  int64_t rows;
  int classes;
  int64_t stride;
  int dt;
};

// Rules of each row (ppocr_logit_rules): null pointers are absent parts.
struct RuleParams {
  const float* bias;  // [n_bias][classes]
  int64_t n_bias;
  const int32_t* row_bias;  // [rows], or null: row r takes table min(r, n_bias - 1)
  const uint32_t* masks;    // [n_masks][ceil(classes / 32)]
  int64_t n_masks;
  const int32_t* row_mask;  // as row_bias
  const int32_t* history;   // [history_len]
  int64_t history_len;
  const int64_t* offsets;  // [rows + 1]
  const float* repetition;  // [rows] or null
  const float* frequency;
  const float* presence;
};

void launch_logit_rules(const LogitRows& in, const RuleParams& rules, void* out, int64_t out_stride, hipStream_t s);

struct TopParams {
  RuleParams rules;
  int k;
  float temperature;
  float* values;     // [rows][k], or null with pairs
  int32_t* indices;  // [rows][k], or null with pairs
  float* rest;       // [rows] or null
  // Model output form: [rows][k] (class, probability) as floats.
  float* pairs;
  // Equal logits: the highest class first (the order of greedy CTC decoding)
  // instead of the lowest.
  int last_ties;
};
void launch_top_logits(const LogitRows& in, const TopParams& p, hipStream_t s);

struct DistillParams {
  const float* values;     // [rows][k]
  const int32_t* indices;  // [rows][k]
  const float* rest;       // [rows] or null
  int k;
  float temperature;
  const float* grad_loss;  // [rows] or null (ones)
  float* loss;             // [rows] or null
  float* state;            // [rows][4]: written with the loss (or null), read by the gradient alone
  void* grad;              // rows of the student's type, or null
  int64_t grad_stride;
};
// Loss (and state), and with p.grad the gradient, in one pass.
void launch_distill(const LogitRows& student, const DistillParams& p, hipStream_t s);
// The gradient from the state that launch_distill left.
void launch_distill_grad(const LogitRows& student, const DistillParams& p, hipStream_t s);

}  // namespace ppocr

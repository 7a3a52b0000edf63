// Operators on rows of logits in device memory: scores of given tokens
// (log probability, entropy, top alternatives) and distillation from a
// teacher's top alternatives, with their gradients.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/detllm.h"

namespace dtl {

// Logits a wave reduces at a time.  Every sum is formed inside such a segment
// of a row, in a fixed order, and the segments are joined in a fixed order: a
// row's results are the same bits whatever the number of rows, and whether one
// workgroup read the row or many.
constexpr int kScoreSeg = 2048;
constexpr int kScoreMaxVocab = 1 << 18;
constexpr int kScoreMaxSegs = kScoreMaxVocab / kScoreSeg;
constexpr int kScoreMaxTop = 128;
constexpr int kDistillMaxK = 256;
constexpr int kDistillStats = 5;
constexpr float kScoreMinTemperature = 1e-4f, kScoreMaxTemperature = 1e4f;

struct ScoreArgs {
  const void* z;
  size_t stride;
  size_t rows;
  int dtype, vocab;
  const void* tokens;  // int32 or int64 (wide), null: none
  int wide;
  float temperature;
  int top;
  float* log_probs;  // null: not wanted
  float* entropy;    // null: not wanted
  float* stats;      // [rows][2]: m and r; null: not wanted
  int32_t* top_ids;
  float* top_log_probs;
  void* scratch;  // score_scratch_bytes
};
size_t score_scratch_bytes(size_t rows, size_t vocab, size_t top);
void launch_token_scores(const ScoreArgs& a, hipStream_t s);

struct ScoreGradArgs {
  const void* z;
  size_t stride;
  size_t rows;
  int dtype, vocab;
  const void* tokens;
  int wide;
  float temperature;
  const float* stats;
  const float* entropy;
  const float* g_log_probs;  // null: zeros
  const float* g_entropy;    // null: zeros
  void* grad;
  size_t grad_stride;
};
void launch_token_scores_grad(const ScoreGradArgs& a, hipStream_t s);

struct DistillArgs {
  const void* z;
  size_t stride;
  size_t rows;
  int dtype, vocab;
  const void* ids;  // [rows][k] int32 or int64 (wide)
  int wide;
  const float* teacher;  // [rows][k]
  int k;
  float temperature;
  int rest;
  const float* weights;  // [rows], null: ones
  float* loss;           // null: not wanted (backward)
  float* stats;          // [rows][kDistillStats], from the forward to the backward
  void* grad;            // null: forward only
  size_t grad_stride;
  void* scratch;
};
size_t distill_scratch_bytes(size_t rows, size_t vocab, bool step);
void launch_distill(const DistillArgs& a, hipStream_t s);
void launch_distill_grad(const DistillArgs& a, hipStream_t s);

}  // namespace dtl

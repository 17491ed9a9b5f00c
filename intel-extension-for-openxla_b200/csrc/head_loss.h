// Interface between the losses at the vocabulary head (api_head_loss.cu) and their tensor-core kernel (head_loss_sm100.cu).
#pragma once

#include "host_common.h"

namespace ixk {
namespace head {

constexpr int kNoColumn = 0x7fffffff;
constexpr int64_t kDirectRows = 128;    // one row block: no tiles to save, the forward pass takes x as it is

// What a row of the batch is measured against: one label, or a list of columns in ascending order with their weights.
struct Targets {
  const void* labels;       // cross entropy: [rows], int32 or int64; nullptr: lists
  int wide;                 // 64-bit labels
  int64_t ignore_index;
  int apart;                // statistics: the label's column is left out of the sum, the caller makes its logit
  const float* gap;         // labels apart, gradient: of x's rows, the label's p - 1
  const int* column;        // distillation: [rows][entries] ascending, kNoColumn behind the last one
  const float* weight;      // [rows][entries]
  const uint16_t* start;    // [rows][starts]: the first entry at or behind column i * kStartUnit
  int starts;
  int entries;              // 1 for labels
};
constexpr int kStartUnit = 256;

// What the tiles' epilogue needs to know of a row, one 16-byte load.
struct alignas(16) RowInfo {
  int row;                  // of the batch
  int label;                // cross entropy; kNoColumn: none
  float lse2, coef;         // gradient: log-sum-exp, base 2; grad_loss times the logits' and the loss's factors
};

// One pass over columns [first, first + count) of the logits x w^T + bias, tile by tile.
struct Pass {
  int dtype;
  bool w_column_major;      // [hidden, vocab] in memory
  int64_t rows, hidden, vocab;
  const void *x, *w, *bias;
  int64_t ldx, ldw;
  float scale;              // of the logits
  const int* active_rows;   // device: rows of x that there are, nullptr: all
  const RowInfo* info;      // device, of x's rows; nullptr (statistics only): the batch's rows as they are
  int64_t first, count;
  Targets targets;
  // statistics
  float2* partial;          // [slots][rows]: maximum and sum of exponentials, base 2
  float* at_target;         // [batch rows][entries]: scaled logits at the targets (not of labels apart)
  // gradient
  const float* range;       // device: what the gradient is multiplied by
  void* grad;               // [rows up to a multiple of 256][count] of dtype, pitch ldg
  int64_t ldg;
};

// Rows of `partial` that a statistics pass fills.
int stat_slots(int64_t rows, int64_t vocab);

int launch_stats(const Pass& p, const DeviceInfo& dev, cudaStream_t stream);
int launch_grad(const Pass& p, const DeviceInfo& dev, cudaStream_t stream);

}  // namespace head
}  // namespace ixk

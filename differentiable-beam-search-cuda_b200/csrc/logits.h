// Operators on rows of raw logits [rows, V]: sampling, the best log-probs of
// a row, and the distillation loss from a teacher's best log-probs.
//
// Two forms. A row to a thread-block cluster: the row is cut into equal slices,
// one per CTA, each read from HBM once into that CTA's shared memory, and what
// needs the whole row (maximum, sums, thresholds, candidate counts) crosses the
// cluster through distributed shared memory; clusters are persistent, cluster c
// takes rows c, c + n, c + 2n, ... The distillation, and small batches of the
// others. And a scan: CTAs list the candidates of parts of rows without
// waiting for one another, a second kernel finishes each row from its lists,
// and rows that lists do not settle go to the clusters.
#pragma once

#include <cstdint>

#include <cuda_runtime.h>

namespace dbs_logits {

enum DataType : int { kF32 = 0, kF16 = 1, kBF16 = 2 };

// Limits of this implementation.
constexpr int kMaxTop = 1024;                 // entries of a top list, slots of a teacher's row
constexpr int64_t kMaxRowBytes = 3000000;      // a row has to fit 16 CTAs' shared memory;
constexpr int64_t kMaxDistillBytes = 1040000;  // 64 KB of each where it is distilled

struct Rows {
    const void* x = nullptr;
    int dtype = kF32;
    int64_t rows = 0;
    int V = 0;
    int64_t stride = 0;   // elements between rows
};

struct SampleArgs {
    Rows in;
    const float* uniforms = nullptr;      // [rows]
    // per-row settings (device, [rows]); null: the scalar below
    const float* temperature = nullptr;
    const int32_t* top_k = nullptr;
    const float* top_p = nullptr;
    const float* min_p = nullptr;
    float temperature_all = 1.0f;
    int top_k_all = 0;
    float top_p_all = 1.0f;
    float min_p_all = 0.0f;
    int32_t* tokens = nullptr;            // [rows]
    void* space = nullptr;                // sample_space() bytes
    const int* left = nullptr;            // set by the launcher: the rows a kernel takes, their number first
};

struct TopArgs {
    Rows in;
    int n = 0;
    float temperature = 1.0f;
    float* log_probs = nullptr;           // [rows, n]
    int32_t* tokens = nullptr;            // [rows, n]
    void* space = nullptr;                // top_space() bytes
    const int* left = nullptr;            // as above
};

enum Reduction : int { kNone = 0, kSum = 1, kMean = 2 };

struct DistillArgs {
    Rows in;
    const float* teacher_log_probs = nullptr;   // [rows, n]
    const void* teacher_tokens = nullptr;       // [rows, n], int32 or int64
    int token_bytes = 4;
    int n = 0;
    float temperature = 1.0f;
    int tail = 1;
    int reduction = kSum;
    float scale = 1.0f;
    float* row_losses = nullptr;                // [rows]
    float* loss = nullptr;                      // the reduced loss; null with kNone
    void* state = nullptr;                      // distill_state_bytes(); written forward, read backward
    int skip_state = 0;                         // backward: the sums are there already
    int join_losses = 0;                        // set by the launcher: the pass adds up the losses at its end
    void* grad = nullptr;                       // [rows, V] contiguous, the logits' type; null: none
    // backward: gradient of the loss (one value, or one for each row)
    const float* grad_loss = nullptr;
    int64_t grad_loss_stride = 0;
    int skip_unit = 0;                          // grad holds the gradient for grad_loss = 1 already
};

// Device memory that a call needs for what passes between its kernels.
int64_t sample_space(const SampleArgs& a);
int64_t top_space(const TopArgs& a);
cudaError_t launch_sample(const SampleArgs& a, cudaStream_t stream);
cudaError_t launch_top(const TopArgs& a, cudaStream_t stream);
cudaError_t launch_distill(const DistillArgs& a, cudaStream_t stream);
int64_t distill_state_bytes(int64_t rows, int n);
cudaError_t launch_distill_backward(const DistillArgs& a, cudaStream_t stream);

}  // namespace dbs_logits

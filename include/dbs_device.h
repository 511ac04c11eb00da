/*
 * Device-resident extension of the dbs C ABI (not part of the reference's
 * ABI version 10; added beside it without changing any existing symbol).
 *
 * The reference interface takes host arrays and returns host-owned results
 * (include/dbs.h:126-256 of maged15/differentiable-beam-search-cuda). These
 * entry points take DEVICE pointers and a cudaStream_t (passed as void*), run
 * the whole decode / backward as stream-ordered kernel launches, and write
 * results straight into caller-owned device buffers. They are what the
 * PyTorch final_scores autograd Function (the reference's
 * python/torch_dbs_extension.py:233-303) and bench.py call.
 *
 * Output layout ("tight"): example b's [T_b, K_b] selected arrays start at
 * sum_{c<b} T_c*K_c, its [T_b, P_b] pool arrays at sum_{c<b} T_c*P_b and its
 * [K_b] final arrays at sum_{c<b} K_c, with P_b = max(K_b, K_b *
 * relaxed_pool_multiplier). For the uniform batch this is plain [B,T,K],
 * [B,T,P] and [B,K].
 */
#ifndef DBS_B200_DBS_DEVICE_H
#define DBS_B200_DBS_DEVICE_H

#include "dbs.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Device output arrays of one decode call. parents, tokens, lengths and
 * from_logprob are required. When pool_scores is NULL only the top beam_size
 * candidates of every step are selected and no pool / relaxed weights are
 * produced (the selected arrays and final scores are unchanged by this: they
 * are the head of the top-P pool). weights (selected softmax) is produced
 * only when non-NULL; relaxed_weights only with pool_scores. */
typedef struct DBSDeviceDecodeOutputs {
    int32_t* parents;
    int32_t* tokens;
    int32_t* lengths;
    uint8_t* from_logprob;
    float* raw_scores;
    float* scores;
    float* weights;
    int32_t* pool_parents;
    int32_t* pool_tokens;
    int32_t* pool_lengths;
    uint8_t* pool_from_logprob;
    float* pool_raw_scores;
    float* pool_scores;
    float* relaxed_weights;
    float* final_raw_scores;
    float* final_scores;
} DBSDeviceDecodeOutputs;

/* Uniform batch decode of device log_probs [B,T,K,V] (K = beam_size).
 * Replaces dbs_decode_batch (reference include/dbs.h:195-203) for device
 * data. With validate_inputs on, the call waits for the stream and fails with
 * -2 "log_probs contains NaN or +Inf" like the reference; otherwise it
 * returns without synchronising. */
DBS_EXPORT int dbs_device_decode_batch(DBSDecoderHandle* handle, const float* log_probs, int batch_size,
                                       int steps, int vocab_size, const DBSDeviceDecodeOutputs* outputs,
                                       void* cuda_stream);

/* Variable-length constrained batch decode of device log_probs
 * [B, max_steps, max_beam_size, V]: the per-example options of
 * dbs_decode_batch_variable (reference include/dbs.h:205-220) plus the
 * repetition penalty and no-repeat n-gram of dbs_decode_constrained_ex
 * (include/dbs.h:165-172, :74-83), which the reference's variable API cannot
 * take. steps / beams / eos / min_lengths are HOST arrays [B] (NULL = handle
 * default), banned [B,V] and forced [B,max_steps] are DEVICE arrays (NULL =
 * none). Outputs use the tight layout. */
DBS_EXPORT int dbs_device_decode_batch_variable_ex(
    DBSDecoderHandle* handle, const float* log_probs, int batch_size, int max_steps, int max_beam_size,
    int vocab_size, const int32_t* steps_per_example, const int32_t* beam_sizes_per_example,
    const int32_t* eos_tokens_per_example, const int32_t* min_lengths_per_example,
    const uint8_t* banned_tokens_per_example, const int32_t* forced_tokens_per_example,
    float repetition_penalty, int no_repeat_ngram_size, const DBSDeviceDecodeOutputs* outputs,
    void* cuda_stream);

/* Surrogate backward of a uniform batch from its device trace (the
 * reference's dbs_backward_sparse / dbs_backward_dense, include/dbs.h:222-247,
 * batched). Gradient inputs are device arrays in the tight layout or NULL.
 * Exactly one of grad_log_probs (dense [B,T,K,V], fully overwritten) or
 * sparse_indices / sparse_values ([B, T*(K+P)] capacity, example b at
 * b*T*(K+P), indices local to the example's [T*K*V]) with sparse_counts [B]
 * must be given. grad_initial_scores [B,K] is optional. Asynchronous. */
DBS_EXPORT int dbs_device_backward_batch(DBSDecoderHandle* handle, int batch_size, int steps,
                                         int vocab_size, const DBSDeviceDecodeOutputs* trace,
                                         const float* grad_selected_weights,
                                         const float* grad_relaxed_weights,
                                         const float* grad_final_scores, float* grad_log_probs,
                                         int64_t* sparse_indices, float* sparse_values,
                                         int64_t* sparse_counts, float* grad_initial_scores,
                                         void* cuda_stream);

/* dbs_device_decode_batch plus an optional buffer to zero: `zero_fill`
 * (count elements, device) is cleared on a helper stream while the step
 * merge runs, and later work on `cuda_stream` sees the zeros. The autograd
 * path uses it for the dense gradient its backward will scatter into. */
DBS_EXPORT int dbs_device_decode_batch_ex(DBSDecoderHandle* handle, const float* log_probs, int batch_size,
                                          int steps, int vocab_size, const DBSDeviceDecodeOutputs* outputs,
                                          float* zero_fill, int64_t zero_fill_count, void* cuda_stream);

/* dbs_device_backward_batch with flags; DBS_DEVICE_GRAD_PREZEROED means the
 * dense grad_log_probs already holds zeros (e.g. from zero_fill above), so
 * only the non-zero entries are written. */
#define DBS_DEVICE_GRAD_PREZEROED 1
DBS_EXPORT int dbs_device_backward_batch_ex(DBSDecoderHandle* handle, int batch_size, int steps,
                                            int vocab_size, const DBSDeviceDecodeOutputs* trace,
                                            const float* grad_selected_weights,
                                            const float* grad_relaxed_weights,
                                            const float* grad_final_scores, float* grad_log_probs,
                                            int64_t* sparse_indices, float* sparse_values,
                                            int64_t* sparse_counts, float* grad_initial_scores, int flags,
                                            void* cuda_stream);

/* Split decode of a uniform batch for row-sharded multi-GPU runs. The decode
 * is a row scan (every [V] row reduced to its best C candidates, C from
 * dbs_device_row_list_capacity) followed by the sequential step merge.
 * dbs_device_scan_rows scans rows [row_begin, row_end) of the batch (global
 * row r = (b*steps + t)*beam_size + k) into caller-owned device arrays that
 * cover all rows: lists [rows * C] (64-bit entries), list_counts [rows],
 * list_bounds [rows]; it validates the input like dbs_device_decode_batch.
 * Once every row is present (e.g. after an all-gather of each rank's range),
 * dbs_device_merge_rows runs the merge (and weights) and writes the same
 * outputs as dbs_device_decode_batch with the same log_probs. The entry
 * format is internal; only this library's scan produces lists the merge
 * accepts. with_pool must match the outputs' pool_scores (NULL or not).
 * No counterpart in the reference (its CPU decoder has no sharding). */
DBS_EXPORT int dbs_device_row_list_capacity(DBSDecoderHandle* handle, int with_pool, int* capacity);
DBS_EXPORT int dbs_device_scan_rows(DBSDecoderHandle* handle, const float* log_probs, int batch_size, int steps,
                                    int vocab_size, int with_pool, int64_t row_begin, int64_t row_end,
                                    uint64_t* lists, int32_t* list_counts, float* list_bounds, void* cuda_stream);
DBS_EXPORT int dbs_device_merge_rows(DBSDecoderHandle* handle, const float* log_probs, int batch_size, int steps,
                                     int vocab_size, const uint64_t* lists, const int32_t* list_counts,
                                     const float* list_bounds, const DBSDeviceDecodeOutputs* outputs,
                                     void* cuda_stream);

/* Sparse backward of a uniform batch that allocates nothing on its call path:
 * same arguments, outputs and results as dbs_device_backward_batch with
 * sparse outputs (grad_log_probs NULL). For callers that must not allocate
 * device memory where they call it (a caching allocator owns the device, a
 * capture or replay region, a latency-critical loop where cudaMalloc's
 * implicit synchronisation is unacceptable). Its scratch is a static device
 * array of 1 MiB per device, which limits it to batch_size * steps <= 262144,
 * steps <= 510 and beam + pool <= 4096 (-2 with a "takes at most" message
 * beyond them). The first call on a device looks the scratch up and loads
 * the module, so make one call before any region that forbids that. The
 * scratch is shared by all calls on a device: calls must not overlap in time
 * (two streams would race); calls in a row on one stream are fine. No
 * counterpart in the reference, whose backward allocates host memory. */
DBS_EXPORT int dbs_device_backward_sparse_noalloc(DBSDecoderHandle* handle, int batch_size, int steps,
                                                  int vocab_size, const DBSDeviceDecodeOutputs* trace,
                                                  const float* grad_selected_weights,
                                                  const float* grad_relaxed_weights,
                                                  const float* grad_final_scores, int64_t* sparse_indices,
                                                  float* sparse_values, int64_t* sparse_counts,
                                                  float* grad_initial_scores, void* cuda_stream);

/* Operators on rows of raw logits (not log-probs), device data only. The
 * reference has no counterpart: it starts at log-probs and has beam selection
 * alone. Common arguments: `logits` holds `rows` rows of `vocab_size`
 * elements of DBS_DTYPE_F32 / F16 / BF16 (`data_type`), row r at
 * r * row_stride elements (0 repeats one row); rows need no alignment beyond
 * their element's, as all arrays of these calls (others are refused). A row holds at most 3000000 bytes. No handle: errors are
 * in dbs_last_global_error. No call allocates, waits or keeps state, so calls
 * may overlap on several streams and be captured into graphs, each with a
 * workspace of its own: device memory, 16-byte aligned, of at least the bytes
 * that the function beside the call names (NULL where that is 0), whose
 * contents mean nothing before and after the call. */

/* One token per row from uniform numbers in [0, 1). With m the row's maximum
 * (NaN counts as -inf) and weights w_i = exp((x_i - m) / temperature), 0 below
 * exp(-708): order the tokens by (logit desc, token asc); keep the first top_k
 * (all where top_k <= 0), of these those before which less than top_p of their
 * mass lies (all where top_p >= 1), of these those with w >= min_p; the best
 * always. The token is the least kept index at which the sum of kept weights
 * up to and including it exceeds u times their total (the last kept one of
 * positive weight where none does: u of 1 or more, or NaN). temperature <= 0 takes the best
 * token, a row without a value above -inf gives -1. Sums are held in 64 bits.
 * temperatures / top_ks / top_ps / min_ps are per-row settings [rows] or NULL
 * for the value beside them. */
DBS_EXPORT int dbs_device_sample(const void* logits, int data_type, int64_t rows, int vocab_size, int64_t row_stride,
                                 const float* uniforms, const float* temperatures, float temperature,
                                 const int32_t* top_ks, int top_k, const float* top_ps, float top_p,
                                 const float* min_ps, float min_p, int32_t* tokens, void* workspace,
                                 void* cuda_stream);
/* top_k and top_p: the call's, or -1 where it gives top_ks or top_ps. */
DBS_EXPORT int dbs_device_sample_workspace_bytes(int data_type, int64_t rows, int vocab_size, int top_k, float top_p,
                                                 int64_t* bytes);

/* The n best tokens of each row (logit desc, token asc; NaN counts as -inf)
 * and their log-probs under softmax(logits / temperature): log_probs and
 * tokens [rows, n], n <= min(vocab_size, 1024); temperature in [1e-30, 1e30]. Places beyond the tokens above
 * -inf hold -inf and -1. */
DBS_EXPORT int dbs_device_top_log_probs(const void* logits, int data_type, int64_t rows, int vocab_size,
                                        int64_t row_stride, int n, float temperature, float* log_probs,
                                        int32_t* tokens, void* workspace, void* cuda_stream);
DBS_EXPORT int dbs_device_top_log_probs_workspace_bytes(int data_type, int64_t rows, int vocab_size, int n,
                                                        int64_t* bytes);

/* Distillation from a teacher's listed log-probs. teacher_tokens [rows, slots]
 * (int32 or int64: token_bytes 4 or 8) and teacher_log_probs [rows, slots],
 * slots <= 1024; a slot whose token is outside [0, vocab_size) is empty. With
 * P = softmax(logits / temperature), S the listed tokens, q_j = exp of a
 * slot's log-prob, P_r = sum of P outside S, and q_r = max(0, 1 - sum q)
 * where `tail` is set and P_r > 0, else 0, a row's loss is
 *   sum_j q_j (log q_j - log P_j) + q_r (log q_r - log P_r),   0 log 0 = 0,
 * and 0 for a row without slots, whatever its logits hold. P_r > 0 is meant as
 * in 64 bits: exponentials by the row's maximum that add up to less than
 * 2^-1075 (masks by the type's lowest value) are none. `reduction`:
 * DBS_REDUCE_NONE (row_losses [rows] alone; loss NULL), _SUM, or _MEAN over
 * the rows with slots; `scale` multiplies the result. row_losses [rows] is
 * needed for every reduction. grad_logits ([rows, vocab_size] contiguous, the
 * logits' type, or NULL) takes the gradient for an incoming gradient of 1, in
 * the same pass over the logits. `state` is dbs_device_distill_state_bytes
 * bytes of device memory, 16-byte aligned, that the call fills and a backward
 * of it reads. A row holds at most 1040000 bytes here, there are at most
 * 2147483647 rows, and the temperature is in [1e-30, 1e30]. */
#define DBS_REDUCE_NONE 0
#define DBS_REDUCE_SUM 1
#define DBS_REDUCE_MEAN 2
DBS_EXPORT int dbs_device_distill(const void* logits, int data_type, int64_t rows, int vocab_size, int64_t row_stride,
                                  const float* teacher_log_probs, const void* teacher_tokens, int token_bytes,
                                  int slots, float temperature, int tail, int reduction, float scale,
                                  float* row_losses, float* loss, void* state, void* grad_logits,
                                  void* cuda_stream);
DBS_EXPORT int dbs_device_distill_state_bytes(int64_t rows, int slots, int64_t* bytes);

/* The gradient of dbs_device_distill for the incoming gradient grad_loss
 * (device; row r's at r * grad_loss_stride, so 0 for one value). The other
 * arguments are the forward call's, `state` as it wrote it. With
 * DBS_DEVICE_GRAD_UNIT in `flags`, grad_logits is what the forward call wrote,
 * and rows whose incoming gradient is 1 stay as they are. */
#define DBS_DEVICE_GRAD_UNIT 2
DBS_EXPORT int dbs_device_distill_backward(const void* logits, int data_type, int64_t rows, int vocab_size,
                                           int64_t row_stride, int slots, float temperature, int tail, int reduction,
                                           float scale, const void* state,
                                           const float* grad_loss, int64_t grad_loss_stride, int flags,
                                           void* grad_logits, void* cuda_stream);

/* Diagnostics of the most recent device decode whose counters have been read
 * back (process-wide): rows the row scan read a second time from HBM (a
 * speculative threshold, learned from earlier rows, kept fewer entries than
 * the row's list length; the list stays exact) and rows the step merge could
 * not prove complete and rescanned from HBM. No counterpart in the reference. */
DBS_EXPORT int dbs_device_last_rescan_counts(DBSDecoderHandle* handle, int64_t* row_rescans,
                                             int64_t* merge_rescans);

/* Kernel launches this library has queued in this process so far (for
 * benchmarks counting the launches of a timed region). No counterpart in
 * the reference. */
DBS_EXPORT int dbs_device_kernel_launches(int64_t* count);

/* Live kernel timing for benchmarks: enable = 1 starts bracketing every
 * device launch with CUDA events on its stream, 0 stops, -1 clears the
 * totals. dbs_device_profile_read waits for the recorded events and returns
 * the summed device milliseconds and launch count of one kernel:
 * 0 validate, 1 row scan, 2 step merge, 3 weights, 4 zero fill, 5 backward.
 * No counterpart in the reference (its stats hold host wall-clock only,
 * src/differentiable_beam.cpp:3115-3143). */
DBS_EXPORT int dbs_device_profile(int enable);
DBS_EXPORT int dbs_device_profile_read(int kernel, double* total_ms, int64_t* launches);
/* Times only the kernels whose bit (1 << kernel id above) is set in `mask`
 * (0 stops timing), so a benchmark can time one kernel inside a timed region
 * with two events per launch of that kernel and none elsewhere. */
DBS_EXPORT int dbs_device_profile_kernels(unsigned mask);

#ifdef __cplusplus
}
#endif

#endif /* DBS_B200_DBS_DEVICE_H */

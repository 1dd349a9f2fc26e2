// Host entry points of the operators for sequences that share a prompt (shared-prefix attention, page fork / free /
// compact, draws from given uniforms), kept apart from ops.h so those translation units build on their own.
#pragma once
#include <torch/extension.h>

namespace bloom {

// Address of the device's status word, for kernels that report through it.  Refuses to make the word inside a graph
// capture, where it would become part of the graph (zeroed by every replay).  (csrc/kernels/sampling.cu)
int* status_word(int64_t device);

// Decode / verify attention with group-shared prefixes (shared_prefix.cu); items, groups, seqs, tile_rows and
// prefix_splits are those of one plan (ops.shared_prefix_plan).
void shared_prefix_attention(const torch::Tensor& q, const torch::Tensor& kv_cache, int64_t layer,
                             const torch::Tensor& block_table, const torch::Tensor& seq_lens, torch::Tensor& out,
                             const torch::Tensor& items, const torch::Tensor& groups, const torch::Tensor& seqs,
                             int64_t q_len, int64_t tile_rows, int64_t prefix_splits, int64_t suffix_splits,
                             double scale);

// KV pages shared between sequences (pages.cu); kv_cache is any contiguous [L, NB, ...].
std::tuple<torch::Tensor, torch::Tensor> kv_fork(torch::Tensor& kv_cache, const torch::Tensor& block_table,
                                                 const torch::Tensor& seq_lens, const torch::Tensor& parents,
                                                 const torch::Tensor& fresh, torch::Tensor& ref);
void kv_free(const torch::Tensor& block_table, torch::Tensor& seq_lens, const torch::Tensor& rows,
             torch::Tensor& ref);
std::tuple<torch::Tensor, torch::Tensor> kv_compact(torch::Tensor& kv_cache, torch::Tensor& block_table,
                                                    const torch::Tensor& seq_lens, torch::Tensor& ref);

// Draws from given uniforms (draw.cu): u / out [B] or [B, n]; top_k / top_p / min_p per row, absent = off.
void sample_uniform(const torch::Tensor& logits, const torch::Tensor& u, const torch::Tensor& temperature,
                    const c10::optional<torch::Tensor>& top_k, const c10::optional<torch::Tensor>& top_p,
                    const c10::optional<torch::Tensor>& min_p, torch::Tensor& out);

}  // namespace bloom

// Host entry points of the block operators' kernels (rotary.cu, block_norm.cu, fp8.cu) for the
// differentiable operators of block_ops.cpp.
#pragma once

#include <torch/types.h>

#include <tuple>

namespace sb {

void rotary_fwd(const torch::Tensor& q, const c10::optional<torch::Tensor>& k, const torch::Tensor& freq,
                const c10::optional<torch::Tensor>& positions, int64_t pos0, bool interleaved, bool inverse,
                double factor, const torch::Tensor& q_out, const c10::optional<torch::Tensor>& k_out);

void residual_norm_fwd(const torch::Tensor& x, const torch::Tensor& branch, const torch::Tensor& w,
                       const c10::optional<torch::Tensor>& b, const c10::optional<torch::Tensor>& post_w,
                       const c10::optional<torch::Tensor>& post_b, const c10::optional<torch::Tensor>& gate,
                       int64_t gate_div, double eps, double post_eps, double scale, bool layer, bool one_plus,
                       bool round_branch, const torch::Tensor& stream, const torch::Tensor& normed,
                       const c10::optional<torch::Tensor>& stats);
bool residual_norm_bwd_fits(int64_t D, int64_t sums);
bool residual_norm_needs_vectors(int64_t D);
bool residual_norm_vectors(const torch::Tensor& rows);
void residual_norm_bwd(const c10::optional<torch::Tensor>& d_stream, const c10::optional<torch::Tensor>& d_normed,
                       const torch::Tensor& stream, const torch::Tensor& branch, const torch::Tensor& w,
                       const c10::optional<torch::Tensor>& post_w, const c10::optional<torch::Tensor>& post_b,
                       const c10::optional<torch::Tensor>& gate, int64_t gate_div, int64_t gate_mode, double scale,
                       bool layer, bool one_plus, const torch::Tensor& stats, const torch::Tensor& dx,
                       const c10::optional<torch::Tensor>& dbranch, const c10::optional<torch::Tensor>& dw,
                       const c10::optional<torch::Tensor>& db, const c10::optional<torch::Tensor>& dpost_w,
                       const c10::optional<torch::Tensor>& dpost_b, const c10::optional<torch::Tensor>& dgate);

std::tuple<torch::Tensor, torch::Tensor> quantize_fp8(const torch::Tensor& x, int64_t block_rows);
// out = rows x times the weight (transposed: over the weight's rows), see fp8.cu
void fp8_product(const torch::Tensor& x, const torch::Tensor& weight, const torch::Tensor& scale,
                 const c10::optional<torch::Tensor>& bias, bool transposed, const torch::Tensor& out,
                 const torch::Tensor& status);
void gemm_fp8(const torch::Tensor& a, const torch::Tensor& a_scale, const torch::Tensor& weight,
              const torch::Tensor& scale, const c10::optional<torch::Tensor>& bias, const torch::Tensor& out,
              const torch::Tensor& status);

}  // namespace sb

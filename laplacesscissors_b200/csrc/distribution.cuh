// Operators on rows of logits (distribution.cu): log probabilities with entropy and
// top alternatives, distillation from a teacher's top logits, and their gradients.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "lsx.h"

namespace lsx {

// Most slots a row may list (given tokens, alternatives, teacher tokens).
constexpr int kMaxSlots = 128;
// An unused slot of a token list.
constexpr uint32_t kUnusedToken = 0xffffffffu;

// Rows of logits: `stride` elements from one row to the next.
struct LogitRows {
    const void* data;
    lsx_dtype kind;
    size_t rows, vocab, stride;
    double temperature;
};

// lsx_token_logprobs_device; outputs may be NULL.
struct LogprobOutputs {
    float* logprob;
    float* entropy;
    float* stats;
    uint32_t* top_ids;
    float* top_logits;
    float* top_logprobs;
};
cudaError_t launch_token_logprobs(cudaStream_t s, int sm_count, const LogitRows& z, const uint32_t* tokens,
                                  size_t token_count, size_t alternatives, const LogprobOutputs& out);

cudaError_t launch_logprobs_gradient(cudaStream_t s, int sm_count, const LogitRows& z, const uint32_t* tokens,
                                     size_t token_count, const float* stats, const float* entropy,
                                     const float* logprob_gradient, const float* entropy_gradient, void* gradient,
                                     size_t gradient_stride);

// A teacher's listed tokens, [rows x slots].
struct TeacherRows {
    const uint32_t* ids;
    const float* logits;
    const float* stats;  // [rows x 2] or NULL
    size_t slots;
};
cudaError_t launch_distill(cudaStream_t s, int sm_count, const LogitRows& z, const TeacherRows& teacher,
                           const float* weights, float* loss, float* stats, void* gradient, size_t gradient_stride);
cudaError_t launch_distill_gradient(cudaStream_t s, int sm_count, const LogitRows& z, const TeacherRows& teacher,
                                    const float* stats, const float* weights, void* gradient, size_t gradient_stride);

}  // namespace lsx

// Log probabilities of given tokens with the entropy and the best alternatives of every row, and their gradient.
// Formulas and the one pass over a row: token_rows.cuh; kernels: token_stats.cuh.
#include "token_stats.cuh"

using namespace b200;

extern "C" int b200_token_logprobs(const void *logits, const int64_t *tokens, float *logprobs, float *entropy, void *stats,
                                   float *top_logprobs, int64_t *top_tokens, int64_t rows, int64_t V, int64_t stride,
                                   int dtype, int top_k, float temperature, int64_t ignore_index, void *stream) {
    const char *who = "b200_token_logprobs";
    if (const int rc = check_rows(who, logits, rows, V, stride, dtype, temperature)) return rc;
    if (top_k < 0 || top_k > kMaxList || top_k > V) {
        set_error("%s: top_k must lie between 0 and %d and not exceed the vocabulary", who, kMaxList);
        return B200_ERR_ARG;
    }
    if (rows > 0 && (!tokens || !logprobs || !entropy || (top_k > 0 && (!top_logprobs || !top_tokens)) ||
                     !lies_on(stats, 16) || !lies_on(tokens, 8) || !lies_on(top_tokens, 8) || !lies_on(logprobs, 4) ||
                     !lies_on(entropy, 4) || !lies_on(top_logprobs, 4))) {
        set_error("%s: null or misaligned pointer (statistics: 16 bytes)", who);
        return B200_ERR_ARG;
    }
    TokenParams p{};
    p.x = logits;
    p.stride = stride;
    p.rows = rows;
    p.V = int(V);
    p.inv_t = 1.f / temperature;
    p.c = float(1.4426950408889634 / double(temperature));
    p.ids = tokens;
    p.ignore = ignore_index;
    p.K = top_k;
    p.out = logprobs;
    p.entropy = entropy;
    p.stats = static_cast<float4 *>(stats);
    p.top_logprobs = top_logprobs;
    p.top_tokens = top_tokens;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    auto run = [&](auto type) {
        using T = decltype(type);
        return top_k > 0 ? launch_stats<T, kTokens, true>(p, dtype, s) : launch_stats<T, kTokens, false>(p, dtype, s);
    };
    return dtype == B200_F32 ? run(0.f) : dtype == B200_F16 ? run(__half()) : run(__nv_bfloat16());
}

extern "C" int b200_token_logprobs_backward(const void *logits, const int64_t *tokens, const void *stats,
                                            const float *d_logprobs, const float *d_entropy, void *grad_logits,
                                            int64_t rows, int64_t V, int64_t stride, int dtype, float temperature,
                                            int64_t ignore_index, void *stream) {
    const char *who = "b200_token_logprobs_backward";
    if (const int rc = check_rows(who, logits, rows, V, stride, dtype, temperature)) return rc;
    if (rows > 0 && (!tokens || !stats || !grad_logits || !lies_on(stats, 16) || !lies_on(tokens, 8) ||
                     !lies_on(d_logprobs, 4) || !lies_on(d_entropy, 4) || !lies_on(grad_logits, dtype_size(dtype)))) {
        set_error("%s: null or misaligned pointer", who);
        return B200_ERR_ARG;
    }
    TokenGradParams p{};
    p.x = logits;
    p.grad = grad_logits;
    p.stride = stride;
    p.rows = rows;
    p.V = int(V);
    p.inv_t = 1.f / temperature;
    p.c = float(1.4426950408889634 / double(temperature));
    p.ids = tokens;
    p.stats = static_cast<const float4 *>(stats);
    p.d_out = d_logprobs;
    p.d_out_step = 1;
    p.d_entropy = d_entropy;
    p.ignore = ignore_index;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == B200_F32   ? launch_grad<float, kTokens>(p, dtype, s)
           : dtype == B200_F16 ? launch_grad<__half, kTokens>(p, dtype, s)
                               : launch_grad<__nv_bfloat16, kTokens>(p, dtype, s);
}

// The C ABI's attention over packed sequences: checks in the order of capi.h, then
// the launch. Nothing here throws.
#include "cuvit/capi.h"
#include "status.hpp"

#include "../kernels/launch.hpp"

#include <cfloat>
#include <cmath>
#include <cstdint>

namespace cuvit::capi {
namespace {

constexpr int kMaxHeads = 65535;
constexpr int kMaxHeadDim = 256;
constexpr std::int64_t kMaxRows = 0x7FFFFFFF;
/// Tokens of either side: the kernels' walks count them in 32 bits and step past the last
/// one by a block.
constexpr int kMaxTokens = 0x7FFFFFFF - 4095;
/// A token's stride, so that a tile of rows stays within a load's 32-bit offsets.
constexpr std::int64_t kMaxTokenBytes = std::int64_t{1} << 23;
/// The scale times log2(e), the factor of the exponents, is finite.
constexpr float kMaxScale = 0x1p127F;

hipStream_t as_hip(cuvit_stream_t stream) { return reinterpret_cast<hipStream_t>(stream); }

bool aligned(const void* p) { return (reinterpret_cast<std::uintptr_t>(p) & 15U) == 0; }

bool aligned4(const void* p) { return (reinterpret_cast<std::uintptr_t>(p) & 3U) == 0; }

/// Zero strides to the packed ones, of @p heads heads.
detail::TokenStrides resolved(const cuvit_token_strides& s, int heads, int head_dim) {
    return {s.token != 0 ? s.token : static_cast<std::int64_t>(heads) * head_dim, s.head != 0 ? s.head : head_dim};
}

/// An operand's strides: not negative, whole pieces, and none that a launch cannot reach.
int check_strides(const detail::TokenStrides& s, int head_dim, std::int64_t size) {
    if (s.token < 0 || s.head < 0) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention strides cannot be negative");
    }
    const std::int64_t piece = 16 / size;
    if (s.token % piece != 0 || s.head % piece != 0 || s.token < head_dim) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT,
                    "Packed attention strides are whole 16-byte pieces, a token's at least head_dim");
    }
    if (s.token > kMaxTokenBytes / size || s.head > (std::int64_t{1} << 40)) {
        return fail(CUVIT_ERROR_LENGTH, "Packed attention takes token strides of at most 2^23 bytes");
    }
    return ok();
}

/// Whether the rows that strides place lie apart. Strides of an extent of 1 are not used.
bool apart(const detail::TokenStrides& s, std::int64_t tokens, std::int64_t heads, std::int64_t head_dim) {
    if (heads == 1) {
        return tokens == 1 || s.token >= head_dim;
    }
    if (tokens == 1) {
        return s.head >= head_dim;
    }
    return s.head >= head_dim && s.token >= head_dim &&
           (s.token >= s.head * (heads - 1) + head_dim || s.head >= s.token * (tokens - 1) + head_dim);
}

/// The sizes, layouts and limits, of a forward or a backward call alike; @p size is an
/// element's bytes, 0 where only the workspace is asked for.
int check_problem(const cuvit_packed_attention_problem& p, std::int64_t size, detail::PackedArgs* args) {
    if (p.kv_heads <= 0 || p.heads % p.kv_heads != 0) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention needs heads that are a multiple of the key heads");
    }
    if (p.head_dim % 8 != 0 || p.head_dim > kMaxHeadDim) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT,
                    "Packed attention needs a head_dim that is a multiple of 8 and at most 256");
    }
    if (p.scale != 0.0F && !(p.scale >= FLT_MIN && p.scale <= kMaxScale)) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT,
                    "Packed attention needs a positive normal scale of at most 2^127, or 0 for its own");
    }
    if (p.heads > kMaxHeads) {
        return fail(CUVIT_ERROR_LENGTH, "Packed attention takes at most 65535 heads");
    }
    if (static_cast<std::int64_t>(p.tokens) * p.heads > kMaxRows ||
        static_cast<std::int64_t>(p.kv_tokens) * p.kv_heads > kMaxRows) {
        return fail(CUVIT_ERROR_LENGTH, "Packed attention takes at most 2^31 - 1 tokens times heads");
    }
    if (p.tokens > kMaxTokens || p.kv_tokens > kMaxTokens) {
        return fail(CUVIT_ERROR_LENGTH, "Packed attention takes at most 2^31 - 4096 tokens");
    }
    *args = detail::PackedArgs{};
    args->sequences = p.sequences;
    args->tokens = p.tokens;
    args->kv_tokens = p.kv_tokens;
    args->heads = p.heads;
    args->kv_heads = p.kv_heads;
    args->group = p.heads / p.kv_heads;
    args->head_dim = p.head_dim;
    args->scale = p.scale != 0.0F ? p.scale : 1.0F / std::sqrt(static_cast<float>(p.head_dim));
    args->causal = p.causal != 0;
    args->q = resolved(p.q, p.heads, p.head_dim);
    args->k = resolved(p.k, p.kv_heads, p.head_dim);
    args->v = resolved(p.v, p.kv_heads, p.head_dim);
    args->out = resolved(p.out, p.heads, p.head_dim);
    if (size != 0) {
        for (const detail::TokenStrides* s : {&args->q, &args->k, &args->v, &args->out}) {
            if (const int status = check_strides(*s, p.head_dim, size); status != CUVIT_OK) {
                return status;
            }
        }
    }
    return ok();
}

bool negative(const cuvit_packed_attention_problem& p) {
    return p.sequences < 0 || p.tokens < 0 || p.kv_tokens < 0 || p.heads < 0 || p.head_dim < 0;
}

/// What a call without sequences, heads or width has: nothing to do.
bool empty(const cuvit_packed_attention_problem& p) { return p.sequences == 0 || p.heads == 0 || p.head_dim == 0; }

int check_starts(const std::int32_t* starts, const std::int32_t* kv_starts, const std::int32_t* kv_lengths,
                 detail::PackedArgs* args) {
    if (starts == nullptr) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention needs the sequences' starts");
    }
    if (kv_starts == nullptr && args->kv_tokens != args->tokens) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention needs kv_starts where keys are not as many as queries");
    }
    if (!aligned4(starts) || !aligned4(kv_starts) || !aligned4(kv_lengths)) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention needs aligned starts and lengths");
    }
    args->starts = starts;
    args->kv_starts = kv_starts != nullptr ? kv_starts : starts;
    args->kv_lengths = kv_lengths;
    return ok();
}

int check_workspace(const void* workspace, std::int64_t bytes, std::int64_t needed) {
    if (needed > 0 && (workspace == nullptr || !aligned(workspace) || bytes < needed)) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT,
                    "Packed attention needs a 16-byte aligned workspace of the bytes that its problem asks for");
    }
    return ok();
}

int launched(hipError_t result, const char* what) {
    if (result == hipErrorInvalidConfiguration) {
        return fail(CUVIT_ERROR_LENGTH, "Packed attention takes less than 2^32 threads");
    }
    return from_hip(result, what);
}

template <typename T>
int attention(const T* q, const T* k, const T* v, const std::int32_t* starts, const std::int32_t* kv_starts,
              const std::int32_t* kv_lengths, T* out, float* lse, void* workspace, std::int64_t workspace_bytes,
              const cuvit_packed_attention_problem* problem, cuvit_stream_t stream) {
    if (problem == nullptr) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention problem cannot be null");
    }
    const cuvit_packed_attention_problem& p = *problem;
    if (empty(p) || p.tokens == 0) {
        return ok();
    }
    if (negative(p)) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention extents cannot be negative");
    }
    if (q == nullptr || out == nullptr || (p.kv_tokens > 0 && (k == nullptr || v == nullptr))) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention operands cannot be null");
    }
    detail::PackedArgs args{};
    if (const int s = check_problem(p, sizeof(T), &args); s != CUVIT_OK) {
        return s;
    }
    if (const int s = check_starts(starts, kv_starts, kv_lengths, &args); s != CUVIT_OK) {
        return s;
    }
    if (!aligned(q) || !aligned(k) || !aligned(v) || !aligned(out) || !aligned4(lse)) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention operands are 16-byte aligned");
    }
    if (!apart(args.out, p.tokens, p.heads, p.head_dim)) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention output rows overlap");
    }
    if (out == q || out == k || out == v) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention cannot work in place");
    }
    if (const int s = check_workspace(workspace, workspace_bytes, detail::packed_attention_workspace(args));
        s != CUVIT_OK) {
        return s;
    }
    return launched(detail::packed_attention(q, k, v, out, lse, workspace, args, as_hip(stream)),
                    "packed_attention launch");
}

template <typename T>
int backward(const T* q, const T* k, const T* v, const std::int32_t* starts, const std::int32_t* kv_starts,
             const std::int32_t* kv_lengths, const detail::PackedGradients<T>& gradients, std::int64_t workspace_bytes,
             const cuvit_packed_attention_problem* problem, cuvit_stream_t stream) {
    if (problem == nullptr) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention problem cannot be null");
    }
    const cuvit_packed_attention_problem& p = *problem;
    if (empty(p) || (p.tokens == 0 && p.kv_tokens == 0)) {
        return ok();
    }
    if (negative(p)) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention extents cannot be negative");
    }
    if ((p.tokens > 0 && (q == nullptr || gradients.out == nullptr || gradients.lse == nullptr ||
                          gradients.grad_out == nullptr || gradients.grad_q == nullptr)) ||
        (p.kv_tokens > 0 &&
         (k == nullptr || v == nullptr || gradients.grad_k == nullptr || gradients.grad_v == nullptr))) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention operands cannot be null");
    }
    detail::PackedArgs args{};
    if (const int s = check_problem(p, sizeof(T), &args); s != CUVIT_OK) {
        return s;
    }
    if (const int s = check_starts(starts, kv_starts, kv_lengths, &args); s != CUVIT_OK) {
        return s;
    }
    const void* const operands[] = {q, k, v, gradients.out, gradients.grad_out};
    const void* const results[] = {gradients.grad_q, gradients.grad_k, gradients.grad_v};
    for (const void* x : operands) {
        if (!aligned(x)) {
            return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention operands are 16-byte aligned");
        }
    }
    for (const void* result : results) {
        if (!aligned(result)) {
            return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention operands are 16-byte aligned");
        }
        for (const void* x : operands) {
            if (result != nullptr && result == x) {
                return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention cannot work in place");
            }
        }
    }
    if (!aligned4(gradients.lse)) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention operands are 16-byte aligned");
    }
    if ((p.tokens > 0 && !apart(args.q, p.tokens, p.heads, p.head_dim)) ||
        (p.kv_tokens > 0 && (!apart(args.k, p.kv_tokens, p.kv_heads, p.head_dim) ||
                             !apart(args.v, p.kv_tokens, p.kv_heads, p.head_dim)))) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Packed attention gradient rows overlap");
    }
    if (const int s = check_workspace(gradients.workspace, workspace_bytes,
                                      detail::packed_attention_backward_workspace(args));
        s != CUVIT_OK) {
        return s;
    }
    return launched(detail::packed_attention_backward(q, k, v, gradients, args, as_hip(stream)),
                    "packed_attention_backward launch");
}

/// The bytes that @p needed says for a problem that a call would take, else 0.
template <typename Needed> std::int64_t workspace(const cuvit_packed_attention_problem* problem, Needed&& needed) {
    detail::PackedArgs args{};
    if (problem == nullptr || negative(*problem) || empty(*problem) || check_problem(*problem, 0, &args) != CUVIT_OK) {
        return 0;
    }
    return needed(args);
}

} // namespace
} // namespace cuvit::capi

using namespace cuvit;

extern "C" {

void cuvit_packed_attention_problem_init(cuvit_packed_attention_problem* problem, int sequences, int tokens, int heads,
                                         int head_dim) {
    if (problem == nullptr) {
        return;
    }
    *problem = cuvit_packed_attention_problem{};
    problem->sequences = sequences;
    problem->tokens = tokens;
    problem->kv_tokens = tokens;
    problem->heads = heads;
    problem->kv_heads = heads;
    problem->head_dim = head_dim;
}

void cuvit_packed_attention_problem_projection(cuvit_packed_attention_problem* problem) {
    if (problem == nullptr) {
        return;
    }
    const std::int64_t slots = static_cast<std::int64_t>(problem->heads) + 2 * static_cast<std::int64_t>(problem->kv_heads);
    problem->q = {slots * problem->head_dim, problem->head_dim};
    problem->k = problem->q;
    problem->v = problem->q;
}

int64_t cuvit_packed_attention_workspace(const cuvit_packed_attention_problem* problem) {
    return capi::workspace(problem, [](const detail::PackedArgs& args) { return detail::packed_attention_workspace(args); });
}

int cuvit_packed_attention_f32(const float* q, const float* k, const float* v, const int32_t* starts,
                               const int32_t* kv_starts, const int32_t* kv_lengths, float* out, float* lse,
                               void* workspace, int64_t workspace_bytes,
                               const cuvit_packed_attention_problem* problem, cuvit_stream_t stream) {
    return capi::attention(q, k, v, starts, kv_starts, kv_lengths, out, lse, workspace, workspace_bytes, problem, stream);
}

int cuvit_packed_attention_bf16(const cuvit_bf16* q, const cuvit_bf16* k, const cuvit_bf16* v, const int32_t* starts,
                                const int32_t* kv_starts, const int32_t* kv_lengths, cuvit_bf16* out, float* lse,
                                void* workspace, int64_t workspace_bytes,
                                const cuvit_packed_attention_problem* problem, cuvit_stream_t stream) {
    return capi::attention(q, k, v, starts, kv_starts, kv_lengths, out, lse, workspace, workspace_bytes, problem, stream);
}

int64_t cuvit_packed_attention_backward_workspace(const cuvit_packed_attention_problem* problem) {
    return capi::workspace(
        problem, [](const detail::PackedArgs& args) { return detail::packed_attention_backward_workspace(args); });
}

int cuvit_packed_attention_backward_f32(const float* q, const float* k, const float* v, const int32_t* starts,
                                        const int32_t* kv_starts, const int32_t* kv_lengths, const float* out,
                                        const float* lse, const float* grad_out, float* grad_q, float* grad_k,
                                        float* grad_v, void* workspace, int64_t workspace_bytes,
                                        const cuvit_packed_attention_problem* problem, cuvit_stream_t stream) {
    return capi::backward(q, k, v, starts, kv_starts, kv_lengths,
                          detail::PackedGradients<float>{out, lse, grad_out, grad_q, grad_k, grad_v, workspace},
                          workspace_bytes, problem, stream);
}

int cuvit_packed_attention_backward_bf16(const cuvit_bf16* q, const cuvit_bf16* k, const cuvit_bf16* v,
                                         const int32_t* starts, const int32_t* kv_starts, const int32_t* kv_lengths,
                                         const cuvit_bf16* out, const float* lse, const cuvit_bf16* grad_out,
                                         cuvit_bf16* grad_q, cuvit_bf16* grad_k, cuvit_bf16* grad_v, void* workspace,
                                         int64_t workspace_bytes, const cuvit_packed_attention_problem* problem,
                                         cuvit_stream_t stream) {
    return capi::backward(q, k, v, starts, kv_starts, kv_lengths,
                          detail::PackedGradients<cuvit_bf16>{out, lse, grad_out, grad_q, grad_k, grad_v, workspace},
                          workspace_bytes, problem, stream);
}

} // extern "C"

// The C ABI's operators of rotary, gated blocks: checks in the order of capi.h,
// then the launch. Nothing here throws.
#include "cuvit/capi.h"
#include "status.hpp"

#include "../kernels/launch.hpp"

#include <cfloat>
#include <cstdint>
#include <utility>

namespace cuvit::capi {
namespace {

constexpr int kMaxHeads = 65535;
constexpr int kMaxHeadDim = 512;
constexpr std::int64_t kMaxTokens = 0x7FFFFFFF;
/// A gated product's k: its kernels step past the end by up to 1024 values, in int.
constexpr int kMaxDepth = 0x7FFFFFFF - 4095;

hipStream_t as_hip(cuvit_stream_t stream) { return reinterpret_cast<hipStream_t>(stream); }

bool negative(const cuvit_head_strides& s) { return s.image < 0 || s.token < 0 || s.head < 0; }

/// Zero strides to the packed ones.
detail::HeadStrides resolved(const cuvit_head_strides& s, int tokens, int heads, int head_dim) {
    detail::HeadStrides out{};
    out.head = s.head != 0 ? s.head : head_dim;
    out.token = s.token != 0 ? s.token : static_cast<std::int64_t>(heads) * head_dim;
    out.image = s.image != 0 ? s.image : static_cast<std::int64_t>(tokens) * heads * head_dim;
    return out;
}

/// Whether the heads that strides place lie apart: each extent's stride steps
/// past all that the extents of smaller strides span. Strides of an extent of 1
/// are not used.
bool apart(const detail::HeadStrides& s, int images, int tokens, int heads, int head_dim) {
    std::pair<std::int64_t, std::int64_t> order[3] = {{s.head, heads}, {s.token, tokens}, {s.image, images}};
    for (int i = 0; i < 2; ++i) { // three of them, by stride
        for (int j = 0; j < 2 - i; ++j) {
            if (order[j].first > order[j + 1].first) {
                std::swap(order[j], order[j + 1]);
            }
        }
    }
    std::int64_t span = head_dim;
    for (const auto& [stride, extent] : order) {
        if (extent == 1) {
            continue;
        }
        if (stride < span || stride > INT64_MAX / 4 / extent) {
            return false;
        }
        span += stride * (extent - 1);
    }
    return true;
}

/// The checks of a rotation; @p with its operands, into *out.
int check_rotation(const cuvit_rotation& r, int head_dim, const float* positions, const float* frequencies,
                   detail::Rotation* out) {
    if (r.pairing != CUVIT_ROTARY_HALVES && r.pairing != CUVIT_ROTARY_ADJACENT) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Rotary pairing is not a cuvit_rotary_pairing value");
    }
    if (r.axes < 0 || r.axes > 3) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "A rotation takes at most three axes");
    }
    std::int64_t pairs = 0;
    *out = detail::Rotation{};
    for (int axis = 0; axis < r.axes; ++axis) {
        if (r.pairs[axis] < 0) {
            return fail(CUVIT_ERROR_INVALID_ARGUMENT, "An axis cannot have negative pairs");
        }
        if (axis > 0) {
            out->first[axis - 1] = static_cast<int>(pairs);
        }
        pairs += r.pairs[axis];
        if (2 * pairs > head_dim) {
            return fail(CUVIT_ERROR_INVALID_ARGUMENT, "A rotation's pairs exceed the head");
        }
    }
    if (r.position_stride < 0) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "The position stride cannot be negative");
    }
    if (pairs > 0 && (positions == nullptr || frequencies == nullptr)) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "A rotation needs positions and frequencies");
    }
    out->positions = positions;
    out->frequencies = frequencies;
    out->position_stride = r.position_stride;
    out->axes = r.axes;
    out->pairs = static_cast<int>(pairs);
    out->adjacent = r.pairing == CUVIT_ROTARY_ADJACENT;
    return ok();
}

int check_heads(int images, int tokens, int heads, int head_dim) {
    if (head_dim % 2 != 0 || head_dim > kMaxHeadDim) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Rotary heads need an even head_dim of at most 512");
    }
    if (heads > kMaxHeads) {
        return fail(CUVIT_ERROR_LENGTH, "Rotary launches take at most 65535 heads");
    }
    if (static_cast<std::int64_t>(images) * tokens > kMaxTokens) {
        return fail(CUVIT_ERROR_LENGTH, "Rotary launches take at most 2^31 - 1 tokens");
    }
    return ok();
}

int check_rotary(const void* input, const float* positions, const float* frequencies, const void* output,
                 const cuvit_rotary_problem* problem, detail::HeadArgs* args, bool* empty) {
    if (problem == nullptr) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Rotary problem cannot be null");
    }
    const cuvit_rotary_problem& p = *problem;
    *empty = p.images == 0 || p.tokens == 0 || p.heads == 0 || p.head_dim == 0;
    if (*empty) {
        return ok();
    }
    if (p.images < 0 || p.tokens < 0 || p.heads < 0 || p.head_dim < 0) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Rotary extents cannot be negative");
    }
    if (input == nullptr || output == nullptr) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Rotary operands cannot be null");
    }
    *args = detail::HeadArgs{};
    if (const int s = check_rotation(p.rotation, p.head_dim, positions, frequencies, &args->rotation); s != CUVIT_OK) {
        return s;
    }
    if (negative(p.input) || negative(p.output)) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Rotary strides cannot be negative");
    }
    if (const int s = check_heads(p.images, p.tokens, p.heads, p.head_dim); s != CUVIT_OK) {
        return s;
    }
    args->images = p.images;
    args->tokens = p.tokens;
    args->heads = p.heads;
    args->q_heads = p.heads;
    args->head_dim = p.head_dim;
    args->input = resolved(p.input, p.tokens, p.heads, p.head_dim);
    args->output = resolved(p.output, p.tokens, p.heads, p.head_dim);
    args->rotation.inverse = p.inverse != 0;
    args->norm = detail::HeadNorm::kNone;
    if (!apart(args->output, p.images, p.tokens, p.heads, p.head_dim)) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Rotary output heads overlap");
    }
    if (input == output &&
        ((p.images > 1 && args->input.image != args->output.image) ||
         (p.tokens > 1 && args->input.token != args->output.token) ||
         (p.heads > 1 && args->input.head != args->output.head))) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Rotary in place needs equal strides");
    }
    return ok();
}

int check_qk_norm(const void* qkv, const float* positions, const float* frequencies, const void* out,
                  const cuvit_qk_norm_problem* problem, detail::HeadArgs* args, bool* empty) {
    if (problem == nullptr) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "QK norm problem cannot be null");
    }
    const cuvit_qk_norm_problem& p = *problem;
    *empty = p.images == 0 || p.tokens == 0 || p.heads == 0 || p.head_dim == 0;
    if (*empty) {
        return ok();
    }
    if (p.images < 0 || p.tokens < 0 || p.heads < 0 || p.head_dim < 0) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "QK norm extents cannot be negative");
    }
    if (qkv == nullptr || out == nullptr) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "QK norm operands cannot be null");
    }
    if (p.kv_heads <= 0) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "QK norm needs key heads");
    }
    if (p.norm != CUVIT_NORM_RMS && p.norm != CUVIT_NORM_LAYER) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "QK norm is not a cuvit_norm value");
    }
    if (!(p.epsilon >= FLT_MIN && p.epsilon <= FLT_MAX)) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "QK norm needs a positive normal epsilon");
    }
    *args = detail::HeadArgs{};
    if (const int s = check_rotation(p.rotation, p.head_dim, positions, frequencies, &args->rotation); s != CUVIT_OK) {
        return s;
    }
    const std::int64_t slots = static_cast<std::int64_t>(p.heads) + 2 * static_cast<std::int64_t>(p.kv_heads);
    if (const int s = check_heads(p.images, p.tokens, slots > kMaxHeads ? kMaxHeads + 1 : static_cast<int>(slots),
                                  p.head_dim);
        s != CUVIT_OK) {
        return s;
    }
    args->images = p.images;
    args->tokens = p.tokens;
    args->heads = p.heads + p.kv_heads;
    args->q_heads = p.heads;
    args->copied = p.kv_heads;
    args->head_dim = p.head_dim;
    args->input = {p.tokens * slots * p.head_dim, slots * p.head_dim, p.head_dim};
    args->output = args->input;
    args->norm = p.norm == CUVIT_NORM_RMS ? detail::HeadNorm::kRms : detail::HeadNorm::kLayer;
    args->epsilon = p.epsilon;
    return ok();
}

template <typename T>
int rotary(const T* input, const float* positions, const float* frequencies, T* output,
           const cuvit_rotary_problem* problem, cuvit_stream_t stream) {
    detail::HeadArgs args{};
    bool empty = false;
    if (const int s = check_rotary(input, positions, frequencies, output, problem, &args, &empty);
        s != CUVIT_OK || empty) {
        return s;
    }
    return from_hip(detail::rotate_heads(input, output, args, as_hip(stream)), "rotary launch");
}

template <typename T>
int qk_norm(const T* qkv, const float* q_gamma, const float* q_beta, const float* k_gamma, const float* k_beta,
            const float* positions, const float* frequencies, T* out, const cuvit_qk_norm_problem* problem,
            cuvit_stream_t stream) {
    detail::HeadArgs args{};
    bool empty = false;
    if (const int s = check_qk_norm(qkv, positions, frequencies, out, problem, &args, &empty); s != CUVIT_OK || empty) {
        return s;
    }
    args.gamma[0] = q_gamma;
    args.gamma[1] = k_gamma;
    args.beta[0] = q_beta;
    args.beta[1] = k_beta;
    return from_hip(detail::rotate_heads(qkv, out, args, as_hip(stream)), "qk_norm_rotary launch");
}

template <typename T>
int qk_norm_backward(const T* qkv, const float* q_gamma, const float* k_gamma, const float* positions,
                     const float* frequencies, const T* grad_out, T* grad_qkv,
                     const detail::HeadGradients& gradients, std::int64_t workspace_bytes,
                     const cuvit_qk_norm_problem* problem, cuvit_stream_t stream) {
    detail::HeadArgs args{};
    bool empty = false;
    if (const int s = check_qk_norm(qkv, positions, frequencies, grad_qkv, problem, &args, &empty); s != CUVIT_OK) {
        return s;
    }
    const bool summed = gradients.gamma[0] != nullptr || gradients.gamma[1] != nullptr ||
                        gradients.beta[0] != nullptr || gradients.beta[1] != nullptr;
    if (empty) {
        // Sums over no tokens: zeros.
        if (!summed || problem->head_dim <= 0 || problem->heads <= 0) {
            return ok();
        }
        return from_hip(detail::rotate_heads_no_tokens(gradients, problem->head_dim, as_hip(stream)),
                        "qk_norm_rotary_backward launch");
    }
    if (grad_out == nullptr) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "QK norm operands cannot be null");
    }
    if (qkv == grad_qkv) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "QK norm gradients cannot replace the forward's input");
    }
    if (summed && (gradients.workspace == nullptr || (reinterpret_cast<std::uintptr_t>(gradients.workspace) & 15U) != 0 ||
                   workspace_bytes < detail::rotate_heads_workspace(problem->head_dim))) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT,
                    "QK norm gradients need a 16-byte aligned workspace of cuvit_qk_norm_rotary_workspace() bytes");
    }
    args.gamma[0] = q_gamma;
    args.gamma[1] = k_gamma;
    return from_hip(detail::rotate_heads_backward(qkv, grad_out, grad_qkv, gradients, args, as_hip(stream)),
                    "qk_norm_rotary_backward launch");
}

/// The checks that a gated product and its gradient share: the extents m and n,
/// the activation and the leading dimensions of C and the preactivations.
int check_gated_sides(const cuvit_gated_problem* problem, detail::GatedArgs* args, bool* empty) {
    if (problem == nullptr) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Gated problem cannot be null");
    }
    const cuvit_gated_problem& p = *problem;
    *empty = p.m == 0 || p.n == 0;
    if (*empty) {
        return ok();
    }
    if (p.m < 0 || p.n < 0) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Gated dimensions cannot be negative");
    }
    *args = detail::GatedArgs{};
    args->m = p.m;
    args->n = p.n;
    return ok();
}

int check_gated_layout(const cuvit_gated_problem& p, detail::GatedArgs* args) {
    if (p.activation < CUVIT_GATE_SILU || p.activation > CUVIT_GATE_GELU_TANH) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Gated activation is not a cuvit_gate value");
    }
    if (p.m > 0x3FFFFFFF || p.n > 0x3FFFFFFF) {
        return fail(CUVIT_ERROR_LENGTH, "Gated products take at most 2^30 - 1 rows and columns");
    }
    args->gate = static_cast<detail::Gate>(p.activation);
    args->ldc = p.ldc != 0 ? p.ldc : p.n;
    args->ld_pre = p.ld_preactivations != 0 ? p.ld_preactivations : 2 * p.n;
    if (args->ldc < p.n || args->ld_pre < 2 * p.n) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "A gated leading dimension is smaller than its row");
    }
    return ok();
}

/// The checks of a gated product with its operands, into *args.
int check_gated_gemm(const void* a, const void* b, const void* c, const cuvit_gated_problem* problem,
                     detail::GatedArgs* args, bool* empty) {
    if (const int s = check_gated_sides(problem, args, empty); s != CUVIT_OK || *empty) {
        return s;
    }
    const cuvit_gated_problem& p = *problem;
    if (p.k < 0) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Gated dimensions cannot be negative");
    }
    if (a == nullptr || b == nullptr || c == nullptr) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Gated operands cannot be null");
    }
    if (const int s = check_gated_layout(p, args); s != CUVIT_OK) {
        return s;
    }
    if (p.k > kMaxDepth) {
        return fail(CUVIT_ERROR_LENGTH, "Gated products take a k of at most 2^31 - 4096");
    }
    args->k = p.k;
    args->lda = p.lda != 0 ? p.lda : p.k;
    args->ldb = p.ldb != 0 ? p.ldb : p.k;
    if (args->lda < p.k || args->ldb < p.k) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "A gated leading dimension is smaller than its row");
    }
    return ok();
}

int gated_launched(hipError_t launched, const char* what) {
    if (launched == hipErrorInvalidConfiguration) {
        return fail(CUVIT_ERROR_LENGTH, "Gated products take less than 2^32 threads");
    }
    return from_hip(launched, what);
}

template <typename T>
int gated_gemm(const T* a, const T* b, const float* bias, T* c, T* preactivations, const cuvit_gated_problem* problem,
               cuvit_stream_t stream) {
    detail::GatedArgs args{};
    bool empty = false;
    if (const int s = check_gated_gemm(a, b, c, problem, &args, &empty); s != CUVIT_OK || empty) {
        return s;
    }
    return gated_launched(detail::gated_gemm(a, b, bias, c, preactivations, args, as_hip(stream)), "gated_gemm launch");
}

template <typename T>
int gated_checkpoint_gemm(const T* a, const T* b, const float* bias, T* c, std::uint8_t* codes, std::uint8_t* scales,
                          const cuvit_gated_problem* problem, cuvit_stream_t stream) {
    detail::GatedArgs args{};
    bool empty = false;
    if (const int s = check_gated_gemm(a, b, codes != nullptr && scales != nullptr ? c : nullptr, problem, &args, &empty);
        s != CUVIT_OK || empty) {
        return s;
    }
    args.codes = codes;
    args.scales = scales;
    return gated_launched(detail::gated_checkpoint_gemm(a, b, bias, c, args, as_hip(stream)),
                          "gated_checkpoint_gemm launch");
}

template <typename T>
int gated_checkpoint_backward(const std::uint8_t* codes, const std::uint8_t* scales, const T* grad,
                              T* grad_preactivations, T* hidden, const cuvit_gated_problem* problem,
                              cuvit_stream_t stream) {
    detail::GatedArgs args{};
    bool empty = false;
    if (const int s = check_gated_sides(problem, &args, &empty); s != CUVIT_OK || empty) {
        return s;
    }
    if (codes == nullptr || scales == nullptr || grad == nullptr || grad_preactivations == nullptr) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Gated operands cannot be null");
    }
    if (grad == grad_preactivations || hidden == grad_preactivations) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Gated gradients cannot replace the product's gradient");
    }
    if (const int s = check_gated_layout(*problem, &args); s != CUVIT_OK) {
        return s;
    }
    args.codes = const_cast<std::uint8_t*>(codes);
    args.scales = const_cast<std::uint8_t*>(scales);
    return from_hip(detail::gated_checkpoint_backward(grad, grad_preactivations, hidden, args, as_hip(stream)),
                    "gated_checkpoint_backward launch");
}

template <typename T>
int gated_backward(const T* preactivations, const T* grad, T* grad_preactivations, const cuvit_gated_problem* problem,
                   cuvit_stream_t stream) {
    detail::GatedArgs args{};
    bool empty = false;
    if (const int s = check_gated_sides(problem, &args, &empty); s != CUVIT_OK || empty) {
        return s;
    }
    if (preactivations == nullptr || grad == nullptr || grad_preactivations == nullptr) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Gated operands cannot be null");
    }
    if (grad == grad_preactivations) {
        return fail(CUVIT_ERROR_INVALID_ARGUMENT, "Gated gradients cannot replace the product's gradient");
    }
    if (const int s = check_gated_layout(*problem, &args); s != CUVIT_OK) {
        return s;
    }
    return from_hip(detail::gated_backward(preactivations, grad, grad_preactivations, args, as_hip(stream)),
                    "gated_backward launch");
}

cuvit_rotation packed_rotation(int axes, const int* pairs, int pairing) {
    cuvit_rotation rotation{};
    rotation.pairing = pairing;
    rotation.axes = axes;
    for (int axis = 0; axis < axes && axis < 3 && pairs != nullptr; ++axis) {
        rotation.pairs[axis] = pairs[axis];
    }
    return rotation;
}

detail::HeadGradients gradients_of(float* q_gamma, float* q_beta, float* k_gamma, float* k_beta, void* workspace) {
    return {{q_gamma, k_gamma}, {q_beta, k_beta}, static_cast<float*>(workspace)};
}

} // namespace
} // namespace cuvit::capi

using namespace cuvit;

extern "C" {

void cuvit_rotary_problem_init(cuvit_rotary_problem* problem, int images, int tokens, int heads, int head_dim,
                               int axes, const int* pairs, int pairing) {
    if (problem == nullptr) {
        return;
    }
    *problem = cuvit_rotary_problem{};
    problem->images = images;
    problem->tokens = tokens;
    problem->heads = heads;
    problem->head_dim = head_dim;
    problem->rotation = capi::packed_rotation(axes, pairs, pairing);
}

int cuvit_rotary_f32(const float* input, const float* positions, const float* frequencies, float* output,
                     const cuvit_rotary_problem* problem, cuvit_stream_t stream) {
    return capi::rotary(input, positions, frequencies, output, problem, stream);
}

int cuvit_rotary_bf16(const cuvit_bf16* input, const float* positions, const float* frequencies, cuvit_bf16* output,
                      const cuvit_rotary_problem* problem, cuvit_stream_t stream) {
    return capi::rotary(input, positions, frequencies, output, problem, stream);
}

void cuvit_qk_norm_problem_init(cuvit_qk_norm_problem* problem, int images, int tokens, int heads, int head_dim,
                                int axes, const int* pairs, int pairing, int norm) {
    if (problem == nullptr) {
        return;
    }
    *problem = cuvit_qk_norm_problem{};
    problem->images = images;
    problem->tokens = tokens;
    problem->heads = heads;
    problem->kv_heads = heads;
    problem->head_dim = head_dim;
    problem->norm = norm;
    problem->epsilon = 1.0e-6F;
    problem->rotation = capi::packed_rotation(axes, pairs, pairing);
}

int cuvit_qk_norm_rotary_f32(const float* qkv, const float* q_gamma, const float* q_beta, const float* k_gamma,
                             const float* k_beta, const float* positions, const float* frequencies, float* out,
                             const cuvit_qk_norm_problem* problem, cuvit_stream_t stream) {
    return capi::qk_norm(qkv, q_gamma, q_beta, k_gamma, k_beta, positions, frequencies, out, problem, stream);
}

int cuvit_qk_norm_rotary_bf16(const cuvit_bf16* qkv, const float* q_gamma, const float* q_beta, const float* k_gamma,
                              const float* k_beta, const float* positions, const float* frequencies, cuvit_bf16* out,
                              const cuvit_qk_norm_problem* problem, cuvit_stream_t stream) {
    return capi::qk_norm(qkv, q_gamma, q_beta, k_gamma, k_beta, positions, frequencies, out, problem, stream);
}

int64_t cuvit_qk_norm_rotary_workspace(const cuvit_qk_norm_problem* problem) {
    return problem != nullptr && problem->head_dim > 0 && problem->head_dim <= capi::kMaxHeadDim
               ? detail::rotate_heads_workspace(problem->head_dim)
               : 0;
}

int cuvit_qk_norm_rotary_backward_f32(const float* qkv, const float* q_gamma, const float* k_gamma,
                                      const float* positions, const float* frequencies, const float* grad_out,
                                      float* grad_qkv, float* grad_q_gamma, float* grad_q_beta, float* grad_k_gamma,
                                      float* grad_k_beta, void* workspace, int64_t workspace_bytes,
                                      const cuvit_qk_norm_problem* problem, cuvit_stream_t stream) {
    return capi::qk_norm_backward(qkv, q_gamma, k_gamma, positions, frequencies, grad_out, grad_qkv,
                                  capi::gradients_of(grad_q_gamma, grad_q_beta, grad_k_gamma, grad_k_beta, workspace),
                                  workspace_bytes, problem, stream);
}

int cuvit_qk_norm_rotary_backward_bf16(const cuvit_bf16* qkv, const float* q_gamma, const float* k_gamma,
                                       const float* positions, const float* frequencies, const cuvit_bf16* grad_out,
                                       cuvit_bf16* grad_qkv, float* grad_q_gamma, float* grad_q_beta,
                                       float* grad_k_gamma, float* grad_k_beta, void* workspace,
                                       int64_t workspace_bytes, const cuvit_qk_norm_problem* problem,
                                       cuvit_stream_t stream) {
    return capi::qk_norm_backward(qkv, q_gamma, k_gamma, positions, frequencies, grad_out, grad_qkv,
                                  capi::gradients_of(grad_q_gamma, grad_q_beta, grad_k_gamma, grad_k_beta, workspace),
                                  workspace_bytes, problem, stream);
}

void cuvit_gated_problem_init(cuvit_gated_problem* problem, int m, int n, int k, int activation) {
    if (problem == nullptr) {
        return;
    }
    *problem = cuvit_gated_problem{};
    problem->m = m;
    problem->n = n;
    problem->k = k;
    problem->activation = activation;
}

int cuvit_gated_gemm_f32(const float* a, const float* b, const float* bias, float* c, float* preactivations,
                         const cuvit_gated_problem* problem, cuvit_stream_t stream) {
    return capi::gated_gemm(a, b, bias, c, preactivations, problem, stream);
}

int cuvit_gated_gemm_bf16(const cuvit_bf16* a, const cuvit_bf16* b, const float* bias, cuvit_bf16* c,
                          cuvit_bf16* preactivations, const cuvit_gated_problem* problem, cuvit_stream_t stream) {
    return capi::gated_gemm(a, b, bias, c, preactivations, problem, stream);
}

int cuvit_gated_backward_f32(const float* preactivations, const float* grad, float* grad_preactivations,
                             const cuvit_gated_problem* problem, cuvit_stream_t stream) {
    return capi::gated_backward(preactivations, grad, grad_preactivations, problem, stream);
}

int cuvit_gated_backward_bf16(const cuvit_bf16* preactivations, const cuvit_bf16* grad,
                              cuvit_bf16* grad_preactivations, const cuvit_gated_problem* problem,
                              cuvit_stream_t stream) {
    return capi::gated_backward(preactivations, grad, grad_preactivations, problem, stream);
}

int64_t cuvit_gated_checkpoint_scales(const cuvit_gated_problem* problem) {
    return problem != nullptr && problem->m > 0 && problem->n > 0
               ? 2 * static_cast<std::int64_t>(problem->m) * ((static_cast<std::int64_t>(problem->n) + 31) / 32)
               : 0;
}

int cuvit_gated_checkpoint_gemm_f32(const float* a, const float* b, const float* bias, float* c, uint8_t* codes,
                                    uint8_t* scales, const cuvit_gated_problem* problem, cuvit_stream_t stream) {
    return capi::gated_checkpoint_gemm(a, b, bias, c, codes, scales, problem, stream);
}

int cuvit_gated_checkpoint_gemm_bf16(const cuvit_bf16* a, const cuvit_bf16* b, const float* bias, cuvit_bf16* c,
                                     uint8_t* codes, uint8_t* scales, const cuvit_gated_problem* problem,
                                     cuvit_stream_t stream) {
    return capi::gated_checkpoint_gemm(a, b, bias, c, codes, scales, problem, stream);
}

int cuvit_gated_checkpoint_backward_f32(const uint8_t* codes, const uint8_t* scales, const float* grad,
                                        float* grad_preactivations, float* hidden, const cuvit_gated_problem* problem,
                                        cuvit_stream_t stream) {
    return capi::gated_checkpoint_backward(codes, scales, grad, grad_preactivations, hidden, problem, stream);
}

int cuvit_gated_checkpoint_backward_bf16(const uint8_t* codes, const uint8_t* scales, const cuvit_bf16* grad,
                                         cuvit_bf16* grad_preactivations, cuvit_bf16* hidden,
                                         const cuvit_gated_problem* problem, cuvit_stream_t stream) {
    return capi::gated_checkpoint_backward(codes, scales, grad, grad_preactivations, hidden, problem, stream);
}

} // extern "C"

// Operators next to the routed-MoE layer (libnetra_layers.so): the block-FP8
// linear layer y = x W^T with its gradients, the root-mean-square norm before it
// (output in 8 bits too) with its gradients, the routing to experts with its gradient, per-expert
// route counts, the router's balance loss with its gradient, and low-rank
// adapters beside a projection.
//
// Block-FP8 linear layer. W [n, k] is e4m3 with one fp32 scale per 128x128
// block (scale grid [ceil(n/128), ceil(k/128)], row-major), as a block-FP8
// checkpoint holds every dense projection; n, k and the rows go up to 2^21 each
// (a call whose workgroups do not fit a launch, of outputs beyond the memory, is
// refused), the last block of n or k may be short. Activations are quantised inside the call by the
// MoE layer's rule: per 1x128, scale = max(amax, 1e-10) * 0x3b124925, code =
// e4m3_rne(v * (1 / scale)). A 128-group that holds an infinity or NaN gets the
// scale NaN, so every output it reaches is NaN. Products are accumulated in
// fp32 per 128-block: acc += (s_x * s_w) * mfma.
//
//   forward          y[t, n]  = sum_b s_x[t, b] s_w[n/128, b] sum_{k in b} q_x q_w
//   input gradient   dx[t, k] = sum_b s_g[t, b] s_w[b, k/128] sum_{n in b} q_g q_w
//   weight gradient  dw[n, k] = sum_t bf16(dy[t, n]) bf16(x[t, k])
// with dy quantised per 1x128 along n for dx. y and dx are bf16; dw is fp32,
// dense [n, k], and not quantised: its contraction runs over the tokens, so FP8
// would need scales along the other dimension of dy and x, two per product.
//
// Precision: the FP8 matrix core aligns the 8 products of each 8 neighbouring k
// to the largest of them and drops what is below 2^-13 of it (measured); with
// the fp32 sums behind it y and dx are off by 1e-5 to 5e-5 of their norm before
// the rounding to bf16 (half a step: 4e-3).
//
// Matrices of activations are row-major with a row stride in elements (at least
// the row length; any alignment of the element type). Input types are
// NETRA_BF16 or NETRA_F32. Outputs must not share memory with inputs; an overlap
// with an activation matrix is refused (different columns of rows with the same
// stride do not overlap). rows may be 0: forward and input gradient then do nothing,
// the weight gradient writes zeros (or leaves dw as it is when it accumulates).
//
// The workspace is scratch of one call: its contents before the call do not
// matter and nothing is kept in it. Calls that may overlap (two streams, two
// graphs that run at once) need workspaces of their own.
//
// Every entry point launches on `stream` of the current device, allocates and
// synchronises nothing (capturable into a HIP graph) and returns 0, a
// hipError_t value, or -1 for invalid arguments, before anything is launched;
// netra_layers_last_error() has the text on the calling thread.
#pragma once

#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { NETRA_BF16 = 0, NETRA_F32 = 1 };

// Weight layout of the linear kernels: w row-major e4m3 [n, k] -> tile16x128
// (include/netra_moe.h) of the matrix, or of its transpose (for the input
// gradient), padded with zeros to multiples of 16 rows and 128 columns.
uint64_t netra_linear_packed_bytes(uint32_t n, uint32_t k, uint32_t transpose);
int netra_linear_pack(const uint8_t* w, uint8_t* packed, uint32_t n, uint32_t k, uint32_t transpose,
                      hipStream_t stream);

// Bytes of workspace (16-byte aligned) one call needs. in_place: both operands of
// the weight gradient are bf16 with n, k and the strides even and 4-byte aligned
// bases; others are first copied to the workspace as aligned bf16.
uint64_t netra_linear_forward_workspace(uint32_t rows, uint32_t n, uint32_t k, uint32_t x_type);
uint64_t netra_linear_input_gradient_workspace(uint32_t rows, uint32_t n, uint32_t k, uint32_t dy_type);
uint64_t netra_linear_weight_gradient_workspace(uint32_t rows, uint32_t n, uint32_t k, uint32_t in_place);

// x [rows, k] -> y bf16 [rows, n]; packed from netra_linear_pack(transpose = 0).
int netra_linear_forward(const void* x, uint32_t x_type, uint64_t x_stride, const uint8_t* packed,
                         const float* scale, uint16_t* y, uint64_t y_stride, uint32_t rows, uint32_t n,
                         uint32_t k, void* workspace, uint64_t workspace_bytes, hipStream_t stream);

// The same for rows that are quantised already: codes and scales as netra_norm_forward leaves them with
// NETRA_CODES_TILES.
uint64_t netra_linear_forward_codes_workspace(uint32_t rows, uint32_t n, uint32_t k);
int netra_linear_forward_codes(const uint8_t* codes, const float* scales, const uint8_t* packed, const float* scale,
                               uint16_t* y, uint64_t y_stride, uint32_t rows, uint32_t n, uint32_t k, void* workspace,
                               uint64_t workspace_bytes, hipStream_t stream);

// dy [rows, n] -> dx bf16 [rows, k]; packed_t from netra_linear_pack(transpose = 1),
// scale the same grid as forward's.
int netra_linear_input_gradient(const void* dy, uint32_t dy_type, uint64_t dy_stride, const uint8_t* packed_t,
                                const float* scale, uint16_t* dx, uint64_t dx_stride, uint32_t rows,
                                uint32_t n, uint32_t k, void* workspace, uint64_t workspace_bytes,
                                hipStream_t stream);

// dy [rows, n], x [rows, k] -> dw fp32 [n, k]; accumulate != 0 adds to dw.
int netra_linear_weight_gradient(const void* dy, uint32_t dy_type, uint64_t dy_stride, const void* x,
                                 uint32_t x_type, uint64_t x_stride, float* dw, uint32_t accumulate,
                                 uint32_t rows, uint32_t n, uint32_t k, void* workspace,
                                 uint64_t workspace_bytes, hipStream_t stream);

// Both gradients in one call (dx and dw must not share memory either).
uint64_t netra_linear_backward_workspace(uint32_t rows, uint32_t n, uint32_t k, uint32_t dy_type, uint32_t in_place);
int netra_linear_backward(const void* dy, uint32_t dy_type, uint64_t dy_stride, const void* x, uint32_t x_type,
                          uint64_t x_stride, const uint8_t* packed_t, const float* scale, uint16_t* dx,
                          uint64_t dx_stride, float* dw, uint32_t accumulate, uint32_t rows, uint32_t n, uint32_t k,
                          void* workspace, uint64_t workspace_bytes, hipStream_t stream);

// counts[e] = number of routes (t, s) with ids[t, s] == e over the tokens whose
// mask byte is nonzero (mask null: all). ids is i32 [tokens, slots] with a row
// stride in elements; ids outside 0 .. experts - 1 (the shared expert's slot,
// -1 for a dropped route) are not counted. accumulate != 0 adds to counts.
// tokens may be 0. tokens * slots < 2^31, experts <= 1024.
uint64_t netra_router_counts_workspace(uint32_t tokens, uint32_t slots, uint32_t experts);
int netra_router_counts(const int32_t* ids, uint64_t ids_stride, const uint8_t* mask, uint32_t tokens,
                        uint32_t slots, uint32_t experts, int32_t* counts, uint32_t accumulate,
                        void* workspace, uint64_t workspace_bytes, hipStream_t stream);

// Balance loss of a softmax router and its gradient. With z = logits + bias
// (bias fp32 [experts] or null, a constant), p = softmax(z) over the experts,
// f_e = experts * counts_e / sum(counts), V the tokens whose mask byte is
// nonzero:
//   loss = coefficient / |V| * sum_{t in V} sum_e f_e p_te
//   grad[t, e] = coefficient / |V| * p_te (f_e - sum_j f_j p_tj), 0 for t not in V
// A perfectly balanced router's loss is `coefficient`. The loss and every
// gradient are 0 where V or the counts are empty, and a token whose z are all
// -inf adds nothing. Masked tokens' logits are not looked at.
// slots != 0: counts are computed from ids as by netra_router_counts and
// written to `counts`; slots 0 (ids is not looked at): counts is an input (for
// instance summed over the ranks of a job). grad (type and shape of logits) may be null.
// counts have to stay below 2^31 in sum; experts <= 1024; row strides of logits and grad
// below 2^27.
uint64_t netra_router_balance_workspace(uint32_t tokens, uint32_t slots, uint32_t experts);
int netra_router_balance(const void* logits, uint32_t logits_type, uint64_t logits_stride, const float* bias,
                         const int32_t* ids, uint64_t ids_stride, uint32_t slots, const uint8_t* mask,
                         uint32_t tokens, uint32_t experts, float coefficient, int32_t* counts, float* loss,
                         void* grad, uint64_t grad_stride, void* workspace, uint64_t workspace_bytes,
                         hipStream_t stream);

// Root-mean-square norm before a projection or the experts.
//   r = x + residual, rounded to the residual's type and written to sum (residual and sum null: r = x)
//   y = r / sqrt(mean(r^2) + eps) * (weight + offset)
// and, for the FP8 products behind it, codes e4m3 of y with one scale per 1x128 by the rule at the
// top (of y in fp32, not of its rounding to y_type). y (bf16 or fp32) or codes and scales may be
// null. codes_layout:
//   NETRA_CODES_ROWS   codes [rows, cols], scales [rows, ceil(cols/128)] (what the bridges take)
//   NETRA_CODES_TILES  what netra_linear_forward_codes takes: tile16x128, scales [ceil(cols/128), rows up to 16];
//                      codes 16-byte aligned
// rows 0 .. 2^21, cols 1 .. 16384; weight [cols] bf16 or fp32. Statistics are fp32: |r| below 1e17, so that a row's sum of
// squares is finite at any length (a row whose sum is not has y 0), and mean(r^2) + eps not below 2^-126.
// sum may be the residual or x, y may be x or the residual (same address, type and stride); any
// other overlap is refused.
enum { NETRA_CODES_ROWS = 1, NETRA_CODES_TILES = 2 };
uint64_t netra_norm_code_bytes(uint32_t rows, uint32_t cols, uint32_t codes_layout);
uint64_t netra_norm_scale_count(uint32_t rows, uint32_t cols, uint32_t codes_layout);
int netra_norm_forward(const void* x, uint32_t x_type, uint64_t x_stride, const void* residual, uint32_t residual_type,
                       uint64_t residual_stride, const void* weight, uint32_t weight_type, float offset, float eps,
                       void* sum, uint64_t sum_stride, void* y, uint32_t y_type, uint64_t y_stride, uint8_t* codes,
                       float* scales, uint32_t codes_layout, uint32_t rows, uint32_t cols, hipStream_t stream);

// Its gradients. r is what was normalised (sum, or x), dy the gradient of y, flow what flows into r
// besides (the residual stream's gradient, of r's type, or null). With g = dy (weight + offset),
// xh = r / sqrt(mean(r^2) + eps):
//   dr = (g - xh mean(g xh)) / sqrt(mean(r^2) + eps) + flow    (of r's type: x's and the residual's)
//   dw = sum over the rows of dy xh                            (fp32 [cols]; accumulate != 0 adds to it)
// dr may be dy, r or flow (same address, type and stride). rows may be 0: dw is then zeros or as it was.
uint64_t netra_norm_gradients_workspace(uint32_t rows, uint32_t cols);
int netra_norm_gradients(const void* dy, uint32_t dy_type, uint64_t dy_stride, const void* r, uint32_t r_type,
                         uint64_t r_stride, const void* flow, uint64_t flow_stride, const void* weight,
                         uint32_t weight_type, float offset, float eps, void* dr, uint64_t dr_stride, float* dw,
                         uint32_t accumulate, uint32_t rows, uint32_t cols, void* workspace, uint64_t workspace_bytes,
                         hipStream_t stream);

// Routing to experts. s = softmax(logits) over the experts or sigmoid(logits); c = s + bias (bias
// fp32 [experts] or null: it moves the choice, not the weights). The experts are `groups` runs of
// equal length; a group's score is its largest c (NETRA_GROUP_MAX) or the sum of its two largest
// (NETRA_GROUP_TOP2), and the top_groups best groups are kept. ids[t, 0 .. k) are the k largest c of those in
// falling order; ties go to the lower index, of groups as of experts. c is compared exactly: by the logits
// where their order decides (no bias, no sums of two), else in 64 bits. A NaN ranks as -inf, also one that is the sum of two.
// (-inf in bias takes an expert out at no cost; a large finite number does so too, but most tokens then need 64 bits throughout.)
//   weights[t, i] = scale * s_i, or scale * s_i / sum over the chosen of s (renormalise; 0 where the sum is 0,
//   as where all of them are below 2^-126)
// shared 1: logits has a column more, the shared expert's gate, and slot k is
// (experts, sigmoid(logits[t, experts])), unscaled. Tokens whose mask byte is 0 get ids -1 and weights 0.
// tokens 0 .. 2^25, experts 1 .. 1024, k + shared 1 .. 16, groups 1 .. 16; ids and weights have row strides in
// elements.
enum { NETRA_SOFTMAX = 0, NETRA_SIGMOID = 1 };
enum { NETRA_GROUP_MAX = 0, NETRA_GROUP_TOP2 = 1 };
int netra_router_select(const void* logits, uint32_t logits_type, uint64_t logits_stride, const float* bias,
                        const uint8_t* mask, uint32_t tokens, uint32_t experts, uint32_t k, uint32_t shared,
                        uint32_t scoring, uint32_t groups, uint32_t top_groups, uint32_t group_score, uint32_t renormalise,
                        float scale, int32_t* ids, uint64_t ids_stride, float* weights, uint64_t weights_stride,
                        hipStream_t stream);

// The weights' gradient carried to the logits, for given choices: with dweights fp32 [tokens, k + shared],
//   grad[t, e] = sum_i dweights[t, i] dweights_i / dlogits_e    (of the logits' type, [tokens, experts + shared])
// ids as above; slots whose id is not an expert (a dropped route) have the weight 0 and no gradient, and
// are left out of the sum that renormalises. An id that stands in several slots counts as often.
// Tokens whose mask byte is 0 get zeros. accumulate != 0 adds to grad (the balance loss's gradient, say).
int netra_router_select_gradient(const float* dweights, uint64_t dweights_stride, const void* logits,
                                 uint32_t logits_type, uint64_t logits_stride, const int32_t* ids, uint64_t ids_stride,
                                 const uint8_t* mask, uint32_t tokens, uint32_t experts, uint32_t k, uint32_t shared,
                                 uint32_t scoring, uint32_t renormalise, float scale, void* grad, uint64_t grad_stride,
                                 uint32_t accumulate, hipStream_t stream);

// Low-rank adapters of many requests beside a shared projection: for every token t with the adapter l,
//   out[t] = y[t] + scale[l] B_l (A_l x[t]),  A_l [rank, k], B_l [n, rank] bf16 (fp32 is rounded when packed)
// and out[t] = y[t] for tokens without one. x bf16 or fp32 [tokens, k] (fp32 is rounded to bf16), y
// and out bf16 [tokens, n], scale fp32 [adapters]. A_l x and all sums are fp32, A_l x enters the
// second product with 16 bits, and the sum with y is rounded once. adapters 1 .. 1024, rank 1 .. 128.
//
// Weights are laid out once: a [adapters, rank, k], b [adapters, n, rank], both of `type`. which:
// 0 packed_a, 1 packed_b; both 16-byte aligned.
uint64_t netra_adapters_packed_bytes(uint32_t adapters, uint32_t rank, uint32_t n, uint32_t k, uint32_t which);
int netra_adapters_pack(const void* a, const void* b, uint32_t type, void* packed_a, void* packed_b, uint32_t adapters,
                        uint32_t rank, uint32_t n, uint32_t k, hipStream_t stream);
// A batch's plan, for every call with the same ids (all layers of a step): ids i32 [tokens], outside 0 .. adapters - 1
// for none. plan 16-byte aligned; calls that read it may overlap. A call whose tokens or
// adapters are not the plan's writes nothing.
uint64_t netra_adapters_plan_bytes(uint32_t tokens, uint32_t adapters);
int netra_adapters_plan(const int32_t* ids, uint32_t tokens, uint32_t adapters, void* plan, uint64_t plan_bytes,
                        hipStream_t stream);
// out may be y (same address and stride); any other overlap of out or the workspace with what the call reads, or of the two,
// is refused. tokens 0 .. 2^21.
uint64_t netra_adapters_add_workspace(uint32_t tokens, uint32_t adapters, uint32_t rank, uint32_t n, uint32_t k);
int netra_adapters_add(const void* x, uint32_t x_type, uint64_t x_stride, const void* packed_a, const void* packed_b,
                       const float* scale, const void* plan, const uint16_t* y, uint64_t y_stride, uint16_t* out,
                       uint64_t out_stride, uint32_t tokens, uint32_t adapters, uint32_t rank, uint32_t n, uint32_t k,
                       void* workspace, uint64_t workspace_bytes, hipStream_t stream);

const char* netra_layers_last_error(void);

#ifdef __cplusplus
}
#endif

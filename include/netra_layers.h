// Operators next to the routed-MoE layer (libnetra_layers.so): the block-FP8
// linear layer y = x W^T with its gradients, per-expert route counts, and the
// router's balance loss with its gradient.
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

const char* netra_layers_last_error(void);

#ifdef __cplusplus
}
#endif

// C entry points of the training kernels, as the autograd module calls them.
// Strides are in elements; every call returns 0, a CUDA error code, or -1 for
// arguments out of range.
#pragma once

#include <cuda_runtime_api.h>

#include <cstdint>

extern "C" {

// --- dropout.cu ---
// y[rows, K] = dropout(x) (+ residual); type: ElemType of all three. 0 <= cut < 65536
// (a call that drops everything needs no kernel). offset_ptr: an int64 on the device
// that is added to `offset`, or null.
int b200_dropout(const void* x, int64_t ldx, const void* residual, int64_t ldr, void* y, int64_t ldy, int64_t rows,
                 int K, int type, uint64_t seed, uint64_t offset, const int64_t* offset_ptr, int cut, float scale,
                 int num_sms, cudaStream_t st);

// --- block_norms.cu ---
// Widest row.
int b200_block_norms_max_width();
// CTAs of the backward pass (rows of its partial sums) for T rows of H columns.
int b200_block_norms_bwd_grid(int64_t T, int H, int type, int num_sms);
// Forward. type: ElemType of x, delta, gate, y and h; w_type: of post and pre, that or
// fp32. gate_kind: 0 none, 1 [H], 2 [T], 3 [T, H]. y may be x. r1, r2: fp32 [T] or null.
int b200_block_norms(const void* x, int64_t ldx, const void* delta, int64_t ldd, const void* post, const void* pre,
                     int w_type, const void* gate, int64_t ldg, int gate_kind, void* y, int64_t ldy, void* h,
                     int64_t ldh, float* r1, float* r2, int64_t T, int H, int type, float eps, float scale,
                     int offset_one, int round_branch, int num_sms, cudaStream_t st);
// Backward from y, delta and the saved r1 / r2. dy or dh may be null (zero); dx,
// ddelta, dgate, dpost and dpre are null where not wanted. dx, ddelta and an element
// gate's gradient have rows of H elements. part: fp32 [number of dpost, dpre and
// channel dgate wanted][b200_block_norms_bwd_grid][H].
int b200_block_norms_bwd(const void* y, int64_t ldy, const void* delta, int64_t ldd, const void* post, const void* pre,
                         int w_type, const void* gate, int64_t ldg, int gate_kind, const float* r1, const float* r2,
                         const void* dy, int64_t lddy, const void* dh, int64_t lddh, void* dx, void* ddelta,
                         void* dgate, void* dpost, void* dpre, float* part, int64_t T, int H, int type, float scale,
                         int offset_one, int num_sms, cudaStream_t st);

// --- linear_ce.cu ---
// What a forward pass leaves for its backward pass, in one buffer: the scored rows
// [T, Kp] bf16, then their target logits, losses and logarithms of the sums of exp fp32
// [T] each, then int32 count, ticket, target [T], token [T], place [T].
int64_t b200_lce_saved_bytes(int T, int Kp);
// Scratch of the forward pass: a (max, sum) pair per row and column tile.
int64_t b200_lce_forward_bytes(int T, int V);
// Scratch of the backward pass: one piece of G (bf16 [T, piece]), dh's sums, and for dW what
// the targets' entries lost (fp32 [T, Kp]) with its map (int32 [V]).
int64_t b200_lce_backward_bytes(int T, int V, int K, int Kp, int piece, int want_dh, int want_dw, int num_sms);
// Forward. h [T, K] and W [V, K] bf16 (W 16-byte aligned with ldw % 8 == 0), targets
// int64. Kp: K rounded up to a multiple of 8. loss fp32 [T]; total [1] or null (mean:
// divided by the scored rows, at least 1).
int b200_lce_forward(const void* h, int64_t ldh, const void* W, int64_t ldw, const int64_t* targets, int64_t ignore,
                     int T, int V, int K, int Kp, float cap, void* saved, void* part, float* loss, float* total,
                     int mean, int num_sms, cudaStream_t st);
// Backward from what the forward pass saved. dloss: element token * dloss_stride.
// dh [T, K] contiguous and dW [V, K] (row stride lddw, a multiple of 8) are null
// where not wanted. piece: columns of the vocabulary at a time, a multiple of 256.
int b200_lce_backward(void* saved, const void* W, int64_t ldw, const float* dloss, int64_t dloss_stride, int mean, int T,
                      int V, int K, int Kp, float cap, int piece, void* scratch, void* dh, void* dW, int64_t lddw,
                      int num_sms, cudaStream_t st);

}  // extern "C"

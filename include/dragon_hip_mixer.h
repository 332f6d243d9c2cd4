/*
 * dragon_hip_mixer.h -- the token mixers of long-sequence language models, FP32 like the rest of libdragon_hip.so:
 * attention with a sliding window and a few first tokens that stay visible, and linear attention with a decay for
 * each head; prompts, single tokens on what earlier tokens left, and gradients.  Neither has a counterpart in the
 * reference, whose one attention block sees every key (dragon_Cuda_attention_forward in dragon_hip_gemm.h).
 *
 * Common to all entries:
 *   - addresses are device memory, 16-byte aligned for float tensors, 4-byte for lengths, decays and dLse;
 *   - head dimensions dK4 (Q, K) and dV4 (V, Y) are multiples of 4 up to 128, pad columns zero as everywhere (those of
 *     the outputs come out as zeros);
 *   - head_inner = 0: tensors [N, heads, L, d4], head_inner = 1: [N, L, heads, d4], with L the capacity QL, VL or L;
 *   - lengths are int32[N] on the device, or 0 for "all of them"; a value outside 0 ... capacity counts as the nearer of
 *     the two.  Rows behind a sequence's length are never read, and come out as zeros;
 *   - work goes to streams[0]; nothing is allocated, kept between calls or read back, so every call may be captured;
 *   - dBuf is the caller's work buffer of at least the bytes that the matching _bufsize names for the same sizes
 *     (buf_size says how many there are); its content means nothing between calls.  Calls that may run at the same time,
 *     replays of graphs among them, need one each.  _bufsize returns -1 for sizes that the call refuses;
 *   - outputs overlap no operand and each other not at all, but dStateOut may be dState;
 *   - hipErrorInvalidValue: a null or misaligned address, a size out of range, a scale that is not finite, a buffer that is
 *     too small.  No kernel has run then;
 *   - results have the same bits from call to call (no sum depends on who arrives first).
 */
#ifndef DRAGON_HIP_MIXER_H
#define DRAGON_HIP_MIXER_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- attention with a sliding window and sinks --------------------------------------------------------------
 * Sequence n has ql <= QL queries and vl <= VL keys; its last query stands at its last key, position(i) = i + vl - ql,
 * so QL = VL is a prompt, a smaller QL the next piece of one, QL = 1 a single token on a cache.  Query i sees key j when
 *     i < ql,  j < vl,  j <= position(i)  and  (window == 0  or  j > position(i) - window  or  j < sinks)
 * (window = 0: no window).  Over the keys it sees
 *     lse[i] = log sum_j exp(scale * <Q[i], K[j]>),   Y[i] = sum_j exp(scale * <Q[i], K[j]> - lse[i]) * V[j];
 * a query that sees none has Y[i] = 0, lse[i] = -infinity.  Q and Y have `head` heads, K and V kv_head, which divides head:
 * query head h reads key / value head h / (head / kv_head).  dLse: float[N, head, QL] (for the gradient) or 0.
 * Keys that no query of the call sees are never read (a decoding cache may hold anything there).  A key that some query sees
 * has to be finite in K and V: a NaN or an infinity there can reach the rows of queries that do not see it. */
int64_t dragon_Cuda_attention_window_bufsize(int32_t N, int32_t head, int32_t kv_head, int32_t QL, int32_t VL, int32_t dK4,
                                             int32_t dV4, int32_t window, int32_t sinks);
int dragon_Cuda_attention_window_forward(const int64_t* streams, int32_t length, int64_t dQ, int64_t dK, int64_t dV, int64_t dY,
                                         int64_t dLse, int64_t dQLens, int64_t dVLens, int64_t dBuf, int64_t buf_size, int32_t N,
                                         int32_t head, int32_t kv_head, int32_t QL, int32_t VL, int32_t dK4, int32_t dV4,
                                         int32_t head_inner, float scale, int32_t window, int32_t sinks);

/* Its gradient: dDeltaQ, dDeltaK, dDeltaV from dDeltaY, with dY and dLse as the forward call of the same operands left them.
 * The gradients of a shared key / value head are the sums over its query heads; rows that nobody sees get zeros.  All three
 * are written whole, none is added to.  Every size takes a work buffer here. */
int64_t dragon_Cuda_attention_window_backward_bufsize(int32_t N, int32_t head, int32_t kv_head, int32_t QL, int32_t VL,
                                                      int32_t dK4, int32_t dV4, int32_t window, int32_t sinks);
int dragon_Cuda_attention_window_backward(const int64_t* streams, int32_t length, int64_t dQ, int64_t dK, int64_t dV, int64_t dY,
                                          int64_t dLse, int64_t dDeltaY, int64_t dDeltaQ, int64_t dDeltaK, int64_t dDeltaV,
                                          int64_t dQLens, int64_t dVLens, int64_t dBuf, int64_t buf_size, int32_t N, int32_t head,
                                          int32_t kv_head, int32_t QL, int32_t VL, int32_t dK4, int32_t dV4, int32_t head_inner,
                                          float scale, int32_t window, int32_t sinks);

/* ---- linear attention with a decay for each head -------------------------------------------------------------
 * A state S[dK4, dV4] per (image, head) forgets by e^g a token:
 *     S_t = e^g S_{t-1} + K[t]^T V[t],    Y[t] = scale * Q[t] S_t,    t = 0 ... len - 1
 * dDecay: float[head] on the device, g <= 0 (-infinity: nothing is kept).  dState: S before the first token,
 * [N, head, dK4, dV4], or 0 for zeros; dStateOut: S after the last, or 0 if nobody wants it.  A call with L tokens and one
 * with the next tokens and the first one's dStateOut as dState give what one call with all of them gives.  Up to 16 tokens
 * the recurrence is computed as it stands (no work buffer), beyond that chunks of the sequence in parallel. */
int64_t dragon_Cuda_linear_attention_bufsize(int32_t N, int32_t head, int32_t L, int32_t dK4, int32_t dV4);
int dragon_Cuda_linear_attention_forward(const int64_t* streams, int32_t length, int64_t dQ, int64_t dK, int64_t dV,
                                         int64_t dDecay, int64_t dState, int64_t dY, int64_t dStateOut, int64_t dLens,
                                         int64_t dBuf, int64_t buf_size, int32_t N, int32_t head, int32_t L, int32_t dK4,
                                         int32_t dV4, int32_t head_inner, float scale);

/* Its gradient with respect to Q, K, V and the first state (the decay is a constant of the head and has none):
 * dDeltaStateOut is the gradient of the last state, or 0 for zeros; dDeltaState may be 0 if nobody wants it. */
int64_t dragon_Cuda_linear_attention_backward_bufsize(int32_t N, int32_t head, int32_t L, int32_t dK4, int32_t dV4);
int dragon_Cuda_linear_attention_backward(const int64_t* streams, int32_t length, int64_t dQ, int64_t dK, int64_t dV,
                                          int64_t dDecay, int64_t dState, int64_t dDeltaY, int64_t dDeltaStateOut,
                                          int64_t dDeltaQ, int64_t dDeltaK, int64_t dDeltaV, int64_t dDeltaState,
                                          int64_t dLens, int64_t dBuf, int64_t buf_size, int32_t N, int32_t head, int32_t L,
                                          int32_t dK4, int32_t dV4, int32_t head_inner, float scale);

#ifdef __cplusplus
}
#endif
#endif /* DRAGON_HIP_MIXER_H */

/*
 * C ABI of the kernel products over sequences: the products of f3m.h for kernels of query and key vectors
 * that stand in an order.
 *
 *   attention with a window    out_i = sum_j exp(scale q_i.k_j) v_j / sum_j exp(scale q_i.k_j), j over the last `window`
 *                              positions up to i and the first `sinks` positions: the exponential kernel summed over a
 *                              near field and a few fixed sources, each row divided by its sum
 *   linear attention           out_t = scale sum_{s<=t} exp(g (t-s)) (q_t.k_s) v_s: a separable kernel, carried as its
 *                              moments S_t = e^g S_{t-1} + k_t v_t^T
 *
 * Every pointer except the parameters is DEVICE memory of the calling thread's current device.  Calls are QUEUED on
 * `stream` (a hipStream_t) and not waited for; they allocate nothing, keep nothing and can be captured into a graph.
 * A call's workspace (size from the _workspace function, which depends on the parameters alone) holds no data between
 * calls; calls that may run at the same time need workspaces of their own.  Outputs must not overlap inputs.
 * Functions return 0 or a positive error code, with the message in f3m_last_error(); a refused call writes nothing.
 * Results have the same bits on every run: nothing is added in an order that can change.
 *
 * Element types: F3M_BF16, F3M_F16, F3M_F32.  Sums, softmax statistics and states are fp32.  Strides are in elements, of the
 * batch, token and head dimension; the last dimension is contiguous.  Vectors are read 16 bytes at a time: base
 * pointers and strides (in bytes) must be multiples of 16 and head sizes multiples of 8 up to 128.
 */
#ifndef F3M_SEQUENCE_H
#define F3M_SEQUENCE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum f3m_dtype { F3M_BF16 = 0, F3M_F16 = 1, F3M_F32 = 2 };

typedef struct f3m_attn_params {
    int dtype;
    int D;                      /* head size of q, k and v */
    int Hq, Hkv;                /* heads; Hq is a multiple of Hkv, query head h reads key head h / (Hq / Hkv) */
    int64_t B, Nq, Nk;          /* batch, rows of q and of k, v */
    int64_t q_stride[3], k_stride[3], v_stride[3], dout_stride[3];
    int64_t window;             /* a row sees the last `window` positions, its own among them; 0 = all up to its own */
    int64_t sinks;              /* and the first `sinks` positions */
    float scale;                /* of either sign; 0 takes all keys as equal; |scale| log2(e) has to be finite */
} f3m_attn_params;

/* Row i of sequence b stands at position kv_lens[b] - q_lens[b] + i and sees no key at or behind kv_lens[b].  q_lens, kv_lens:
 * int32 (B) or NULL (all Nq, Nk); values are taken into [0, Nq] and [0, Nk].  Rows at or behind q_lens[b], and rows that see no key, get
 * out = 0 and lse = -inf.  out: contiguous (B, Nq, Hq, D); lse: fp32 (B, Nq, Hq) or NULL.  k and v are read only where some row of the
 * same piece of rows sees the key, so what lies behind kv_lens or before all windows may hold anything. */
int f3m_window_attention_workspace(const f3m_attn_params *params, int grad, size_t *bytes);
int f3m_window_attention(const f3m_attn_params *params, const void *q, const void *k, const void *v, const int32_t *q_lens,
                         const int32_t *kv_lens, void *out, float *lse, void *workspace, size_t workspace_bytes, void *stream);
/* Gradients of sum(out * dout) from the forward call's out and lse.  out and dq contiguous (B, Nq, Hq, D), dk and dv
 * contiguous (B, Nk, Hkv, D): every element is written, zero where nothing reaches it. */
int f3m_window_attention_grad(const f3m_attn_params *params, const void *q, const void *k, const void *v, const void *out,
                              const float *lse, const void *dout, const int32_t *q_lens, const int32_t *kv_lens, void *dq,
                              void *dk, void *dv, void *workspace, size_t workspace_bytes, void *stream);

typedef struct f3m_linear_params {
    int dtype;
    int Dk, Dv;                 /* head sizes of q, k and of v */
    int H;
    int64_t B, N;
    int64_t q_stride[3], k_stride[3], v_stride[3], dout_stride[3];
    float scale;                /* finite and not 0 */
} f3m_linear_params;

/* log_decay: fp32 (H), the natural logarithm g of each head's factor, g <= 0 (-inf: only the token itself).  initial_state, final_state:
 * contiguous fp32 (B, H, Dk, Dv), either NULL (zero; not wanted).  lens: int32 (B) or NULL; tokens at or behind lens[b] are not
 * read, their rows of out are 0 and the final state is that of the last token before.  out: contiguous (B, N, H, Dv). */
int f3m_linear_attention_workspace(const f3m_linear_params *params, int grad, size_t *bytes);
int f3m_linear_attention(const f3m_linear_params *params, const void *q, const void *k, const void *v, const float *log_decay,
                         const float *initial_state, const int32_t *lens, void *out, float *final_state, void *workspace,
                         size_t workspace_bytes, void *stream);
/* Gradients of sum(out * dout) + sum(final_state * dfinal_state); dfinal_state, initial_state and dinitial_state may be NULL.  dq,
 * dk (B, N, H, Dk) and dv (B, N, H, Dv) are contiguous and wholly written. */
int f3m_linear_attention_grad(const f3m_linear_params *params, const void *q, const void *k, const void *v,
                              const float *log_decay, const float *initial_state, const void *dout, const float *dfinal_state,
                              const int32_t *lens, void *dq, void *dk, void *dv, float *dinitial_state, void *workspace,
                              size_t workspace_bytes, void *stream);
/* One token: state = e^g state + k v^T in place, out = scale q^T state.  N is 1 and the token stride is not read; out (B, H, Dv) and
 * state (B, H, Dk, Dv) are contiguous. */
int f3m_linear_attention_step(const f3m_linear_params *params, const void *q, const void *k, const void *v,
                              const float *log_decay, float *state, void *out, void *stream);

#ifdef __cplusplus
}
#endif
#endif

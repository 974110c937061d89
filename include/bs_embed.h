/*
 * bs_embed.h -- C-ABI of the encoder operators of libbs_hip.so (MI355X, gfx950).
 *
 * The index of bs_hip.h holds float32 vectors and is searched with float32 vectors; these are
 * the operators of the text encoder that makes both, on the GPU and stream that search them:
 * attention over packed sequences, also behind a shared prefix, products with their epilogue, gated
 * products, layer norm, norms of heads with rotary positions, and gradients of the latter three.
 * The reference starts from vectors in files and has no counterpart.
 *
 * Conventions
 *   - every pointer is device memory of the current device; streams are passed as void* (a
 *     hipStream_t, or NULL for the null stream).  Calls are asynchronous: they launch kernels
 *     on `stream`, allocate nothing, record no event and may be captured into a HIP graph.
 *   - return 0 on success, a negative BS_E* code (bs_hip.h) on error; bs_last_error() returns
 *     the text.  Arguments are checked before anything is launched.
 *   - strides count elements.  The features of a row (the elements of a head) are contiguous,
 *     rows may lie any distance >= the row's length apart and start at any element.
 *   - a workspace belongs to the call until its kernels have run.  Its size depends on the
 *     sizes of the call alone: the *_workspace functions.
 *   - inputs are not written; outputs must not overlap inputs or the workspace, except where
 *     an entry says so.
 *   - sums, row statistics, softmax maxima and sums are float32; results are rounded once, to
 *     the nearest value of their type (attention rounds its weights too, see there).  Two calls
 *     on the same inputs give the same bits.
 */
#ifndef BS_EMBED_H
#define BS_EMBED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
typedef enum { BS_F32 = 0, BS_F16 = 1, BS_BF16 = 2 } bs_type;

/* activations of bs_linear:  none z;  relu max(z, 0);  gelu z (1 + erf(z / sqrt 2)) / 2;
 * gelu_tanh z (1 + tanh(sqrt(2 / pi) (z + 0.044715 z^3))) / 2;  silu z / (1 + exp(-z)) */
typedef enum { BS_ACT_NONE = 0, BS_ACT_RELU = 1, BS_ACT_GELU = 2, BS_ACT_GELU_TANH = 3, BS_ACT_SILU = 4 } bs_activation;

/* Layer norm of `rows` rows of `cols` features (1..16384), type BS_F32, BS_F16 or BS_BF16:
 *   y = (x - mean) * rstd * weight + bias,  rstd = 1 / sqrt(var + eps),  var over cols.
 * weight and bias (cols each, wtype: `type` or BS_F32) may be NULL: 1 and 0.  mean and rstd
 * (rows float32 each) may be NULL.  y may be x itself with x's stride. */
int bs_layer_norm(const void* x, int64_t x_stride, const void* weight, const void* bias, int wtype, float eps,
                  void* y, int64_t y_stride, float* mean, float* rstd, uint64_t rows, uint32_t cols, int type,
                  void* stream);

/* Gradients of bs_layer_norm from dy, x and the saved mean and rstd:
 *   g = dy * weight,  xh = (x - mean) * rstd
 *   dx = rstd * (g - mean(g) - xh * mean(g * xh)),  dweight = sum of dy * xh over the rows,
 *   dbias = sum of dy over the rows
 * dx may be NULL, dweight and dbias (cols each, wtype) too, both or neither; weight NULL is 1.
 * dx may be dy or x itself with its stride.  The sums over the rows have a fixed order (no
 * atomics).  workspace: bs_layer_norm_backward_workspace bytes, 16-byte aligned; not needed
 * without dweight. */
int bs_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const float* mean,
                           const float* rstd, const void* weight, int wtype, void* dx, int64_t dx_stride, void* dweight,
                           void* dbias, uint64_t rows, uint32_t cols, int type, void* workspace, uint64_t workspace_bytes,
                           void* stream);
int bs_layer_norm_backward_workspace(uint64_t rows, uint32_t cols, int type, uint64_t* bytes);

/* out = act(x w^T + bias) + residual:  x rows x inner, w cols x inner, bias cols, all of `type`
 * (BS_F16 or BS_BF16); residual and out rows x cols of out_type (`type` or BS_F32).  bias and
 * residual may be NULL; residual may be out itself with its stride.  rows x ceil(cols / 128) up
 * to 2^31 - 256, inner and cols 1..2^24, strides < 2^24.  Products are summed in float32.  workspace:
 * bs_linear_workspace bytes (0 where the call does not split the inner dimension), 16-byte
 * aligned. */
int bs_linear(const void* x, int64_t x_stride, const void* w, int64_t w_stride, const void* bias, const void* residual,
              int64_t residual_stride, void* out, int64_t out_stride, uint64_t rows, uint32_t inner, uint32_t cols,
              int type, int out_type, int activation, void* workspace, uint64_t workspace_bytes, void* stream);
int bs_linear_workspace(uint64_t rows, uint32_t inner, uint32_t cols, uint64_t* bytes);

/* Attention over packed sequences.  q: q_tokens x heads x head_dim, k and v: k_tokens x
 * kv_heads x head_dim, out as q; `type` BS_F16 or BS_BF16.  Sequence s owns the query tokens
 * q_offsets[s] .. q_offsets[s + 1] - 1 and the key tokens k_offsets[s] .. k_offsets[s + 1] - 1
 * (int32, ascending, from 0; a length may be 0).  Head h reads key/value head
 * h / (heads / kv_heads).  With nq and nk tokens of a sequence, query i sees key j
 *   for j < nk, and if causal, j <= i + nk - nq (the last query sees the last key).
 *   out = sum_j p_j v_j,  p = softmax over the visible keys of scale * (q . k_j)
 *   lse (float32, q_tokens x heads, or NULL) = log of the sum of exp(scale * (q . k_j))
 * The weights exp(..) are rounded to `type` for their product with the values; their sum, which
 * divides it, and lse take them as they are.  So out is off by up to 2^-9 (BS_BF16) or 2^-12
 * (BS_F16) of sum_j p_j |v_j| besides its own rounding, and in BS_F16 by 2^-32 of
 * max_j p_j sum_j |v_j|.
 * A query that sees no key gets out 0 and lse -infinity.  Keys and values that a query does not
 * see never touch its result, NaN and infinities included.  Tokens outside every sequence are
 * neither read nor written.  Offsets are read on the device, and ones that are not ascending or
 * past the tokens given leave the result undefined but nothing outside the buffers is touched.
 * longest_q, longest_k: the longest sequence (0: unknown); they choose the split, not the
 * result's meaning: a wrong one costs time only. */
typedef struct {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    float* lse;
    const int32_t* q_offsets; /* sequences + 1, or NULL: one sequence of all tokens */
    const int32_t* k_offsets;
    int64_t q_stride, q_head_stride; /* elements between tokens and between heads; 16-byte     */
    int64_t k_stride, k_head_stride; /* aligned rows: base addresses multiples of 16 bytes and */
    int64_t v_stride, v_head_stride; /* strides multiples of 8                                 */
    int64_t out_stride, out_head_stride;
    uint32_t q_tokens, k_tokens; /* < 2^31 */
    uint32_t sequences;          /* >= 1 */
    uint32_t heads, kv_heads;    /* heads a multiple of kv_heads, up to 1024 */
    uint32_t head_dim;           /* 8..128, a multiple of 8 */
    uint32_t longest_q, longest_k;
    int32_t type;
    int32_t causal;
    float scale; /* finite, at most 1e30 */
} bs_attention_args;

/* workspace: bs_attention_workspace bytes for the same args (pointers are not looked at), 16-byte
 * aligned; 0 where the keys are not split. */
int bs_attention(const bs_attention_args* args, void* workspace, uint64_t workspace_bytes, void* stream);
int bs_attention_workspace(const bs_attention_args* args, uint64_t* bytes);

/* Norm of every head of queries and keys and the rotation by their positions, in one pass.
 * q: tokens x heads x head_dim, k: tokens x kv_heads x head_dim (kv_heads 0: none), `type`
 * BS_F32, BS_F16 or BS_BF16.  With n = x / sqrt(mean(x^2) + eps) * weight over a head's elements
 * (x itself without `norm`; weight q_weight or k_weight, head_dim each of wtype, NULL: 1), the
 * first `rotary` elements are turned in pairs i = 0 .. rotary / 2 - 1 and the others are n:
 *   (a, b) -> magnitude * (a cos - b sin, b cos + a sin),  angle = position * frequencies[i]
 * where a pair is (i, i + rotary / 2), or (2 i, 2 i + 1) if `interleaved`.  Angles are reduced in
 * float64, so far positions lose nothing; squares are summed in float32, which holds those of
 * elements up to 2^60 and, where eps does not cover them (as 0), of heads whose largest element is
 * 2^-60 or more.  Elements of a head are contiguous; *_out may be the call's own q and k (or q_grad
 * and k_grad) with their strides. */
typedef struct {
    const void* q;
    const void* k;
    const void* q_grad; /* of the results; backward alone */
    const void* k_grad;
    void* q_out; /* the results; backward: the gradients of q and k */
    void* k_out;
    const void* q_weight; /* head_dim, or NULL */
    const void* k_weight;
    void* q_weight_grad; /* backward alone, may be NULL */
    void* k_weight_grad;
    const int32_t* positions;  /* tokens, any values, or NULL: 0, 1, .. */
    const double* frequencies; /* rotary / 2, radians per position */
    int64_t q_stride, q_head_stride;
    int64_t k_stride, k_head_stride;
    int64_t q_grad_stride, q_grad_head_stride;
    int64_t k_grad_stride, k_grad_head_stride;
    int64_t q_out_stride, q_out_head_stride;
    int64_t k_out_stride, k_out_head_stride;
    uint32_t tokens;          /* < 2^31 */
    uint32_t heads, kv_heads; /* 1..1024, 0..1024 */
    uint32_t head_dim;        /* even, 2..256 */
    uint32_t rotary;          /* even, 0..head_dim */
    int32_t interleaved;
    int32_t norm;
    int32_t type;
    int32_t wtype; /* of weights and their gradients: type or BS_F32 */
    float eps;
    float magnitude;
} bs_head_norm_rotary_args;

int bs_head_norm_rotary(const bs_head_norm_rotary_args* args, void* stream);

/* Its gradients from q, k and the gradients of the results.  With d the gradients turned back
 * (times magnitude) and r = 1 / sqrt(mean(x^2) + eps):
 *   q_out, k_out: r * (d weight - x r^2 mean(d weight x))  (d without `norm`; q and k are not read)
 *   q_weight_grad, k_weight_grad: the sums of d x r over tokens and heads, in a fixed order
 * workspace: bs_head_norm_rotary_backward_workspace bytes, 16-byte aligned; not needed without
 * weight gradients. */
int bs_head_norm_rotary_backward(const bs_head_norm_rotary_args* args, void* workspace, uint64_t workspace_bytes, void* stream);
int bs_head_norm_rotary_backward_workspace(const bs_head_norm_rotary_args* args, uint64_t* bytes);

/* Gated products:  out = act(x w_gate^T) * (x w_up^T),  x rows x inner, w_gate and w_up cols x
 * inner, out rows x cols, all of `type` (BS_F16 or BS_BF16); inner 1..2^24, cols 1..2^23, strides <
 * 2^24.  gate and up (rows x cols each, contiguous, or both NULL): x w_gate^T and x w_up^T, as the
 * gradients take them.  Products are summed and multiplied in float32. */
int bs_gated(const void* x, int64_t x_stride, const void* w_gate, int64_t w_gate_stride, const void* w_up, int64_t w_up_stride,
             void* out, int64_t out_stride, void* gate, void* up, uint64_t rows, uint32_t inner, uint32_t cols, int type,
             int activation, void* stream);

/* Its gradients from dh, the gradient of out, and the saved gate and up:
 *   dgate = dh up act'(gate),  dup = dh act(gate), both rounded to `type` for their products (so in
 *   BS_F16 they are infinite past 65504 and lose bits below 2^-14)
 *   dx = dgate w_gate + dup w_up,  dw_gate = dgate^T x,  dw_up = dup^T x
 * (relu's slope at 0 is 0; infinite gates have the activations' limits; factors are multiplied in
 * float32 in this order, so dh up has to lie within its range).  dx (rows x inner) may be NULL,
 * dw_gate and dw_up (cols x inner) too, both or neither; all contiguous.  The sums over the rows have a fixed order.  workspace:
 * bs_gated_backward_workspace bytes, 16-byte aligned. */
int bs_gated_backward(const void* dh, int64_t dh_stride, const void* x, int64_t x_stride, const void* w_gate,
                      int64_t w_gate_stride, const void* w_up, int64_t w_up_stride, const void* gate, int64_t gate_stride,
                      const void* up, int64_t up_stride, void* dx, void* dw_gate, void* dw_up, uint64_t rows, uint32_t inner,
                      uint32_t cols, int type, int activation, void* workspace, uint64_t workspace_bytes, void* stream);
int bs_gated_backward_workspace(uint64_t rows, uint32_t inner, uint32_t cols, uint64_t* bytes);

/* Attention of sequences that share their first keys: as bs_attention, but every query sees the
 * `tokens` keys of the prefix besides those that it sees of its own sequence, and the softmax is
 * over both.  The prefix is read once for the rows of all sequences where sequences are short, and
 * by each tile of rows where they fill tiles.  Its type, kv_heads and head_dim are args'; a prefix
 * of 0 tokens is bs_attention.  A query's own keys may be none.  Strides of keys and values, the
 * prefix's too, are < 2^22.  Queries outside every sequence may be read, not written.
 * workspace: bs_attention_shared_prefix_workspace bytes for the same sizes, 16-byte aligned; up to
 * twice 256 MB, or twice q_tokens heads (head_dim + 2) 4 bytes where that is more (a part for every
 * row over the prefix, and one over the own keys): 1.7 GB for 100000 single tokens, 32 heads of 128. */
typedef struct {
    const void* k;
    const void* v;
    int64_t k_stride, k_head_stride; /* aligned as those of bs_attention_args */
    int64_t v_stride, v_head_stride;
    uint32_t tokens; /* < 2^31 */
} bs_attention_prefix;

int bs_attention_shared_prefix(const bs_attention_args* args, const bs_attention_prefix* prefix, void* workspace,
                               uint64_t workspace_bytes, void* stream);
int bs_attention_shared_prefix_workspace(const bs_attention_args* args, const bs_attention_prefix* prefix, uint64_t* bytes);

#ifdef __cplusplus
}
#endif
#endif

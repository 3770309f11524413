/* libturtle_hip token-attention kernels (turtlevsr_amd/csrc/token.hip, token_attn_fwd.hip,
 * token_attn_bwd.hip), bound by
 * turtlevsr_amd/token_ops.py.
 *
 * Tokens are rows of heads: element (b, s, h, d) of a tensor at base[b * sb + s * ss + h * sh + d], strides in
 * elements, base and strides multiples of 16 bytes; D % 8 == 0, D <= 128. `dtype` 0 = fp32, 1 = bf16, 2 = fp16.
 * Results are dense [B][S][H][D] unless stated. All work is enqueued on `stream` (a hipStream_t); nothing is
 * allocated or synchronised. Return 0 or an error (negative: bad argument; positive: hipError_t).
 */
#ifndef TURTLE_TOKEN_H
#define TURTLE_TOKEN_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Rotation of channel pairs (2 i, 2 i + 1), i < npair: pair i turns by pos[axis[i]] * freq[i] / 2^64 revolutions
 * (freq: the pair's revolutions per unit of position, scaled by 2^64). */
typedef struct {
  uint64_t freq[64];
  uint8_t axis[64];
  int32_t npair;
  int32_t naxis;      /* positions per token, 1..4 */
} turtle_token_axes;

/* one tensor of a rotation call; x == NULL: absent */
typedef struct {
  const void* x;      /* input [B][S][H][D], strided */
  const void* dy;     /* backward only: gradient of y, strided (gb, gs, gh) */
  void* y;            /* forward: result; backward: gradient of x; dense */
  const float* w;     /* [D] gain of the norm, or NULL */
  int64_t sb, ss, sh;
  int64_t gb, gs, gh;
  int32_t H;
  int32_t pad;
} turtle_token_side;

/* y = R x of one or two tensors of the same tokens (inverse = 1: R^T, the gradient of it). pos [S][naxis]
 * (pos_b = 0) or [B][S][naxis] (pos_b = S * naxis), int32 or int64 (pos64 = 1). */
int turtle_token_rope(const turtle_token_side* a, const turtle_token_side* b, const turtle_token_axes* axes, const void* pos,
                      int64_t pos_b, int pos64, int64_t B, int64_t S, int D, int inverse, int dtype, void* stream);
/* y = R (w * x / sqrt(mean(x^2) + eps)) per token and head, of one or two tensors. */
int turtle_token_norm_rope_fwd(const turtle_token_side* a, const turtle_token_side* b, const turtle_token_axes* axes,
                               const void* pos, int64_t pos_b, int pos64, int64_t B, int64_t S, int D, float eps, int dtype,
                               void* stream);
/* its backward: side.y = dx; dw fp32 [2][D] (rows: sides a, b) or NULL, written, with ws of
 * turtle_token_norm_rope_workspace(B * S, D) bytes; fixed summation order. */
size_t turtle_token_norm_rope_workspace(int64_t tokens, int D);
int turtle_token_norm_rope_bwd(const turtle_token_side* a, const turtle_token_side* b, const turtle_token_axes* axes,
                               const void* pos, int64_t pos_b, int pos64, int64_t B, int64_t S, int D, float eps, float* dw,
                               void* ws, size_t ws_bytes, int dtype, void* stream);

/* Attention. Query i of sequence b stands at i + Sk - Sq, key j at j. z = scale q.k; softcap > 0:
 * z = softcap tanh(z / softcap) (scale, softcap, scale / softcap and both times log2 e finite in fp32); slopes [Hq] or NULL: z -= slope |distance|. Visible pairs: causal = 0, or key place
 * <= query place, or key place < prefix[b] (prefix NULL: 0); and, with documents (qdoc [B][Sq], kdoc [B][Sk]), equal
 * numbers >= 0. Query head h reads key head h / (Hq / Hk). A query that sees nothing gives zeros and no gradient.
 * Paged (table != NULL): key j of sequence b is row j % page of page table[b][j / page] of the pools k / v
 * ([npages][page][Hk][D], strides kb = pages, ks = rows, kh = heads); kv_lens / q_lens [B] (q_lens NULL: Sq) are the
 * keys and queries of each sequence, query i stands at kv_lens - q_lens + i, rows past q_lens give zeros; keys of
 * pages outside [0, npages) are seen by nobody. */
typedef struct {
  const void *q, *k, *v;
  int64_t qb, qs, qh, kb, ks, kh, vb, vs, vh;
  int32_t B, Sq, Sk, Hq, Hk, D;
  float scale, softcap;
  const float* slopes;
  const int32_t *prefix, *qdoc, *kdoc;
  int32_t causal;
  int32_t page, npages, maxpages;
  const int32_t *table, *kv_lens, *q_lens;
  void* o;            /* dense [B][Sq][Hq][D] */
  void* o_lo;         /* training: o's rounding remainder, as o (fp32: NULL), or NULL */
  float* lse;         /* training: [B][Hk][Sq * Hq / Hk] in log2 units, or NULL */
  void* ranges;       /* documents: scratch of turtle_token_attn_ranges bytes, kept for the backward (which writes marks there) */
  void* ws;           /* scratch of turtle_token_attn_workspace bytes (NULL when that is 0) */
  size_t ws_bytes;
} turtle_token_attn_args;

size_t turtle_token_attn_ranges(const turtle_token_attn_args* a);
size_t turtle_token_attn_workspace(const turtle_token_attn_args* a, int dtype);
int turtle_token_attn_fwd(const turtle_token_attn_args* a, int dtype, void* stream);

/* backward (not paged): q, k, v, o, o_lo, lse, ranges as the forward left them, ws scratch of
 * turtle_token_attn_bwd_workspace(&f, dtype) bytes (qdoc set where documents are used); dout strided (gb, gs, gh); dq, dk, dv
 * dense, dq or (dk and dv) NULL when not wanted; delta: scratch, B * Sq * Hq floats. Fixed summation order. */
typedef struct {
  turtle_token_attn_args f;
  const void* dout;
  int64_t gb, gs, gh;
  void *dq, *dk, *dv;
  float* delta;
} turtle_token_attn_grads;
size_t turtle_token_attn_bwd_workspace(const turtle_token_attn_args* a, int dtype);
int turtle_token_attn_bwd(const turtle_token_attn_grads* g, int dtype, void* stream);

#ifdef __cplusplus
}
#endif
#endif

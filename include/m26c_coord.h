/* C ABI of the coordinator-side operators between the return of a block and the next token: the block join
 * (rank sum, norm after the block, gate, residual, norm before the next block, wire rows), products with
 * MXFP4 weights for few rows, and log probabilities of given tokens with entropy and top alternatives.
 *
 * Plain pointers and sizes; every pointer except the argument structs, handles and error buffers is a device pointer of the
 * current device; `stream` is a hipStream_t (or null) of that device. The calls only launch (m26c_w4_new apart) and may be
 * captured into a graph. Return value: 0 on success, 1 for a bad argument (nothing is launched then), otherwise the
 * hipError_t of the failed launch. Nothing is kept between calls but what a caller passes in, so calls on different
 * streams may run at once as long as they write different memory. Outputs may not overlap inputs but where that is said. A
 * graph reads what its calls were given at each replay, a handle's weights among them: they have to live as long as it.
 *
 * The reference does these steps in separate kernels of its coordinator (crates/mimo26-coordinator/kernels/glue.cu, lm8.cu, sample.cu);
 * the entries here have no counterpart of the same form.
 */
#ifndef M26C_COORD_H
#define M26C_COORD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- block join --------------------------------------------------------------------------------------
 *   z  = ((p0 + p1) + p2) + p3              BF16 planes added in order in FP32
 *   z  = z * post_weight / sqrt(mean(z^2) + eps)        where post_weight is given
 *   h' = h + scale * gate * z                           FP32
 *   n  = h' * pre_weight / sqrt(mean(h'^2) + eps)
 * Outputs: h' (FP32), and n as BF16 (nearest even) and / or as wire rows: E4M3 codes with one UE8M0 byte per 32 values by
 * the rule of m26c_quantize_hidden, taken from the FP32 n. Sums are FP32 (a row whose sum of squares passes FP32's range is
 * normed to zero; squares under 2^-126 lose bits, which shows beside an eps as small only). A NaN or an infinity of a row stays in its row.
 * The plan holds what a program keeps from call to call. Pitches count elements (bytes for payload and scales); rows of
 * `cols` values, 1 <= cols <= 16384, a multiple of 32 for wire rows. Any alignment of the element type is accepted. A row's values
 * do not depend on the other rows; the order of its sums, and with that their last bits, depends on cols and, between
 * 2048 and 8192 of them, on whether the call has 512 rows or more. */
typedef struct m26c_join {
    int cols;
    int planes;               /* 1..4 */
    long plane_pitch;         /* of every plane, >= cols */
    long h_pitch;             /* of h and h_out, >= cols */
    long norm_pitch;          /* >= cols */
    const float* pre_weight;  /* [cols] */
    const float* post_weight; /* [cols] or null */
    int gate_cols;            /* 0: no gate, 1: one value per row, cols: one per value */
    long gate_pitch;          /* elements from a row's gate to the next; 0: the same for all rows */
    float scale;
    float eps;                /* > 0 */
    size_t payload_pitch, scales_pitch;
} m26c_join;

/* h_out may be h (in place); no other output may overlap an input. gate is read when gate_cols is not 0. norm may be
 * null, payload and scales may both be null; at least one of the two forms, or h_out alone, is written. */
int m26c_block_join(const m26c_join* plan, long rows, const float* h, const uint16_t* p0, const uint16_t* p1, const uint16_t* p2,
                    const uint16_t* p3, const float* gate, float* h_out, uint16_t* norm, uint8_t* payload, uint8_t* scales,
                    void* stream);

/* ---- products with MXFP4 weights -----------------------------------------------------------------------
 * y[r][j] = sum over k of x[r][k] * e2m1(code[j][k]) * 2^(scale[j][k / 32] - 127)
 * Weights in the form the experts' MXFP4 has in a checkpoint: [n][k / 2] payload bytes, low nibble = even k, 16-byte aligned,
 * [n][k / 32] scale bytes at any alignment; k a multiple of 32, n and k up to 2^24, and so are the pitches of x and y.
 * m26c_w4_new lays them out once in the order the matrix pipe reads, on the current device, and waits for that; the sources may
 * be freed afterwards. Scale bytes have to lie in [2, 252] wherever a group holds a nonzero code (the format's range in which
 * every weight is a normal number); a group of zeros may carry any byte.
 * Returns 1 for a bad argument or a stream that is being captured, 2 for a failed allocation or launch, 3 for a scale byte out
 * of that range. */
typedef struct m26c_w4 m26c_w4;
int m26c_w4_new(const uint8_t* payload, const uint8_t* scales, long n, long k, void* stream, m26c_w4** out, char* err, size_t errlen);
void m26c_w4_free(m26c_w4* w);

/* x: BF16 rows at x_pitch elements, 16-byte aligned and the pitch a multiple of 8. y: FP32, or BF16 (nearest even) when
 * y_bf16 is not 0, rows at y_pitch elements. Sums are FP32; their order, and with that the last bits, depends on rows, n and k. Made
 * for up to 64 rows; any number is taken, 16 or 32 at a time, which widens the weights again for each (4096 x 4096: 512 rows 28 us,
 * 2048 rows 179). The current device has to be the one the weights are on. */
int m26c_w4_matvec(const m26c_w4* w, const uint16_t* x, long x_pitch, int rows, void* y, int y_bf16, long y_pitch, void* stream);

/* The same on wire rows: E4M3 codes and one UE8M0 byte per 32 values, at their own pitches in bytes (request-frame rows are
 * read in place); payload 8-byte aligned, its pitch a multiple of 8. Codes are taken exactly for scale bytes 3..246. Byte
 * 255 and NaN codes make their row NaN; above 246 a code past BF16's range counts as infinite; for bytes 0..2 a code's value
 * is rounded to a multiple of 2^-133 (nearest even). */
int m26c_w4_matvec_fp8(const m26c_w4* w, const uint8_t* payload, size_t payload_pitch, const uint8_t* scales, size_t scales_pitch,
                       int rows, void* y, int y_bf16, long y_pitch, void* stream);

/* ---- log probabilities -------------------------------------------------------------------------------------
 * Per row of `vocab` logits l (FP32, or BF16 when bf16 is not 0; `pitch` elements from row to row, any alignment of the type),
 * with t = scale * l (0 < scale <= 2^20: one over a temperature), m = max t, Z = sum exp(t - m):
 *   given_logprob[r][i] = t[given[r][i]] - m - ln Z     NaN for an id outside [0, vocab) (padding)
 *   entropy[r]          = ln Z - (1 / Z) sum exp(t - m) (t - m)
 *   top_ids[r][0..top), top_logprob: the largest logits in descending order, equal ones by the lower id
 * A logit of -infinity is a masked token: probability 0, log probability -infinity, never an alternative; where fewer than
 * `top` are left, the id is -1 and the log probability -infinity. A row with nothing left gives -infinity, entropy 0
 * and no alternatives. NaN or +infinity in a row makes its log probabilities and entropy NaN (ids stay ordered; a
 * NaN is never an alternative). Log probabilities are never above 0 and entropies never below. given / given_logprob may be
 * null when n_given is 0, the top arrays when top is 0, entropy always. 0 <= top <= min(32, vocab), vocab and n_given <= 2^30.
 * `workspace`: at least m26c_token_logprobs_workspace(rows, vocab, top) bytes, 16-byte aligned, its content irrelevant before
 * and after; may be null when that is 0. Fewer rows may need more; 8192 * (16 + 8 * top) bytes do for any call. Calls that may
 * overlap need workspaces of their own. A row's values do not depend on the other rows; which sums are formed first, and with
 * that the last bits, depends on rows and vocab and, in long rows, on a row's address modulo 16. */
size_t m26c_token_logprobs_workspace(int rows, int vocab, int top);
int m26c_token_logprobs(const void* logits, int bf16, long pitch, int rows, int vocab, float scale, const int* given, int n_given,
                        float* given_logprob, float* entropy, int top, int* top_ids, float* top_logprob, void* workspace,
                        size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif

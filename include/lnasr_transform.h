/*
 * lnasr_transform.h -- feature transforms of liblnasr_hip.so: affine maps per speaker or class, and a projection with low-rank
 * adapters, with their gradients.  Contexts, errors and the conventions of pointers are lnasr_hip.h's; the ctypes table is
 * `TRANSFORM_SIGNATURES` in ln-asr_amd/lnasr/_ffi.py.
 */
#ifndef LNASR_TRANSFORM_H
#define LNASR_TRANSFORM_H

#include "lnasr_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* storage types beside LNASR_F64 and LNASR_F32 */
#define LNASR_F16 2
#define LNASR_BF16 3

/* Sends the context's further calls to another stream of its device (a hipStream_t; NULL is the default stream), behind what
 * was enqueued so far; own != 0: back to the context's own stream.  For callers whose device arrays are produced on a stream
 * of theirs.  The stream has to live until the context is sent elsewhere or destroyed; refused while either stream is being
 * captured.  A call of the feature transforms on device memory may be captured into a graph once it has run (its workspaces
 * then exist and stay, after the context is destroyed too); it is left out of the profile.  Graphs of one context share its
 * workspaces: a replay, other replays and the context's own calls run one after the other, as on one stream.
 * The stream belongs to the context, not to the thread that chose it: threads with streams of their own take a context each, or
 * choose and call under a lock of theirs (as the Python layer does). */
int lnasr_ctx_use_stream(lnasr_ctx* ctx, void* stream, int own);
/* 1: the context's stream is being captured (or is the default stream while another one is), 0: it is not; negative: an error */
int lnasr_ctx_capturing(lnasr_ctx* ctx);

/*
 * Between the features (lnasr_mfcc) and the bank (lnasr_decode ...): an affine transform per speaker or class, and a projection
 * that all rows share with a low-rank adapter per speaker beside it; with gradients.  The reference has none of these.
 *   Rows are packed; segment s (an utterance, a request) holds rows offsets[s] .. offsets[s + 1] - 1 of `rows` (offsets [S + 1]
 * int64, not falling; segments may be empty).  slots [S] int32 names the group (speaker) of each segment, several may name the
 * same one; NULL: segment s is group s, S == G.  Rows that belong to no segment are left as they were in y and dx.
 *   dtype: LNASR_F64, F32, F16 or BF16, the type of every matrix; sums are held in 64 bits for F64, in 32 for the others, and
 * rounded once.  ld*: elements from one row to the next.  No alignment is asked for beyond that of the type.
 *   Arrays may be host or device memory as everywhere; host offsets and slots are checked, device ones are brought into range
 * (values out of order then give numbers without meaning, no access out of bounds).  An output may not overlap an input or
 * another output, from its first element to its last (columns of one buffer beside each other do).  With device arrays the call
 * only enqueues.  Threads may share a context for the calls below: they run one after the other (the context's other entry points
 *   belong to one thread at a time). */

/* y[r] = W[k] x[r] + bias[k], k the group of row r: x [rows, din], w [G, dout, din], bias [G, dout] or NULL, y [rows, dout].
 * A host slot outside [0, G) is refused, rows of such a device slot are left as they were. */
int lnasr_affine(lnasr_ctx* ctx, int dtype, const void* x, int64_t rows, int din, int64_t ldx, const int64_t* offsets,
                 const int32_t* slots_or_null, int S, const void* w, const void* bias_or_null, int G, int dout, void* y, int64_t ldy);
/* From dy = dL/dy: dx[r] = W[k]^T dy[r], dw[k] = sum over the rows of group k of dy x^T, dbias[k] = sum of dy (a group without
 * rows: zeros).  Each may be NULL (dbias only with dw); x is read for dw only, w for dx only.  The sums run in the order of the
 * batch: the same bits every time. */
int lnasr_affine_grad(lnasr_ctx* ctx, int dtype, const void* x, int64_t rows, int din, int64_t ldx, const int64_t* offsets,
                      const int32_t* slots_or_null, int S, const void* w, int G, int dout, const void* dy, int64_t lddy,
                      void* dx_or_null, int64_t lddx, void* dw_or_null, void* dbias_or_null);
/* y[r] = W x[r] + bias + scale[k] B[k] (A[k] x[r]): w [dout, din], bias [dout] or NULL, a [G, rank, din], b [G, dout, rank],
 * scale [G] fp64 or NULL (1).  Slot -1: the projection alone.  The middle (scale A x; in the gradients scale B^T dy, too) is held in
 * 64 bits for F64, in 32 for the others. */
int lnasr_projection(lnasr_ctx* ctx, int dtype, const void* x, int64_t rows, int din, int64_t ldx, const int64_t* offsets,
                     const int32_t* slots_or_null, int S, const void* w, const void* bias_or_null, int dout, const void* a,
                     const void* b, const double* scale_or_null, int G, int rank, void* y, int64_t ldy);
/* dx = W^T dy + scale A^T B^T dy, da[k] = sum scale (B^T dy) x^T, db[k] = sum dy (scale A x)^T, dw = sum dy x^T over the rows of
 * all segments, dbias = sum dy.  Each may be NULL (dbias only with dw); an input that no wanted gradient needs is not read. */
int lnasr_projection_grad(lnasr_ctx* ctx, int dtype, const void* x, int64_t rows, int din, int64_t ldx, const int64_t* offsets,
                          const int32_t* slots_or_null, int S, const void* w, int dout, const void* a, const void* b,
                          const double* scale_or_null, int G, int rank, const void* dy, int64_t lddy, void* dx_or_null,
                          int64_t lddx, void* da_or_null, void* db_or_null, void* dw_or_null, void* dbias_or_null);

#ifdef __cplusplus
}
#endif
#endif /* LNASR_TRANSFORM_H */

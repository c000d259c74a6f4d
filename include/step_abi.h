/*
 * step_abi.h — C ABI of the MI355X (gfx950) operators of a training step that
 * stand next to the gradient exchange of ring_abi.h: the embedding lookup and
 * its gradient, the sum of the rows an allgather of sparse gradients delivers,
 * and the orthogonalised update of a matrix.
 *
 * The reference gathers an IndexedSlices instead of reducing it
 * (tensorflow/contrib/mpi_collectives/__init__.py:146-157) and leaves what
 * comes before and behind the exchange to the framework around it.
 *
 * Conventions, as in ring_abi.h: plain C, an int status, every device entry
 * point asynchronous on the stream it is given (a hipStream_t as void*; NULL =
 * the default stream) on the calling thread's current device. Nothing here
 * allocates, synchronises or keeps anything between calls: scratch memory is
 * the caller's `workspace`, whose size a *_workspace function tells, so every
 * call may be recorded into a HIP graph, and calls on several streams are
 * independent as long as each has a workspace of its own. A workspace needs no
 * initialisation and starts on a 256-byte boundary.
 */
#ifndef STEP_ABI_H_
#define STEP_ABI_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define STEP_ABI_VERSION 1

/* Element types; the first three have the codes of enum ring_dtype. */
enum step_dtype { STEP_F32 = 0, STEP_I32 = 1, STEP_I64 = 2, STEP_BF16 = 3, STEP_F16 = 4 };

/* Status codes, those of enum ring_status. */
enum step_status {
  STEP_OK = 0,
  STEP_ERR_DTYPE = 1,    /* an element type the call does not take */
  STEP_ERR_ARGUMENT = 2, /* null pointer with a non-zero size, a workspace that is too small ... */
  STEP_ERR_HIP = 3,      /* a HIP runtime call failed: step_last_hip_error() */
  STEP_ERR_LIMIT = 5     /* more than 2^31 - 1 tokens or rows, 67,107,840 columns, or 2^32 - 1 lanes of a launch:
                            2^26 tokens of a lookup of rows of 4 KiB, 2^27 of their gradient (half as many at 8 KiB),
                            2^30 rows of a gradient; a matrix to orthogonalise of more than 2^20 a side or 2^33 entries */
};

int step_abi_version(void);
const char* step_status_string(int status);
/* hipError_t of the most recent failing HIP call on this thread (0 if none). */
int step_last_hip_error(void);

/* ---- embedding ------------------------------------------------------------
 * Ids are STEP_I32 or STEP_I64, `tokens` of them one behind the other. An id
 * outside [0, rows) (a padding id of -1, say) reads nothing: its row of the
 * lookup is zero, and it contributes nothing to a gradient or a sum. Values are
 * STEP_F32, STEP_BF16 or STEP_F16; the columns of a row are contiguous, rows
 * are `*_stride` elements apart. */

/* out[t, :] = round(scale * f32(weight[ids[t], :])); out is contiguous. */
int step_embedding_lookup(const void* ids, int id_type, size_t tokens, const void* weight, int dtype, size_t rows,
                          size_t width, size_t weight_stride, float scale, void* out, void* stream);

/* out[v, :] = round(scale * sum of f32(grad[t, :]) over the t with ids[t] = v),
 * for every row v < rows (0 where no token has it). The sum is taken in 32 bits
 * in the order of t, for a row with more than step_embedding_piece(tokens) (64 at
 * least) tokens in pieces of at most that many whose sums are added in order: the
 * same bits on every call. out is contiguous, of grad's type. */
size_t step_embedding_piece(size_t tokens);
size_t step_embedding_gradient_workspace(size_t tokens, size_t rows, size_t width);
int step_embedding_gradient(const void* ids, int id_type, size_t tokens, const void* grad, int dtype, size_t rows,
                            size_t width, size_t grad_stride, float scale, void* out, void* workspace,
                            size_t workspace_bytes, void* stream);

/* The same sum with one row for each distinct id in [0, rows), in ascending
 * order: out_ids[u] (of id_type) and out_values[u, :] for u < *out_count, a
 * 64-bit count in device memory. out_ids and out_values have room for
 * min(tokens, rows) rows; what lies behind the last row is left as it was. */
size_t step_sum_slices_workspace(size_t tokens, size_t rows, size_t width);
int step_sum_slices(const void* ids, int id_type, size_t tokens, const void* values, int dtype, size_t rows,
                    size_t width, size_t values_stride, float scale, void* out_ids, void* out_values,
                    int64_t* out_count, void* workspace, size_t workspace_bytes, void* stream);

/* ---- orthogonalised updates --------------------------------------------------
 * Newton-Schulz steps on the update U of each matrix,
 *   X = U / (|U|_F + eps), then `steps` (1 to 64) times  A = X X^T,  X = a X + (b A + c A A) X
 * (on the transposed matrix if rows > cols; the result is the same), with
 * coefficients[3 k .. 3 k + 2] = a, b, c of step k in host memory.
 *
 * A list of matrices is one call: all of them go through each product in one
 * launch (lists of more than 64 batches, 32 shapes or 2^26 elements in several
 * rounds that use the workspace in turn). Matrices are contiguous, `count` of them one behind
 * the other.
 *
 * precise = 0: the products take fp16 operands (the rest of the iterate is kept
 * beside them): the norm of the difference is 0.05 to 0.3 % of the result's, about
 * bfloat16's own rounding; up to 0.6 % with fewer than eight rows (or columns).
 * precise = 1: three products of split operands: about 1e-6 off; matrices of at
 * most 64 x 256 (or 256 x 64) always have these, whatever else is in the list. Iterates must
 * stay below 64 in every entry and X X^T below 4, which coefficients that bring
 * singular values towards 1 see to. */
typedef struct step_matrix {
  const void* grad;  /* U, or the gradient (step_muon) */
  float* momentum;   /* step_muon: the momentum buffer, updated; else unused */
  void* out;         /* the result, or the weights (step_muon), updated */
  size_t rows, cols; /* at most 2^20 a side, 2^33 entries */
  size_t count;
  float rate;        /* step_muon: learning rate of this batch's matrices */
} step_matrix;

/* The side of the tiles that a product of the first round of a list is cut into: product = 0 X X^T, 1 A A, 2 B X, 3 the
 * last B X. 0 if the list takes no such product (it is empty, or its matrices are small). For tests and tuning. */
int step_orthogonalize_side(const step_matrix* list, size_t length, int precise, int product);

/* Bytes of workspace for a list: 0 if none is needed. */
size_t step_orthogonalize_workspace(const step_matrix* list, size_t length, int precise);
int step_orthogonalize(const step_matrix* list, size_t length, int dtype, int out_dtype, int precise, int steps,
                       const float* coefficients, float eps, void* workspace, size_t workspace_bytes, void* stream);

/* One optimizer step: momentum = mu momentum + grad; U = grad + mu momentum
 * (nesterov) or momentum; out = keep out - rate NS(U). Gradient and weights
 * have type dtype; the new weights are computed in 32 bits and rounded once. */
int step_muon(const step_matrix* list, size_t length, int dtype, int precise, int steps, const float* coefficients,
              float eps, float momentum, int nesterov, float keep, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* STEP_ABI_H_ */

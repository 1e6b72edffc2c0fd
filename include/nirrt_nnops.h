/* nirrt_nnops.h - C ABI of the dense operators of the guidance network's layers and of its training step in libnirrt_hip.so (gfx950).
 *
 * Conventions as in nirrt_pointops.h: pointers are DEVICE addresses unless marked HOST, `stream` is a hipStream_t (0 = default stream),
 * the tensors and the stream belong to the calling thread's CURRENT device, every function returns 0 on success and < 0 on error
 * (-1 bad argument, -2 HIP error); nothing throws, nothing waits for the device, and all launches can be captured into a graph.
 * Workspaces are the caller's: at least the bytes that the _workspace function of the same sizes returns, 256-byte aligned, in use until
 * the launches have run (two captured graphs that may replay at the same time need one each).
 * Element types: NIRRT_NN_F32 / _BF16 / _F16; sums are held in 32 bits.  Matrices are row-major with a row stride in elements (ld >= row
 * length); dimensions are at most 2^31 - 4096, their products may be larger. */
#ifndef NIRRT_NNOPS_H
#define NIRRT_NNOPS_H
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { NIRRT_NN_F32 = 0, NIRRT_NN_BF16 = 1, NIRRT_NN_F16 = 2 };
enum { NIRRT_NN_ACT_NONE = 0, NIRRT_NN_ACT_RELU = 1, NIRRT_NN_ACT_GELU = 2, NIRRT_NN_ACT_SILU = 3 };

/* y = act(x w^T + b) + r: x (m, k), w (n, k), b (n,) or NULL, r (m, n) or NULL, y (m, n).  z (m, n) contiguous or NULL receives the
 * pre-activation x w^T + b for nirrt_nn_linear_backward.  The workspace's size depends on the operands' addresses and strides (whole aligned
 * 16-byte chunks or not); workspace may be NULL if it is 0. */
int64_t nirrt_nn_linear_workspace(int dtype, const void *x, int64_t ldx, const void *w, int64_t ldw, int64_t m, int64_t n, int64_t k);
int nirrt_nn_linear(int dtype, int act, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *b, const void *r, int64_t ldr,
                    void *y, int64_t ldy, void *z, int64_t m, int64_t n, int64_t k, void *workspace, void *stream);

/* Gradients of nirrt_nn_linear: dz = dy act'(z) (rounded to the element type), dx = dz w, dw = dz^T x, db = column sums of dz.  z as the
 * forward pass left it (NULL for NIRRT_NN_ACT_NONE; the forward's y may stand for z with NIRRT_NN_ACT_RELU and no r); dy (m, n).  dx
 * (m, k), dw (n, k) contiguous, db (n,): each may be NULL (not wanted).  The gradient of r is dy itself. */
int64_t nirrt_nn_linear_backward_workspace(int dtype, int act, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *dy, int64_t lddy,
                                           int64_t m, int64_t n, int64_t k);
int nirrt_nn_linear_backward(int dtype, int act, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *z, const void *dy,
                             int64_t lddy, void *dx, void *dw, void *db, int64_t m, int64_t n, int64_t k, void *workspace, void *stream);

/* Softmax cross entropy of the classes' scores l = x w^T + b without keeping them: x (rows, k), w (classes, k), b (classes,) or NULL,
 * target int64 (rows,), class_weight f32 (classes,) or NULL.  A row whose target is ignore_index counts for nothing; any other target
 * outside [0, classes) gives NaN.  lse (rows, 2) = the largest l and log sum exp(l - it), nll (rows,) = weight * (log sum exp l - l[target]) (0 where ignored),
 * total (3,) = {sum of nll, sum of the weights, their quotient}, all f32.  Rows may lie any distance apart; k elements are
 * 4 MB at most, and more than 8 classes take less than 2^29 rows.
 * More than 8 classes: the workspace ends in room for a copy of x, X = rows * k' elements, and one of w, W = classes * k' (k' = k rounded
 * up to 16 bytes; X and W each rounded up to 256 bytes).  A copy is made where base, row stride and k are not all multiples of 16 bytes,
 * or the stride is above 4 MB; a caller whose x or w needs none may leave its bytes out. */
int64_t nirrt_nn_cross_entropy_workspace(int dtype, int64_t rows, int64_t classes, int64_t k);
int nirrt_nn_cross_entropy(int dtype, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *b, const int64_t *target,
                           const float *class_weight, int64_t ignore_index, float *lse, float *nll, float *total, int64_t rows,
                           int64_t classes, int64_t k, void *workspace, void *stream);

/* Its gradients: c_i = dloss_i * weight(target_i) (0 where ignored), g_iv = c_i (exp(l_iv - lse_i) - [v = target_i]), dx = g w, dw = g^T x,
 * db = column sums of g.  dloss f32: `dloss_stride` 1 = one value per row, 0 = one value for all rows; where `total` is given, it is
 * divided by total[1] (the mean over the weights).  lse as the forward pass left it.  dx (rows, k), dw (classes, k) contiguous,
 * db (classes,); each may be NULL.  More than 8 classes: the workspace ends in room for a copy of w, W bytes as above, which may be left
 * out where w needs none. */
int64_t nirrt_nn_cross_entropy_backward_workspace(int dtype, int64_t rows, int64_t classes, int64_t k);
int nirrt_nn_cross_entropy_backward(int dtype, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *b, const int64_t *target,
                                    const float *class_weight, int64_t ignore_index, const float *lse, const float *dloss,
                                    int dloss_stride, const float *total, void *dx, void *dw, void *db, int64_t rows, int64_t classes,
                                    int64_t k, void *workspace, void *stream);

/* norm (1,) f32 = the 2-norm of all elements of `count` contiguous tensors; tensors HOST arrays of device addresses, element counts and
 * types.  The sums run in a fixed order: the same tensors give the same bits. */
typedef struct nirrt_nn_tensor {
    const void *data;     /* DEVICE */
    void *out;            /* DEVICE: where nirrt_nn_scale_by_norm writes (may be data itself); not used by nirrt_nn_norm */
    int64_t n;
    int32_t dtype, out_dtype;
} nirrt_nn_tensor;
int64_t nirrt_nn_norm_workspace(const nirrt_nn_tensor *tensors, int32_t count);
int nirrt_nn_norm(const nirrt_nn_tensor *tensors, int32_t count, float *norm, void *workspace, void *stream);
/* out = data * min(1, max_norm / (norm + 1e-6)) for every tensor, norm read on the device.  A NaN norm gives NaN everywhere. */
int nirrt_nn_scale_by_norm(const nirrt_nn_tensor *tensors, int32_t count, const float *norm, float max_norm, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* NIRRT_NNOPS_H */

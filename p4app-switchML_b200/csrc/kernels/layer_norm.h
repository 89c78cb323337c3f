/* Layer norm over the last dimension, forward and backward.
 *
 *   s = x + residual (rounded to the type of x; s = x without a residual)
 *   y = (s - mean(s)) / sqrt(var(s) + eps) * weight + bias
 *
 * x, residual, y, sum, dy, dsum, dx: [rows, features], contiguous, all of `type`. weight and bias: [features] of `wtype`,
 * each may be NULL (ones and zeros). mean and rstd: one fp32 per row. Types: SML_NORM_F32, SML_NORM_BF16.
 * All pointers are aligned to their element (others are refused); up to 2^30 features. Statistics and sums are fp32.
 * Return 0, or < 0: -1 bad argument, -4 launch.
 */
#ifndef SWITCHML_LAYER_NORM_H_
#define SWITCHML_LAYER_NORM_H_

#ifdef __cplusplus
extern "C" {
#endif

enum { SML_NORM_F32 = 0, SML_NORM_BF16 = 1 };

/* `sum` receives s where there is a residual (else it is not written and may be NULL); mean and rstd may be NULL together. */
int switchml_layer_norm_forward(const void* x, const void* residual, const void* weight, const void* bias, void* y, void* sum,
                                float* mean, float* rstd, long long rows, int features, float eps, int type, int wtype,
                                void* stream);
/* Floats of workspace that the backward pass needs for these sizes. */
long long switchml_layer_norm_workspace(long long rows, int features, int type);
/* dx = d(loss)/ds, with dsum (may be NULL: zeros), the gradient that reached s by another way, added; dweight and dbias, of
 * `wtype`, may be NULL (not wanted). `workspace` need not be initialised. The same bits in every run. */
int switchml_layer_norm_backward(const void* dy, const void* dsum, const void* s, const void* weight, const float* mean,
                                 const float* rstd, void* dx, void* dweight, void* dbias, float* workspace, long long rows,
                                 int features, int type, int wtype, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SWITCHML_LAYER_NORM_H_ */

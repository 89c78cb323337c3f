/* AdamW over many tensors in one launch, and the norm of all their gradients.
 *
 * One step of a tensor, every operation rounded to fp32 once, in this order:
 *   g' = g * clip
 *   m  = m * beta1 + g' * (1 - beta1)
 *   v  = v * beta2 + (g' * (1 - beta2)) * g'
 *   p  = p * (1 - lr * decay) - lr / (1 - beta1^t) * (m / (sqrt(v) / sqrt(1 - beta2^t) + eps))
 * (the line for p may be a few units in the last place of its second term off, and a v below 2^-126 counts as 2^-126 there).
 *
 * Moments are fp32 or take 8 bits each. Then 32 values share a scale 2^(e - 134), stored as the byte e - 7 (e8m0), where
 * e is the exponent field of the largest magnitude among the 32, at least 8; the largest of them comes to lie in
 * [128, 256). A value over its scale, y, is rounded to e4m3 up or down at random: with t = y, or y + 2^-6 below 2^-6 (where
 * e4m3 has equal steps), the bits of t plus 20 random bits lose their last 20. A second moment above zero gets at least the
 * code 1. Where a value is not finite, its whole block is NaN from then on. The random bits: 16 from the hash of
 * (seed, step, place) and a final 1 000; the first moment takes the low half of the hash, the second the high half.
 *
 * A parameter in bf16 has a remainder of 16 bits, and both together are the fp32 value p of the formulas: the parameter is
 * its bits plus 0x8000 without the low half, the remainder that low half. So the value is (param << 16) + remainder, the
 * remainder taken as signed. What else writes to the parameter is off by half of a bf16 step at most; nothing
 * takes the parameter back to what it was.
 *
 * Parameters and gradients lie at any multiple of their element. Flat buffers are read in whole vectors: fp32 ones (moments with
 * bits = 32, what switchml_adamw_masters writes) begin at a multiple of 32 bytes, remainders of 16, moments with bits = 8 of 8.
 *
 * Return 0, or < 0: -1 bad argument, -4 launch.
 */
#ifndef SWITCHML_ADAMW_H_
#define SWITCHML_ADAMW_H_

#ifdef __cplusplus
extern "C" {
#endif

enum { SML_ADAMW_F32 = 0, SML_ADAMW_BF16 = 1 };

/* A tensor's state begins at a multiple of this many values. */
enum { SML_ADAMW_ALIGN = 256 };
/* Tensors of one launch, at most. */
enum { SML_ADAMW_TENSORS = 384 };

typedef struct SmlAdamwTensor {
  void* param;
  const void* grad;   /* of the parameter's type; not read by switchml_adamw_masters */
  long long numel;
  unsigned place;     /* state begins at value place * SML_ADAMW_ALIGN of the flat buffers */
  int step;           /* index into SmlAdamwState.steps */
} SmlAdamwTensor;

typedef struct SmlAdamwState {
  void* exp_avg;                    /* flat: fp32, or bytes with bits = 8 */
  void* exp_avg_sq;
  unsigned char* exp_avg_scale;     /* flat, one byte for 32 values; NULL with bits = 32 */
  unsigned char* exp_avg_sq_scale;
  short* remainder;                 /* flat, of bf16 parameters; NULL with fp32 ones */
  int* steps;                       /* steps taken, one for each tensor; counted on by the kernel */
  int* ticket;                      /* one int, zero between launches */
  int bits;                         /* 32 or 8 */
  unsigned seed;
  unsigned long long first;         /* number of the first value of the flat buffers, for the random bits */
} SmlAdamwState;

typedef struct SmlAdamwStep {
  double lr, beta1, beta2, eps, decay;
  const float* lr_tensor;           /* fp32 in device memory, in place of lr; or NULL */
  const float* norm;                /* of all gradients; or NULL: no clipping */
  float max_norm;                   /* where the norm is not finite the step is left out: nothing changes */
} SmlAdamwStep;

/* One step of `count` tensors of one type (any number: cut into launches). */
int switchml_adamw_step(const SmlAdamwTensor* tensors, int count, const SmlAdamwState* state, const SmlAdamwStep* step, int type,
                        void* stream);
/* The fp32 values of `count` tensors of one type, each at its place of the flat buffer `out`, zeros up to the next
 * multiple of SML_ADAMW_ALIGN. */
int switchml_adamw_masters(const SmlAdamwTensor* tensors, int count, const short* remainder, float* out, int type, void* stream);

typedef struct SmlNormTensor {
  const void* data;
  long long numel;
  int type;
} SmlNormTensor;

/* Doubles of workspace for `count` tensors. */
long long switchml_grad_norm_workspace(int count);
/* out = sqrt of the sum of squares of all tensors, summed in fp64; the same bits in every run. At most 2^43 values in all.
 * `workspace` need not be initialised. `ticket`: one int, zero between launches, saves a launch; or NULL. */
int switchml_grad_norm(const SmlNormTensor* tensors, int count, double* workspace, int* ticket, float* out, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SWITCHML_ADAMW_H_ */

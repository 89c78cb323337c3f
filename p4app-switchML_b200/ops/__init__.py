"""Kernel-level operations: the CPU oracle, the single-GPU emulation of the aggregation
kernels, the tcgen05 weight-gradient GEMM, and what a training step does around its gradients: layer norm
forward and backward, the norm of all gradients, AdamW over all tensors."""

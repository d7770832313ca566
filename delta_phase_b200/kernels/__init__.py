"""Fused B200 kernels and their functional API (drop-in for ``delta_phase.kernels``)."""
from .chunk_delta import (
    DeltaPhaseCudaFunction,
    DeltaPhaseTritonFunction,
    LaplaceCudaFunction,
    chunkwise_forward,
    complex_beta_chunkwise,
    cuda_available,
    decode_step,
    delta_phase_chunkwise_fused,
    gram_matrix_cuda,
    gram_matrix_triton,
    laplace_chunkwise,
    phasor,
    triton_available,
)
from .distill import DistillCudaFunction, distill_loss, distill_loss_and_grad
from .gated_scan import GatedScanCudaFunction, gated_scan, gated_scan_step
from .layer_norm import LayerNormCudaFunction, layer_norm

__all__ = [
    "delta_phase_chunkwise_fused",
    "triton_available",
    "DistillCudaFunction",
    "GatedScanCudaFunction",
    "LayerNormCudaFunction",
    "DeltaPhaseTritonFunction",
    "DeltaPhaseCudaFunction",
    "LaplaceCudaFunction",
    "cuda_available",
    "chunkwise_forward",
    "complex_beta_chunkwise",
    "decode_step",
    "distill_loss",
    "distill_loss_and_grad",
    "gated_scan",
    "gated_scan_step",
    "gram_matrix_cuda",
    "gram_matrix_triton",
    "laplace_chunkwise",
    "layer_norm",
    "phasor",
]

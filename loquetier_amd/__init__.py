"""loquetier_amd: MI355X-native Segmented Multi-LoRA Multiplication (SMLM) and what stands
between a decoder layer's projections.

The SMLM path of Loquetier: the HIP kernels and their C ABI (csrc/, include/smlm.h)
and the Python operator surface the reference's LoRA layer calls (ops/_kernels.py,
kernel_utils.py, mixed_lora.py, segments.py).  Beside it, over the same flat batch: norms
and rotation of queries and keys (kernel_utils.py), a paged key-value cache and the
attention over it (kvcache.py); and around a fine-tuning step the norms with the residual's
addition and the loss over the vocabulary (kernel_utils.py) and the update of all adapters
(optim.py).
"""
__version__ = "0.1.0"

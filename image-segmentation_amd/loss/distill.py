"""Distillation from a teacher's stored top logits, a loss beside Dice and focal with the same call form `loss(pred, target)`.
The reference trains on label maps only and has no counterpart.  CUDA tensors run the HIP kernels of segk.distill; CPU tensors
the same formulas in torch ops."""
from segk.distill import TopLogits, distill_loss_topk, top_logits  # noqa: F401

from .ops import AttentionGeometry, AttentionPlan, CudaOps, KernelError, TokenHistory, load_library

__all__ = ["AttentionGeometry", "AttentionPlan", "CudaOps", "KernelError", "TokenHistory",
           "load_library"]

"""Import-path shim: ``kernels.grouped_gemm`` beside the other operators of the ``kernels`` package."""
from flydsl_b200.kernels.grouped_gemm import (grouped_gemm, grouped_gemm_dgrad, grouped_gemm_wgrad,  # noqa: F401
                                              grouped_linear)

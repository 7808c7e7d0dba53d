"""Import-path shim: ``kernels.moe_routing`` beside the other operators of the ``kernels`` package."""
from flydsl_b200.kernels.moe_routing import (RoutedRows, moe_combine, moe_permute, route_rows,  # noqa: F401
                                             topk_gating)

"""Import-path shim: ``kernels.lora`` beside the other operators of the ``kernels`` package."""
from flydsl_b200.kernels.lora import lora_add  # noqa: F401

"""umsx: B200-native MoE-layer hot path of appatalks/unified-memory-scheduler.

The compute runs in libumsx.so (hand-written sm_100a CUDA behind a C ABI,
include/umsx.h); this package holds the Python bindings and the layer configs.
The directory name is not a Python identifier, so __graft_entry__.load_package()
registers it as `umsx_b200`.
"""
from . import configs, umsx  # noqa: F401
from .umsx import (MoeLayer, MoeStack, UmsxError, combine, fp8_grouped_mm, fp8_mm, fp8_quantize, group_rows,  # noqa: F401
                   grouped_mm, grouped_mm_dw, grouped_mm_dx, kernel_launches, lib, load_gguf_experts)

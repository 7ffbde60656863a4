"""glaucis_b200: B200-native (sm_100a) kernels for the two kernels scored by the
Glaucis kernel evaluator — the block-wise FP8 grouped matmul and the chunked
Gated Linear Attention forward — behind the reference templates' call
signatures, and the operators that stand around the experts' products of a
mixture-of-experts layer: RMS norm into their operands, router, exchange of
rows, and 4-bit products for generated tokens.  See include/glaucis_b200.h for
the C ABI."""
from . import _lib
from .ops import (chunk_gla, chunk_gla_fwd, device_status, gmm_fp8_blockwise, gmm_fp8_fwd, gmm_w4_fwd,
                  moe_combine, moe_dispatch, moe_dispatch_quant, moe_route, quant_act_1x128,
                  quant_w4_128x1, quant_w_128x128, rms_norm, rms_norm_quant_1x128)

__all__ = ["chunk_gla", "chunk_gla_fwd", "device_status", "gmm_fp8_blockwise", "gmm_fp8_fwd",
           "gmm_w4_fwd", "moe_combine", "moe_dispatch", "moe_dispatch_quant", "moe_route",
           "quant_act_1x128", "quant_w4_128x1", "quant_w_128x128", "rms_norm",
           "rms_norm_quant_1x128", "_lib"]

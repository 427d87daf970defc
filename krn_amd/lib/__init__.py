"""krn's library calls on gfx950: `matmul` with its fused epilogues, dispatched over the reference's AMD candidate
order (hipBLASLt, then krn's own tile program); microscaled 4-bit matrices with their quantisation and product
(`mx_quantize`, `mx_dequantize`, `mx_matmul`), and a mixture-of-experts layer on them (`moe`)."""

from krn_amd.lib.lib import Declined, Epilogue, NoCandidate, Operands, Problem, choice, matmul
from krn_amd.lib.lib_moe import moe
from krn_amd.lib.lib_mx import MxMatrix, mx_dequantize, mx_matmul, mx_quantize

__all__ = ["Declined", "Epilogue", "MxMatrix", "NoCandidate", "Operands", "Problem", "choice", "matmul", "moe",
           "mx_dequantize", "mx_matmul", "mx_quantize"]

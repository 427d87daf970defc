"""krn's library calls on gfx950: `matmul` with its fused epilogues, dispatched over the reference's AMD candidate
order (hipBLASLt, then krn's own tile program); microscaled 4-bit matrices with their quantisation and product
(`mx_quantize`, `mx_dequantize`, `mx_matmul`), and a mixture-of-experts layer on them (`moe`); a paged key-value cache with
what fills it and attends over it (`rotary_append`, `cache_attention`)."""

from krn_amd.lib.lib import Declined, Epilogue, NoCandidate, Operands, Problem, choice, matmul
from krn_amd.lib.lib_cache import KvCache, Rotary, Sequences, cache_attention, rotary_append
from krn_amd.lib.lib_moe import moe
from krn_amd.lib.lib_mx import MxMatrix, mx_dequantize, mx_matmul, mx_quantize

__all__ = ["Declined", "Epilogue", "KvCache", "MxMatrix", "NoCandidate", "Operands", "Problem", "Rotary", "Sequences",
           "cache_attention", "choice", "matmul", "moe", "mx_dequantize", "mx_matmul", "mx_quantize", "rotary_append"]

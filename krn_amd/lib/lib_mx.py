"""Microscaled 4-bit matrices (OCP MX, MXFP4): values to them and back, and the product of two.

A row of k values is ceil(k / 32) blocks; a block is 32 e2m1 codes (magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one e8m0
byte s, its values code * 2^(s - 127), NaN for s = 255. The reference has no 4-bit type: these operations stand beside its
`lib.matmul` (reference src/krn/lib/lib.py:581-615), whose epilogues the product takes.
"""

from krn_amd.dtypes import BF16, F16, F32, U8, Dtype, of
from krn_amd.lib.calls import LibraryCall, Work, tensor
from krn_amd.lib.lib import FLOATS, Epilogue
from krn_amd.runtime import library
from krn_amd.runtime.hip import HIPDevice, HIPStream, HIPTensor

BLOCK = 32


class MxMatrix:
    """A matrix of `k` values a row in microscaled 4 bits: `codes` (rows, 16 * blocks) bytes, two codes a byte with the
    first in the low nibble, and `scales` (rows, blocks) bytes, both u8 tensors; blocks = ceil(k / 32). The codes of a last
    block past k are zero, and so codes and scales of whole blocks are the format's usual ones as they lie."""

    def __init__(self, codes: HIPTensor, scales: HIPTensor, k: int) -> None:
        tensor(codes, "codes", 2, (U8,))
        tensor(scales, "scales", 2, (U8,))
        if not isinstance(k, int) or k < 1:
            raise ValueError(f"an MX matrix has rows of one value or more, got k = {k!r}")
        rows, blocks = codes.shape[0], -(-k // BLOCK)
        if codes.shape != (rows, 16 * blocks) or scales.shape != (rows, blocks):
            raise ValueError(f"rows of {k} values are {16 * blocks} bytes of codes and {blocks} scales, got codes "
                             f"{codes.shape} and scales {scales.shape}")
        self.codes, self.scales, self.shape, self.device = codes, scales, (rows, k), codes.device

    @classmethod
    def empty(cls, device: HIPDevice, rows: int, k: int) -> "MxMatrix":
        """Uninitialized, for `mx_quantize(..., out=...)`."""
        blocks = -(-k // BLOCK)
        return cls(device.empty(U8, rows, 16 * blocks), device.empty(U8, rows, blocks), k)

    @property
    def pointers(self) -> tuple[int, int]:
        return self.codes.pointer, self.scales.pointer

    def __repr__(self) -> str:
        return f"MxMatrix{list(self.shape)}"


def matrix(value: object, what: str) -> MxMatrix:
    if not isinstance(value, MxMatrix):
        raise TypeError(f"{what} is an MxMatrix (mx_quantize makes one), not {type(value).__name__}")
    return value


@LibraryCall
def mx_quantize(x, *, out: MxMatrix | None = None) -> Work:
    """The MX matrix of `x`, (rows, k) of f32, f16 or bf16: a block's scale is the power of two that brings its largest
    magnitude into [4, 8), a code the nearest e2m1 value of the scaled element, halves to even, 6 beyond 6. A block with
    a NaN or an infinity gets scale 255: all of it reads as NaN."""
    tensor(x, "x", 2, (F32, F16, BF16))
    rows, k = x.shape
    if k < 1:
        raise ValueError("x has rows of one value or more")
    if out is not None and matrix(out, "out").shape != (rows, k):
        raise ValueError(f"out has shape {out.shape}, x {(rows, k)}")
    result = out if out is not None else MxMatrix.empty(x.device, rows, k)
    call = library.mx_quantize_call(x.dtype, x.pointer, *result.pointers, rows, k)
    return Work("mx_quantize", x.device, result, (x, result), lambda stream: call(stream.handle))


@LibraryCall
def mx_dequantize(a, *, dtype: Dtype = BF16, out=None) -> Work:
    """The values of an MX matrix as f32, f16 or bf16 (`dtype`, or the type of `out`). f32 holds every value of finite
    magnitude exactly, bf16 too; f16 rounds."""
    matrix(a, "a")
    element = out.dtype if isinstance(out, HIPTensor) else of(dtype)
    if element not in FLOATS:
        raise ValueError(f"the values of an MX matrix are written as f16, bf16 or f32, not {element}")
    if out is not None and tensor(out, "out", 2, FLOATS).shape != a.shape:
        raise ValueError(f"out has shape {out.shape}, the matrix {a.shape}")
    result = out if out is not None else a.device.empty(element, *a.shape)
    call = library.mx_dequantize_call(*a.pointers, element, result.pointer, *a.shape)
    return Work("mx_dequantize", a.device, result, (a, result), lambda stream: call(stream.handle))


@LibraryCall
def mx_matmul(a, b, *, epilogue: Epilogue = Epilogue.NONE, bias=None, dtype: Dtype = BF16, out=None) -> Work:
    """`a @ b.T` of the MX matrices a (m, k) and b (n, k), the layout of a linear layer's weight, with an epilogue of
    `lib.matmul`; float32 sums, rounded once to f32, f16 or bf16 (`dtype`, or the type of `out`). A bias is a vector of
    n values of the result's type. `out` shares no memory with an operand or the bias."""
    epilogue = Epilogue(epilogue)
    (m, k), (n, kb) = matrix(a, "a").shape, matrix(b, "b").shape
    if k != kb:
        raise ValueError(f"mx_matmul needs (m, k) @ (n, k) transposed, got {a.shape} and {b.shape}")
    element = out.dtype if isinstance(out, HIPTensor) else of(dtype)
    if element not in FLOATS:
        raise ValueError(f"an MX product is f16, bf16 or f32, not {element}")
    if out is not None and tensor(out, "out", 2, FLOATS).shape != (m, n):
        raise ValueError(f"out has shape {out.shape}, the product {(m, n)}")
    ops = []
    if epilogue.has_bias:
        if bias is None or tensor(bias, "bias", 1, FLOATS).shape != (n,) or bias.dtype != element:
            raise ValueError(f"{epilogue.value} needs a bias vector of {n} {element} values")
        ops.append((library.ADD_COL + library.VECTOR_KINDS[element], 0.0, bias.pointer))
    activation = epilogue.value.removeprefix("bias_")
    if activation in library.ACTIVATIONS:
        ops.append((library.ACTIVATIONS[activation], 0.0, 0))
    result = out if out is not None else a.device.empty(element, m, n)
    need = library.mx_gemm_workspace(m, n, k)
    call = library.mx_gemm_call(a.pointers, b.pointers, result.pointer, element, m, n, k, ops, need)

    def run(stream: HIPStream) -> None:
        if need:
            stream.with_workspace("mx_matmul", need, call)
        else:
            call(0, stream.handle)

    return Work("mx_matmul", a.device, result, (a, b, bias, result), run)

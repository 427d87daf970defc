"""A mixture-of-experts layer for the few tokens of a decoding step, its experts' weights in microscaled 4 bits. No
counterpart in the reference, whose library has the one product (src/krn/lib/lib.py:76-79 `Op`)."""

from krn_amd.dtypes import BF16, F16
from krn_amd.lib.calls import LibraryCall, Work, tensor
from krn_amd.lib.lib_mx import matrix
from krn_amd.runtime import library


@LibraryCall
def moe(x, router, gate_up, down, *, top_k: int, out=None) -> Work:
    """y_t = sum over the `top_k` experts e of token t of w_te * down_e (silu(gate_e x_t) * up_e x_t).

    x is (tokens, hidden) of f16 or bf16, at most 64 tokens, and `router` (experts, hidden) of the same type. A token's
    experts are those with the largest x_t . router_e, ties going to the lower index and NaN counting as the largest; w_t is
    the softmax of those logits. `gate_up` is the MxMatrix of experts * 2 * inner rows of hidden values, for every expert
    its inner gate rows and then its inner up rows; `down` the one of experts * hidden rows of inner values. At most 1024
    experts and 16 of them for a token. Logits are float32 sums, so experts whose logits differ by less than such a sum's
    error may change places; the inner values are rounded to 2^-16, everything else is float32 up to the result, (tokens,
    hidden) of x's type, which shares no memory with the inputs."""
    tensor(x, "x", 2, (F16, BF16))
    tensor(router, "router", 2, (x.dtype,))
    (tokens, hidden), experts, inner = x.shape, router.shape[0], matrix(down, "down").shape[1]
    if router.shape != (experts, hidden):
        raise ValueError(f"router has shape {router.shape}, x {x.shape}: an expert's row is as long as a token")
    if matrix(gate_up, "gate_up").shape != (experts * 2 * inner, hidden) or down.shape != (experts * hidden, inner):
        raise ValueError(f"{experts} experts of {inner} inner values on {hidden} need gate_up {(experts * 2 * inner, hidden)} "
                         f"and down {(experts * hidden, inner)}, got {gate_up.shape} and {down.shape}")
    if not isinstance(top_k, int) or not 1 <= top_k <= experts:
        raise ValueError(f"top_k is between 1 and the {experts} experts, got {top_k!r}")
    if out is not None and tensor(out, "out", 2, (x.dtype,)).shape != x.shape:
        raise ValueError(f"out has shape {out.shape}, x {x.shape}")
    result = out if out is not None else x.device.empty(x.dtype, tokens, hidden)
    need = library.moe_workspace(x.dtype, tokens, hidden, inner, experts, top_k)
    call = library.moe_call(x.dtype, x.pointer, router.pointer, gate_up.pointers, down.pointers, result.pointer, tokens,
                            hidden, inner, experts, top_k, need)
    return Work("moe", x.device, result, (x, router, gate_up, down, result),
                lambda stream: stream.with_workspace("moe", need, call))

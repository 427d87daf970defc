"""Calls of the MX product and the expert layer that share things: threads on one stream and on several, two graphs and eager
calls over workspaces, and the smallest and largest sizes of the layer. Sums are exact, so results are compared bit for bit."""

import threading

import numpy as np
import pytest

from krn_amd.dtypes import BF16, F32
from krn_amd.lib import moe, mx_matmul
from krn_amd.runtime import library
from tests import moe_layers, mx_products
from tests.test_gpu_moe_exact import OnDevice
from tests.test_gpu_mx import to_device, values, words

pytestmark = pytest.mark.gpu

SPLIT = (40, 130, 8192)  # K in parts, through the workspace


def split_product(device, seed):
    """(left, right, exact result) of a product whose K is split."""
    m, n, k = SPLIT
    rng = np.random.default_rng(seed)
    a, b = mx_products.matrix(rng, m, k), mx_products.matrix(rng, n, k, mx_products.centred(k))
    return to_device(device, *a, k), to_device(device, *b, k), mx_products.values(a, k) @ mx_products.values(b, k).T


@pytest.mark.parametrize("streams", [1, 3])
def test_threads_that_call_at_once(device, streams):
    """Six threads, ten calls each of a split product and a layer, on one stream's workspace or on three: every result is the
    one of a call alone."""
    assert " parts" in library.mx_gemm_kernel(*SPLIT)
    products = [split_product(device, seed) for seed in range(6)]
    layer = OnDevice(device, moe_layers.Layer(np.random.default_rng(0), "bf16", 256, 96, 8))
    router = device.to_device(words(layer.layer.router, "bf16")[0], BF16)
    tokens = [device.to_device(words(layer.layer.tokens(np.random.default_rng(s), 6), "bf16")[0], BF16) for s in range(6)]
    alone = [moe(x, router, layer.gate_up, layer.down, top_k=3).to_host() for x in tokens]
    device.sync()
    on = [device.stream() for _ in range(streams)]
    outs = [[(device.empty(F32, *SPLIT[:2]), device.empty(BF16, 6, 256)) for _ in range(10)] for _ in range(6)]
    device.sync()
    failed = []

    def work(t):
        try:
            with on[t % streams]:
                for product, y in outs[t]:
                    mx_matmul(*products[t][:2], out=product)
                    moe(tokens[t], router, layer.gate_up, layer.down, top_k=3, out=y)
        except BaseException as error:
            failed.append(error)

    threads = [threading.Thread(target=work, args=(t,)) for t in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for stream in on:
        stream.sync()
    for t in range(6):
        for product, y in outs[t]:
            np.testing.assert_array_equal(product.to_host(), products[t][2])
            np.testing.assert_array_equal(y.to_host(), alone[t])


def test_split_products_in_two_graphs_and_between_their_replays(device):
    """Graphs hold workspaces of their own: replays on two streams at once, with eager calls between, give each its result."""
    (a, b, first), (c, d, second), (e, f, third) = (split_product(device, seed) for seed in range(3))
    outs = [device.empty(F32, *SPLIT[:2]) for _ in range(3)]
    one = device.graph(mx_matmul.bind(a, b, out=outs[0]))
    two = device.graph(mx_matmul.bind(c, d, out=outs[1]))
    eager = mx_matmul.bind(e, f, out=outs[2])
    streams = [device.stream() for _ in range(2)]
    device.sync()
    for _ in range(4):
        for out in outs:
            out.copy_from(np.zeros(SPLIT[:2], np.float32))
        with streams[0]:
            one()
        with streams[1]:
            two()
            eager()
        for stream in streams:
            stream.sync()
        for out, want in zip(outs, (first, second, third)):
            np.testing.assert_array_equal(out.to_host(), want)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", [(1, 1, 1, 1, 1), (2, 1, 3, 2, 2), (5, 3, 1, 4, 1), (64, 7, 5, 3, 2),
                                                                (64, 32, 32, 1024, 16), (2, 33, 65, 1024, 1), (64, 65, 33, 16, 16)])
def test_the_layers_smallest_and_largest_numbers(device, kind, tokens, hidden, inner, experts, top_k):
    rng = np.random.default_rng(hidden + inner)
    layer = OnDevice(device, moe_layers.Layer(rng, kind, hidden, inner, experts))
    x = layer.layer.tokens(rng, tokens)
    layer.layer.assert_exact(x)
    layer.check(layer(x, top_k), x, top_k)


def test_a_result_given_back_by_every_form_of_the_call(device):
    a, b, want = split_product(device, 5)
    assert (mx_matmul(a, b, dtype=F32).to_host() == want).all()
    bound = mx_matmul.bind(a, b, dtype=F32)
    bound.submit().wait()
    np.testing.assert_array_equal(bound.result.to_host(), want)
    out = device.empty(F32, *SPLIT[:2])
    mx_matmul.submit(a, b, out=out).wait()
    np.testing.assert_array_equal(values(out), want)

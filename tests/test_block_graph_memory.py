"""CPU tests of the memory that plans with attention take."""
import re

import pytest

from ferrograd_amd.graph import (CROSS_ENTROPY, MEAN_SQUARED_ERROR, Graph, Metadata, Optim,
                                 SimpleDType, f32_bits)

T, C, HEADS, STARTS = 4096, 256, 4, 5


def arena(layers, trained, loss):
    """Bytes of a plan of attention layers over one another's output, keys and values (or
    only values) inputs without a gradient."""
    g, meta = Graph(loss, Optim.sgd().lower), Metadata.new()
    t, c, n = (meta.new_field() for _ in range(3))
    with g.define_ops() as ops:
        starts = ops.input([n], SimpleDType.U32)
        x = ops.input([t, c])
        for _ in range(layers):
            k, v = (ops.input([t, c], requires_grad=name in trained) for name in "kv")
            x = ops.attention(x, k, v, starts, HEADS, scale=0.125)
        if loss is CROSS_ENTROPY:
            ops.softmax(x)
    return int(re.search(r"arena: (\d+) bytes",
                         g.describe([f32_bits(1e-3), T, C, STARTS])).group(1))


@pytest.mark.parametrize("loss", [MEAN_SQUARED_ERROR, CROSS_ENTROPY])
@pytest.mark.parametrize("trained", ["", "k", "v", "kv"])
def test_gradients_that_nobody_reads_take_no_memory_of_their_own(loss, trained):
    """A layer more costs its output and log-sums, and the gradients that there are: of the
    output and of the trained operands."""
    sizes = [arena(n, trained, loss) for n in (2, 3, 4)]
    tensor = T * C * 4
    layer = (2 + len(trained)) * tensor + T * HEADS * 4
    # (A plan's tensors start at offsets of their own, less than 128 KiB apart each.)
    slack = 6 * (128 << 10)
    assert layer <= sizes[1] - sizes[0] <= layer + slack
    assert layer <= sizes[2] - sizes[1] <= layer + slack
    if len(trained) < 2:  # what the call writes of the others is there once
        once = (2 - len(trained)) * tensor
        assert abs(arena(2, trained, loss) + once - arena(2, "kv", loss)) <= slack

"""Every form of tiles that linear's tensor-core kernel may take, whatever the
rule that chooses them prefers: columns, two CTAs a tile, k divided by a
cluster, results in pieces and value by value."""
import pytest
import torch

import gateddeltanet_b200 as gdn
import layer_plain as plain
from test_gpu_layer_ops import BF16, F32, operands, padded, rand

pytestmark = pytest.mark.gpu
FORMS = [(1, 1), (1, 2), (1, 4), (1, 8), (2, 1)]  # CTAs to a tile, CTAs that divide k
INPUTS = {False: 2072, True: 4112}  # 33 blocks of k: uneven parts


@pytest.fixture(scope="module")
def ops():
    from gateddeltanet_b200 import build
    build.build()
    from gateddeltanet_b200 import ops
    return ops


def tiles(ctas, columns, split):
    assert gdn.lib().gdn_b200_test_linear_tiles(ctas, columns, split) == 0


@pytest.mark.parametrize("columns", range(32, 257, 32))
@pytest.mark.parametrize("ctas,split", FORMS)
@pytest.mark.parametrize("eight", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("activation", [None, "swiglu"])
def test_tiles(ops, columns, ctas, split, eight, activation):
    tokens = 300 if ctas == 2 else 100
    for outputs in (132, 131):  # in pieces of four, value by value
        rows = outputs * (2 if activation else 1)
        a = operands(tokens, INPUTS[eight], rows, eight)
        bias, residual = rand(rows, seed=3), rand(tokens, outputs, seed=4)
        for r in (None, residual):
            want, off = plain.linear(**a, bias=bias, activation=activation, residual=r)
            for dtype in (F32, BF16):
                out, big = padded(torch.zeros(tokens, outputs, device="cuda", dtype=dtype), 3, 4)
                tiles(ctas, columns, split)
                plain.check(ops.linear(**a, bias=bias, activation=activation, residual=r, out=out), want, off, str((outputs, dtype)))
                assert bool((big[tokens:] == 7).all()) and bool((big[:, outputs:] == 7).all())


@pytest.mark.parametrize("columns", [32, 64, 96, 224, 256])
@pytest.mark.parametrize("ctas", [1, 2])
def test_more_tiles_than_run_at_once(ops, columns, ctas):
    a = operands(1500, 200, 3000, False)
    want, off = plain.linear(**a)
    tiles(ctas, columns, 1)
    plain.check(ops.linear(**a, dtype=F32), want, off)


@pytest.mark.parametrize("tokens", [1, 9, 16])
def test_tiles_of_a_few_tokens(ops, tokens):
    a = operands(tokens, 2072, 132, False)
    want, off = plain.linear(**a)
    for split in (1, 4):
        tiles(1, 64, split)
        plain.check(ops.linear(**a, dtype=F32), want, off)


@pytest.mark.parametrize("ctas,columns,split", [(1, 16, 1), (1, 48, 1), (1, 288, 1), (0, 64, 1), (3, 64, 1), (2, 64, 1), (1, 64, 3), (1, 64, 16), (1, 64, 0),
                                                (1, 64, 8)])
def test_impossible_tiles_are_refused(ops, ctas, columns, split):
    """100 tokens are too few for two CTAs, 16 blocks of k too few for eight parts; the next call is as ever."""
    a = operands(100, 1024, 132, False)
    want = ops.linear(**a, dtype=F32)
    tiles(ctas, columns, split)
    with pytest.raises(RuntimeError, match="launch failed"):
        ops.linear(**a, dtype=F32)
    assert torch.equal(ops.linear(**a, dtype=F32), want)

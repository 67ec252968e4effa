"""The layer operators take outputs that lie between the runs of their other
tensors, heads between heads too, and refuse what shares a byte with one
(no GPU needed)."""
import random

import pytest

import gateddeltanet_b200 as gdn
from test_layer_ops_cpu import FAKE, FAR, linear_args, norm_args
from test_ops_cpu import lib  # noqa: F401


@pytest.mark.parametrize("change", [
    # three or four tensors of heads side by side: x, out, the gate and the residual in turn
    dict(x_head=192, x_token=768, out=FAKE + 128, out_head=192, out_token=768, gate=FAKE + 256, gate_head=192, gate_token=768),
    dict(x_head=192, x_token=768, out=FAKE, out_head=192, out_token=768, gate=FAKE + 128, gate_head=192, gate_token=768),
    dict(x_head=128, x_token=512, out_head=128, out_token=512, residual=FAKE + 128, residual_head=128, residual_token=512, residual_dtype=1),
    # tokens between the tokens of heads that are further apart
    dict(x_token=128, x_head=640, out=FAKE + 128, out_token=128, out_head=640),
    # other numbers of bytes a value, the same bytes from run to run
    dict(x_head=192, x_token=768, out=FAKE + 128, out_dtype=0, out_head=96, out_token=384)], ids=str)
def test_heads_between_heads_are_taken(lib, change):  # noqa: F811
    assert lib.gdn_b200_rms_norm(norm_args(**change)) == -1
    assert "device" in gdn.last_error()  # refused for the device alone


@pytest.mark.parametrize("change", [
    dict(x_head=192, x_token=768, out=FAKE + 126, out_head=192, out_token=768), dict(x_head=192, x_token=768, out=FAKE + 258, out_head=192, out_token=768),
    dict(x_head=192, x_token=768, out=FAKE + 128, out_head=160, out_token=768), dict(x_head=192, x_token=768, out=FAKE + 128, out_head=192, out_token=832),
    dict(x_head=192, x_token=768, out=FAKE + 132, out_dtype=0, out_head=192, out_token=768)], ids=str)
def test_what_is_not_quite_between_is_refused(lib, change):  # noqa: F811
    assert lib.gdn_b200_rms_norm(norm_args(**change)) == -1
    assert "overlap" in gdn.last_error()


def bytes_of(at, token, head, tokens, heads, dim, size):
    return {at + (t * token + h * head + i) * size + b for t in range(tokens) for h in range(heads) for i in range(dim) for b in range(size)}


def test_no_shared_byte_is_taken(lib):  # noqa: F811
    """Random small tensors near one another, against their sets of bytes."""
    rng = random.Random(1)
    taken = 0
    for _ in range(20000):
        tokens, heads, dim = rng.randint(1, 3), rng.randint(1, 3), rng.randint(1, 3)
        unit = rng.randint(1, 12)
        stride = lambda: rng.choice((dim, unit * rng.randint(1, 4), rng.randint(0, 20)))  # noqa: E731
        x_token, x_head, out_token, out_head = (stride() for _ in range(4))
        if rng.random() < 0.5:
            out_token, out_head = x_token, x_head
        at = FAKE + 2 * rng.randint(-12, 12)
        rc = lib.gdn_b200_rms_norm(norm_args(tokens=tokens, heads=heads, dim=dim, x_token=x_token, x_head=x_head, out=at, out_token=out_token,
                                             out_head=out_head))
        assert rc == -1
        x, out = bytes_of(FAKE, x_token, x_head, tokens, heads, dim, 2), bytes_of(at, out_token, out_head, tokens, heads, dim, 2)
        in_place = at == FAKE and (tokens == 1 or x_token == out_token) and (heads == 1 or x_head == out_head)
        if "device" in gdn.last_error():
            taken += 1
            assert in_place or not x & out
            assert len(out) == 2 * tokens * heads * dim
    assert taken > 4000


def test_projections_between_rows(lib):  # noqa: F811
    """The result in the gap between the rows of weight, which are as far apart and more."""
    fit = dict(weight=FAR, weight_row=256, out=FAR + 128, out_row=256, outputs=50)
    assert lib.gdn_b200_linear(linear_args(**fit)) == -1 and "device" in gdn.last_error()
    assert lib.gdn_b200_linear(linear_args(**{**fit, "outputs": 100}, out_dtype=0)) == -1 and "overlaps" in gdn.last_error()
    assert lib.gdn_b200_linear(linear_args(**{**fit, "out": FAR + 126})) == -1 and "overlaps" in gdn.last_error()

"""The serving operators (gateddeltanet_b200/ops.py) where they were once
wrong, unsafe or unseen; tolerances are those of test_gpu_ops_delta.py and
test_gpu_ops_logits.py unless a test derives its own."""
import pytest
import torch

import ops_plain as plain
from test_gpu_ops_delta import STATE_TOL, compare, inputs, out_tol

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from gateddeltanet_b200 import build
    build.build()
    from gateddeltanet_b200 import ops
    return ops


@pytest.mark.parametrize("rule", ["delta_step", "delta_chunk"])
@pytest.mark.parametrize("starts", [[10, 3, 5], [4, 8, 0, 0], [5, 8, 3, 2], [0, 5, 9, 0, 0], [70, 0]], ids=str)
@pytest.mark.parametrize("pad", [0, 200])
def test_decreasing_starts_end(ops, rule, starts, pad):
    """They give no particular values, but the call ends and touches nothing outside its tensors; with 200 empty
    sequences more, delta_step's pipeline has them."""
    starts = starts[:1] * pad + starts
    a, o = inputs([70] + [0] * (len(starts) - 2), 8, 8, 128, 128, torch.bfloat16, seed=40)
    o["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    wide = torch.full((90, 8, 128), 7.0, device="cuda", dtype=torch.bfloat16)
    state = torch.full((a["state"].shape[0] + 2, 8, 128, 128), 7.0, device="cuda")
    state[1:-1] = a["state"]
    getattr(ops, rule)(**{**a, "state": state[1:-1]}, **o, out=wide[10:80])
    torch.cuda.synchronize()
    assert bool((wide[:10] == 7).all()) and bool((wide[80:] == 7).all())
    assert bool((state[0] == 7).all()) and bool((state[-1] == 7).all())

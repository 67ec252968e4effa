"""The example server (examples/serve.py): prompt, new tokens and constraints
together as they would be used."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def serve():
    from gateddeltanet_b200 import build
    build.build()
    spec = importlib.util.spec_from_file_location("serve", os.path.join(REPO, "examples", "serve.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_generation_under_constraints(serve):
    model = serve.Model(vocab=1003, hidden=256, layers=2, heads=2, head_dim=64, seed=3)
    gen = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 1003, (n,), generator=gen).tolist() for n in (1, 70, 33, 200)]
    allowed = [set(range(0, 1003, 7)), set(range(1003)), {5, 6}, set(range(900, 1003))]
    masks = torch.zeros(4, (1003 + 31) // 32, dtype=torch.int64)
    for i, ids in enumerate(allowed):
        for v in ids:
            masks[i, v // 32] |= 1 << (v % 32)
    masks = torch.where(masks >= 2 ** 31, masks - 2 ** 32, masks).int().cuda()
    table, lens, states = serve.generate(model, prompts, 12, masks=masks, bias={5: -100.0})
    table, lens = table.tolist(), lens.tolist()
    for i, p in enumerate(prompts):
        assert lens[i] == len(p) + 12 and table[i][:len(p)] == p
        assert set(table[i][len(p):lens[i]]) <= allowed[i]
    assert set(table[2][33:45]) == {6}  # 5 is biased away
    assert all(bool(s.isfinite().all()) for s in states)
    # the same tokens as one prompt lead to the same states: the last pick has not been fed
    fed = [t[:n - 1] for t, n in zip(table, lens)]
    again = serve.generate(model, fed, 1)[2]
    for a, b in zip(states, again):
        # BF16 activations between the layers: the rounding of one changes by the order of a sum
        assert float((a - b).norm() / b.norm()) < 2e-2


def test_command(serve, capsys, monkeypatch):
    monkeypatch.setattr("sys.argv", ["serve.py", "--streams", "3", "--layers", "1", "--new", "4"])
    serve.main()
    assert "3 streams" in capsys.readouterr().out

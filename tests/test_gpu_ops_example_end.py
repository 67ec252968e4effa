"""The example server (examples/serve.py) where a stream cannot go on."""
import pytest
import torch

from test_gpu_ops_example import serve  # noqa: F401

pytestmark = pytest.mark.gpu


def test_a_stream_that_may_say_nothing_ends(serve):  # noqa: F811
    """Its length and its states stay, no token is fed for it, and the others go on as without it."""
    model = serve.Model(vocab=1003, hidden=256, layers=2, heads=2, head_dim=64, seed=3)
    gen = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, 1003, (n,), generator=gen).tolist() for n in (5, 70, 33)]
    masks = torch.full((3, 32), -1, dtype=torch.int32, device="cuda")
    masks[1] = 0
    table, lens, states = serve.generate(model, prompts, 6, masks=masks)
    assert lens.tolist() == [11, 70, 39] and table[1, :70].tolist() == prompts[1]
    assert bool((table >= 0).all()) and bool((table[1, 70:] == 0).all())
    only = serve.generate(model, prompts, 1, masks=masks)[2]  # the prompts alone: a last pick is not fed
    for s, t in zip(states, only):
        assert torch.equal(s[1], t[1]) and not torch.equal(s[0], t[0])
    masks[1] = -1
    free = serve.generate(model, prompts, 6, masks=masks)[0]
    assert torch.equal(free[0], table[0]) and torch.equal(free[2], table[2])


def test_empty_prompts_are_refused(serve):  # noqa: F811
    model = serve.Model(vocab=1003, hidden=256, layers=1, heads=1, head_dim=64, seed=3)
    for prompts in ([], [[1, 2], []]):
        with pytest.raises(ValueError, match="prompt"):
            serve.generate(model, prompts, 2)

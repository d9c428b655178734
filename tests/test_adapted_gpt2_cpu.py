"""Options of the GPT-2-shaped command with adapters that are refused before a device is looked for."""

import pytest

from aihwkit_b200 import gpt2_inference as G


def test_adaptation_of_several_ranks_is_refused(monkeypatch):
    """Each rank would train a model of its own."""
    import torch.distributed as dist

    monkeypatch.setenv("WORLD_SIZE", "2")
    with pytest.raises(SystemExit, match="one process"):
        G.main(["--adapters", "2", "--adapt-steps", "1"])
    monkeypatch.setattr(dist, "is_initialized", lambda: True)
    monkeypatch.setattr(dist, "get_world_size", lambda group=None: 2)
    with pytest.raises(RuntimeError, match="one process"):
        G.adapt(None, None, 2, 1)


@pytest.mark.parametrize("world", [1, 2, 4, 8])
@pytest.mark.parametrize("adapters", [1, 3, 4, 16])
def test_sequences_use_the_adapters_in_turn_over_all_ranks(world, adapters):
    local = 16 // world
    got = [int(i) for rank in range(world) for i in G.sequence_adapters(rank * local, local, adapters, "cpu")]
    assert got == [j % adapters for j in range(16)]


def test_adaptation_without_a_next_token_is_refused():
    """The mean over no tokens is not a number, and a step on it would leave none of the weights one."""
    import torch

    with pytest.raises(SystemExit, match="two tokens"):
        G.main(["--adapters", "2", "--adapt-steps", "1", "--seq", "1"])
    with pytest.raises(RuntimeError, match="two tokens"):
        G.adapt(None, torch.zeros(2, 1, dtype=torch.long), 2, 1)

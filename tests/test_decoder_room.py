"""What the decoder example refuses on the host, before any launch: tokens past
a cache's room or the model's positions, lengths and batches that do not fit.
On the CPU a call that is not refused here fails at its first operator instead."""

import pytest
import torch

from forma_b200.api import TensorError
from forma_b200.decoder import Decoder, DecoderConfig, Prompt

CFG = DecoderConfig(vocab=50, embed=64, heads=2, kv_heads=1, layers=2, mlp=64, window=8, sinks=2, positions=40)


@pytest.fixture
def dec():
    return Decoder(CFG, "cpu")


def started(dec, length, sequences, room):
    rows = min(length, CFG.sinks + CFG.window - 1)
    layer = tuple(torch.zeros(1, rows, CFG.head_dim, dtype=torch.bfloat16) for _ in range(2))
    return dec.start(Prompt(length, [layer] * CFG.layers), sequences, room)


def tokens(g, n):
    return torch.zeros(g, n, dtype=torch.int32)


def refused(state, call):
    before, longest = state.lengths, state.lengths.tolist()
    with pytest.raises(ValueError):
        call()
    assert state.lengths is before and state.lengths.tolist() == longest


def accepted(call):
    with pytest.raises(TensorError):  # past the checks: the first operator has no device memory
        call()


def test_room(dec):
    state = started(dec, 5, 3, 10)
    refused(state, lambda: dec.extend(state, tokens(3, 11)))
    refused(state, lambda: dec.generate(state, tokens(3, 1)[:, 0], 11))
    refused(state, lambda: dec.score(state, tokens(3, 11), tokens(3, 11)))
    accepted(lambda: dec.extend(started(dec, 5, 3, 10), tokens(3, 10)))
    longest = state.require(3, 7, CFG.positions)
    state.advance(7, longest)
    refused(state, lambda: dec.extend(state, tokens(3, 4)))
    refused(state, lambda: dec.generate(state, tokens(3, 1)[:, 0], 4))
    assert state.require(3, 3, CFG.positions) == 7
    state.advance(3, 7)
    refused(state, lambda: dec.extend(state, tokens(3, 1)))


def test_lengths_from_outside(dec):
    """Set back, replaced or written in place: read again; beyond the room: refused."""
    state = started(dec, 5, 2, 10)
    state.advance(10, state.require(2, 10, CFG.positions))
    state.lengths = torch.tensor([9, 2], dtype=torch.int32)
    assert state.require(2, 1, CFG.positions) == 9
    refused(state, lambda: dec.extend(state, tokens(2, 2)))
    state.lengths[0] = 3
    assert state.require(2, 7, CFG.positions) == 3
    refused(state, lambda: dec.extend(state, tokens(2, 8)))
    state.lengths.fill_(11)
    refused(state, lambda: dec.extend(state, tokens(2, 0)))
    state.lengths = torch.tensor([-1, 2], dtype=torch.int32)
    refused(state, lambda: dec.extend(state, tokens(2, 1)))


def test_positions_and_batch(dec):
    state = started(dec, 30, 2, 20)
    refused(state, lambda: dec.extend(state, tokens(2, 11)))
    accepted(lambda: dec.extend(started(dec, 30, 2, 20), tokens(2, 10)))
    one = started(dec, 5, 1, 10)
    refused(one, lambda: dec.extend(one, tokens(3, 1)))
    with pytest.raises(ValueError):
        dec.read(torch.zeros(41, dtype=torch.int32))
    accepted(lambda: dec.read(torch.zeros(40, dtype=torch.int32)))


def test_no_steps(dec):
    state = started(dec, 5, 3, 10)
    chosen, scores = dec.generate(state, tokens(3, 1)[:, 0], 0)
    assert chosen.shape == scores.shape == (3, 0)
    assert chosen.dtype == torch.int32 and scores.dtype == torch.float32
    assert state.lengths.tolist() == [0, 0, 0]

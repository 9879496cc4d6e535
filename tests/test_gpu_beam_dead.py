"""Beams without a score (-inf, NaN) in ``beam_select``: their candidates are all equal, so the lowest tokens come first."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_beams import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_all_beams_dead(lngram, dtype):
    g = torch.Generator(device="cuda").manual_seed(0)
    logits = torch.randn(2, 3, 700, generator=g, device="cuda").to(dtype)
    scores, tokens, parents = lngram.beam_select(logits, torch.full((2, 3), -math.inf, device="cuda"), width=5)
    assert (scores == -math.inf).all() and (parents == 0).all() and tokens.tolist() == [[0, 1, 2, 3, 4]] * 2


def test_a_dead_beam_beside_one_of_few_tokens(lngram):
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn(1, 2, 5000, generator=g, device="cuda")
    logits[0, 1] = -math.inf
    logits[0, 1, 1234] = 0
    scores, tokens, parents = lngram.beam_select(logits, torch.tensor([[-math.inf, -2.0]], device="cuda"), width=4)
    assert scores.tolist() == [[-2.0] + [-math.inf] * 3]
    assert tokens.tolist() == [[1234, 0, 1, 2]] and parents.tolist() == [[1, 0, 0, 0]]


def test_an_ended_dead_beam_offers_no_eos(lngram):
    logits = torch.zeros(2, 2, 40, device="cuda")
    done = torch.tensor([[True, False], [True, True]], device="cuda")
    scores, tokens, parents = lngram.beam_select(logits, torch.full((2, 2), -math.inf, device="cuda"), width=3, done=done, eos=7)
    assert (scores == -math.inf).all() and tokens.tolist() == [[0, 1, 2]] * 2 and (parents == 0).all()


def test_a_score_of_nan_counts_as_none(lngram):
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = torch.randn(1, 3, 90, generator=g, device="cuda")
    for done in (None, torch.tensor([[True, False, False]], device="cuda")):
        got = lngram.beam_select(logits, torch.tensor([[math.nan, -math.inf, math.nan]], device="cuda"), width=4, done=done,
                                 eos=None if done is None else 5)
        assert (got[0] == -math.inf).all() and got[1].tolist() == [[0, 1, 2, 3]] and (got[2] == 0).all()


@pytest.mark.parametrize("vocab, width", [(3, 6), (40, 8), (700, 32), (20011, 9)])
def test_masked_vocabularies_and_dead_and_ended_beams(lngram, vocab, width):
    """Fewer finite candidates than the width, in every mixture."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = torch.randn(60, 4, vocab, generator=g, device="cuda") * 3
    allowed = torch.rand(60, 4, vocab, generator=g, device="cuda") < 1.5 / vocab
    logits = torch.where(allowed, logits, -math.inf)
    logits[::3] = torch.randn(20, 4, vocab, generator=g, device="cuda")
    scores = -torch.rand(60, 4, generator=g, device="cuda") * 6
    scores[torch.rand(60, 4, generator=g, device="cuda") < 0.6] = -math.inf
    done = torch.rand(60, 4, generator=g, device="cuda") < 0.3
    check(lngram, logits, scores, width)
    check(lngram, logits, scores, width, done, vocab // 2)

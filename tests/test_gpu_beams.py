"""Beam search's operators on the GPU against plain implementations in 64 bits.

Scores: log of the sum from fp32 sums of fast exponentials, each within 2^-21 of (1 + |x - max|) relative; joined and
ranked in 64 bits, rounded to fp32 once: 2^-21 (1 + 30) + 2^-24 |score| is a bound, for logits within 30 of the largest
where it counts.  Tokens and parents are equal, ties included; random cases leave no two of the best candidates closer
than their bound without being checked for it.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(logits, scores, width, done=None, eos=None):
    c = torch.log_softmax(logits.double(), -1)
    c = torch.where(c.isnan().any(-1, keepdim=True), -math.inf, c)
    c = scores.double()[..., None] + c
    if done is not None:
        ended = torch.full_like(c, -math.inf)
        ended[..., eos] = scores.double()
        c = torch.where(done[..., None], ended, c)
    values, order = torch.sort(c.flatten(1), descending=True, stable=True)
    vocab = logits.shape[2]
    return values, order // vocab, order % vocab, width


def check(lngram, logits, scores, width=None, done=None, eos=None, close=True):
    width = logits.shape[1] if width is None else width
    got, tokens, parents = lngram.beam_select(logits, scores, width=width, done=done, eos=eos)
    values, beam, token, _ = reference(logits, scores, width, done, eos)
    want = values[:, :width]
    tol = 2.0 ** -21 * 31 + 2.0 ** -24 * want.abs().nan_to_num(posinf=0, neginf=0)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine) and (got[~fine] == -math.inf).all()
    assert ((got.double() - want).abs()[fine] <= tol[fine]).all()
    same = (tokens == token[:, :width]) & (parents == beam[:, :width])
    if not same.all():
        # only candidates that lie within the bound of one another may have changed places
        assert close
        flat = parents * logits.shape[2] + tokens
        for g, k in (~same).nonzero().tolist():
            place = (beam[g] * logits.shape[2] + token[g] == flat[g, k]).nonzero()[0, 0]
            assert (values[g, place] - values[g, k]).abs() <= 2 * tol[g, k]
    assert got.dtype == torch.float32 and tokens.dtype == torch.int64 and parents.dtype == torch.int64


DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("groups, beams, vocab, width", [
    (1, 1, 1, 1), (1, 1, 5, 4), (3, 2, 7, 3), (1, 4, 32000, 4), (2, 1, 32000, 8), (5, 3, 999, 3), (2, 32, 4097, 32), (17, 8, 12345, 8),
    (64, 5, 257, 5), (1, 2, 160001, 16), (2, 32, 1, 32), (300, 4, 100, 4),
])
def test_select(lngram, dtype, groups, beams, vocab, width):
    g = torch.Generator(device="cuda").manual_seed(vocab + beams)
    logits = (torch.randn(groups, beams, vocab, generator=g, device="cuda") * 3).to(DT[dtype])
    scores = -torch.rand(groups, beams, generator=g, device="cuda") * 8 - 3
    check(lngram, logits, scores, width)


@pytest.mark.parametrize("vocab", [6, 1000, 33333])
def test_ties_go_to_the_lowest(lngram, vocab):
    """Logits of few values, and beams that are the same: the order of equal candidates is that of their index."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    row = torch.randint(0, 3, (4, 1, vocab), generator=g, device="cuda").to(torch.bfloat16)
    check(lngram, row.expand(4, 5, vocab).contiguous(), torch.zeros(4, 5, device="cuda"), 9, close=False)
    check(lngram, torch.zeros(2, 3, vocab, device="cuda"), torch.zeros(2, 3, device="cuda"), 7, close=False)
    same = torch.full((2, 3, vocab), 1.5, device="cuda", dtype=torch.float16)
    check(lngram, same, torch.tensor([[-1.0, -3.0, -1.0], [0.0, 0.0, 0.0]], device="cuda"), 12, close=False)


def test_rising_and_falling_logits(lngram):
    """The longest chains of replacements: every value is larger than all before it, or smaller."""
    up = torch.arange(50000, device="cuda", dtype=torch.float32)[None, None] * 1e-3
    for x in (up, up.flip(2), torch.cat((up, up.flip(2)), 1).contiguous()):
        check(lngram, x, torch.zeros(x.shape[:2], device="cuda"), 32)


def test_ended_beams(lngram):
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn(6, 4, 5000, generator=g, device="cuda")
    scores = -torch.rand(6, 4, generator=g, device="cuda") * 6
    done = torch.tensor([[0, 0, 0, 0], [1, 0, 0, 0], [0, 1, 1, 0], [1, 1, 1, 1], [1, 1, 1, 0], [0, 0, 0, 1]], device="cuda").bool()
    for eos in (0, 2, 4999):
        check(lngram, logits, scores, 4, done, eos)
        check(lngram, logits, scores, 9, done, eos)  # beyond what ended beams offer: -inf, by index
    check(lngram, logits[..., :3].contiguous(), scores, 11, done, 1)


def test_masked_and_bad_rows(lngram):
    """-inf where the vocabulary is masked, rows with nothing left, NaN and +inf: such rows offer -inf, the others theirs."""
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = torch.randn(4, 3, 3000, generator=g, device="cuda")
    logits[0, :, 5:] = -math.inf
    logits[1, 0] = -math.inf
    logits[1, 1, 77] = math.nan
    logits[2, 2, 2999] = math.inf
    logits[3] = -math.inf
    logits[3, 1, 10] = 0
    scores = torch.zeros(4, 3, device="cuda")
    check(lngram, logits, scores, 3)
    check(lngram, logits, scores, 32)
    lowest = torch.randn(1, 2, 4000, generator=g, device="cuda").half()
    lowest[0, 0, 1:] = torch.finfo(torch.float16).min
    check(lngram, lowest, torch.zeros(1, 2, device="cuda"), 6)
    check(lngram, logits, torch.tensor([-math.inf, 0.0, -1.0], device="cuda").expand(4, 3).contiguous(), 5)


def test_strided_rows(lngram):
    """Logits in a padded vocabulary, beginning at odd addresses."""
    g = torch.Generator(device="cuda").manual_seed(3)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn(3, 4, 10007, generator=g, device="cuda").to(dtype)
        check(lngram, wide[..., 3:9002], torch.zeros(3, 4, device="cuda"))


@pytest.mark.parametrize("groups, beams", [(1, 1), (3, 4), (2, 5), (4, 8), (1, 16), (5, 32)])
@pytest.mark.parametrize("shape, dtype", [((7,), torch.uint8), ((33, 5), torch.uint8), ((40, 64), torch.bfloat16), ((3, 3, 3), torch.float32),
                                          ((), torch.int64), ((129, 1), torch.float16), ((0, 4), torch.float32)])
def test_reorder(lngram, groups, beams, shape, dtype):
    g = torch.Generator(device="cuda").manual_seed(beams)
    x = torch.randint(0, 100, (groups * beams, *shape), generator=g, device="cuda").to(dtype)
    parents = torch.randint(0, beams, (groups, beams), generator=g, device="cuda")
    rows = (parents + torch.arange(groups, device="cuda")[:, None] * beams).flatten()
    want = x[rows]
    lngram.beam_reorder(parents, x)
    assert torch.equal(x, want)


def test_reorder_states_together_within_a_length(lngram):
    g = torch.Generator(device="cuda").manual_seed(4)
    parents = torch.tensor([[1, 0, 1], [2, 2, 2]], device="cuda")
    rows = torch.tensor([1, 0, 1, 5, 5, 5], device="cuda")
    states = [torch.randint(0, 9, (6, 50, 3), generator=g, device="cuda", dtype=torch.uint8),
              torch.randn(6, 50, 16, generator=g, device="cuda"), torch.randn(6, 50, generator=g, device="cuda").half(),
              torch.randn(6, 3, 50, 8, generator=g, device="cuda")[:, 1]] * 1
    states += [torch.randn(6, 50, 2, generator=g, device="cuda") for _ in range(7)]  # more than a launch takes
    old = [x.clone() for x in states]
    lngram.beam_reorder(parents, *states, length=37)
    for x, o in zip(states, old):
        assert torch.equal(x[:, :37], o[rows][:, :37]) and torch.equal(x[:, 37:], o[:, 37:])
    lngram.beam_reorder(parents, *states, length=0)
    lngram.beam_reorder(parents)


def test_reorder_of_parents_out_of_range(lngram):
    err = lngram._lib.device_error
    err()
    x = torch.arange(12.0, device="cuda").view(4, 3)
    lngram.beam_reorder(torch.tensor([[1, -1, 4, 0]], device="cuda"), x)
    assert err() == 4
    assert x.tolist() == [[3, 4, 5], [3, 4, 5], [6, 7, 8], [0, 1, 2]]


def test_captured_on_two_streams(lngram):
    """Two captured graphs with workspaces of their own, replayed side by side."""
    g = torch.Generator(device="cuda").manual_seed(5)
    inputs = [(torch.randn(8, 4, 30000, generator=g, device="cuda"), -torch.rand(8, 4, generator=g, device="cuda")) for _ in range(2)]
    want = [lngram.beam_select(*x) for x in inputs]
    streams, graphs, outs = [torch.cuda.Stream() for _ in inputs], [], []
    for x, s in zip(inputs, streams):
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(lngram.beam_select(*x))
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for got, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(got, w))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_rows_of_the_lowest_and_largest_values(lngram, dtype):
    """A mask of the type's lowest value over a whole row leaves equal candidates, one over all but a few leaves those;
    logits of the largest values do not overflow."""
    info = torch.finfo(DT[dtype])
    g = torch.Generator(device="cuda").manual_seed(6)
    logits = torch.randn(3, 2, 3001, generator=g, device="cuda").to(DT[dtype])
    logits[0, 0] = info.min
    logits[1, 0, 7:] = info.min
    logits[2, 1] = info.max
    logits[2, 0, 3] = info.max
    check(lngram, logits, torch.zeros(3, 2, device="cuda"), 5)

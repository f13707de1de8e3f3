"""Beam selection against the definition in 64 bits.

Tolerances: a chosen score is rounded to fp32 once (2^-24 of its value); before that
its denominator's log is off by the exponentials' relative error: 2^-22 (ex2), 2^-24
|t| (the rounding of t = (x - top) log2 e, of which 2^t |t| <= 0.54 is felt), and the
sums', which keep what their additions lose: below 6e-7 in all.  Parents and tokens
are equal: the inputs leave candidates of different beams further apart than that
(checked), those of one beam are compared by their logits alone."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from oracle import decoding as od

STEP = 2.0 ** -24


def compare(logits, scores, width, **kw):
    from voom_b200.runtime.beam import beam_select

    want, parents, tokens = od.beam_select(logits.cpu(), scores.cpu(), width)
    got = beam_select(logits, scores, width, **kw)
    assert got.scores.dtype == torch.float32 and got.parents.dtype == got.tokens.dtype == torch.int32
    assert got.scores.shape == got.parents.shape == got.tokens.shape == (logits.shape[0], width)
    assert torch.equal(got.parents.cpu(), parents)
    assert torch.equal(got.tokens.cpu(), tokens)
    s = got.scores.cpu().double()
    none = parents < 0
    assert bool((s[none] == -math.inf).all())
    err = (s[~none] - want[~none]).abs()
    assert err.numel() == 0 or bool((err <= 6e-7 + STEP * want[~none].abs()).all()), float(err.max())
    return got


def made(B, beams, V, dtype, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    logits = (spread * torch.randn((B, beams, V), generator=g)).to(dtype)
    return logits.cuda(), (-5.0 * torch.rand((B, beams), generator=g)).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,beams,V,width", [(1, 1, 1, 1), (1, 1, 7, 7), (1, 1, 7, 12), (2, 3, 33, 6), (1, 4, 1000, 8),
                                             (3, 5, 8191, 10), (2, 8, 8193, 16), (1, 2, 50001, 64), (40, 4, 4099, 5),
                                             (1, 64, 300, 64), (1, 33, 2000, 31), (130, 3, 515, 6), (1, 1, 200019, 2)])
def test_sizes_and_types(dtype, B, beams, V, width):
    compare(*made(B, beams, V, dtype), width)


@pytest.mark.gpu
def test_long_rows_of_one_block():
    """More rows than blocks at a time: a block reads a row alone and looks at its groups several times."""
    compare(*made(150, 4, 70001, torch.float32, 11), 8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift", [0, 1, 3, 7])
def test_rows_anywhere(dtype, shift):
    """Rows that start and end at any element, in a wider storage with NaN around them."""
    big = torch.full((2, 3, 5200), math.nan, dtype=dtype, device="cuda")
    x, s = made(2, 3, 4097, dtype, 5)
    big[:, :, shift:shift + 4097] = x
    compare(big[:, :, shift:shift + 4097], s, 6)
    compare(big.transpose(0, 1)[:, :, shift:shift + 4097], s.transpose(0, 1).contiguous(), 4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ties_go_to_the_lower_token(dtype):
    for V in (40, 3001, 50000):
        x = torch.zeros((1, 2, V), dtype=dtype, device="cuda")
        s = torch.tensor([[-1.0, -1.0]], device="cuda")  # the beams tie as well
        got = compare(x, s, 8)
        assert got.tokens.tolist() == [list(range(8))] and got.parents.tolist() == [[0] * 8]
        # coarse logits: many ties everywhere, the best ones late in the row
        x = torch.randint(-2, 3, (2, 3, V), generator=torch.Generator().manual_seed(V)).to(dtype).cuda()
        x[:, :, V - 3:] = 3.0
        compare(x, torch.tensor([[-1.0, -2.25, -1.5], [-3.0, -0.5, -0.25]], device="cuda"), 12)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [3, 32, 33, 64])
def test_adversarial_orders(width):
    """Rising rows (every value enters the lists), falling ones, and all the best in one lane's place."""
    V = 30000
    rise = torch.arange(V, dtype=torch.float32) / 1000
    lane = torch.zeros(V)
    lane[torch.arange(0, V, 256)] = torch.arange(0, V, 256) / 500.0
    x = torch.stack((rise, rise.flip(0), lane))[None].cuda()
    compare(x, torch.tensor([[-1.0, -1.3, -0.2]], device="cuda"), width)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_masked_tokens_and_beams(dtype):
    x, s = made(4, 4, 3001, dtype, 2)
    s[0, 1:] = -math.inf  # a first step
    s[1] = -math.inf      # an ended request
    x[2, 0, 5:] = -math.inf  # five tokens left
    x[2, 1:] = -math.inf     # none
    x[3, 0, 17] = math.nan   # rows without candidates
    x[3, 1, 18] = math.inf
    got = compare(x, s, 8)
    assert bool((got.parents[1] == -1).all()) and bool((got.parents[2, 5:] == -1).all())
    assert not bool(((got.parents[3] == 12) | (got.parents[3] == 13)).any())
    s[3, 2] = math.nan
    got = compare(x, s, 8)
    assert bool((got.parents[3] == 15).all())
    x[:] = -math.inf
    assert bool((compare(x, s, 3).tokens == -1).all())
    low = torch.finfo(dtype).min  # masks of the type's lowest value: a value like others
    x, s = made(1, 2, 600, dtype, 3)
    x[:, 0, 2:] = low
    x[:, 1] = low
    compare(x, s, 5)


@pytest.mark.gpu
def test_peaked_and_shifted_rows():
    """One token takes nearly all; rows far from zero; a long flat row's sum."""
    x, s = made(2, 3, 20000, torch.float32, 4)
    x[0, 0, 777] = 60.0
    x[0, 1] += 1000.0
    x[0, 2] -= 30000.0
    x[1, 0] = 1e-3 * torch.randn(20000, generator=torch.Generator().manual_seed(6)).cuda()
    compare(x, s, 9)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 600])
def test_long_rising_rows(rows):
    """Rows that rise all along: a maximum that is raised a thousand times costs the sum nothing.  The terms' error
    is 2^-22 (ex2) and 2^-25 (its argument); a group's 16 are added in eight steps of 2^-24 at most, one after
    another; beyond, sums keep what they lose: 2^-22 + 2^-25 + 8 * 2^-24 < 7.5e-7."""
    from voom_b200.runtime.beam import beam_select

    V = 1 << 22
    for rise in (4.0, 40.0, 4000.0):
        row = (torch.arange(V, dtype=torch.float64) * (rise / V)).to(torch.float32).cuda()
        x = row.expand(rows, 1, V)  # as many rows as make a block read each by itself
        got = beam_select(x, torch.zeros((rows, 1), device="cuda"), 5)
        want = row[-1].double() - torch.logsumexp(row.double(), 0)
        top = torch.sort(row, descending=True, stable=True)[1][:5]
        assert torch.equal(got.tokens, top.to(torch.int32).expand(rows, 5)), rise
        err = (got.scores[:, 0].double() - want).abs().max()
        assert float(err) <= 7.5e-7 + STEP * abs(float(want)), (rise, float(err))


@pytest.mark.gpu
def test_rows_of_values_past_two_to_the_twenty():
    """Logits so large that fp32 holds no part of an exponent, at either end, and a row that is one value alone."""
    for shift in (3e5, 1e7, -1e7, 1e30, -1e30):
        x, s = made(2, 3, 5003, torch.float32, 16)
        x[0, 1] = x[0, 1] * 4 + shift
        x[1, 0] = shift
        x[1, 2, 100:] = -torch.finfo(torch.float32).max
        compare(x, s, 6)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,V", [(torch.float16, 50257), (torch.bfloat16, 50257), (torch.float32, 9001), (torch.float16, 200019)])
@pytest.mark.parametrize("beams,width", [(8, 8), (3, 7)])
def test_equal_beams_go_by_beam(dtype, V, beams, width):
    """Beams with the same logits and the same score tie token by token, wherever in 16 bytes their rows start."""
    x, _ = made(2, 1, V, dtype, 12)
    x = x.expand(2, beams, V).contiguous()
    got = compare(x, torch.full((2, beams), -1.5, device="cuda"), width)
    best = x[:, 0].float().argmax(1)
    assert got.parents[:, :min(beams, width)].tolist() == [[b * beams + i for i in range(min(beams, width))] for b in range(2)]
    assert got.tokens[:, :min(beams, width)].tolist() == [[int(t)] * min(beams, width) for t in best]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,V", [(torch.float16, 50257), (torch.float32, 30011)])
def test_candidates_a_few_2_to_the_minus_24_apart(dtype, V):
    """Scores are compared in 64 bits: equal rows whose scores are one fp32 step apart, and rows whose sums
    differ by 1e-8 of themselves."""
    beams = 7
    x, _ = made(3, 1, V, dtype, 13)
    x = x.expand(3, beams, V).contiguous()
    for b in range(3):
        top = x[b, 0].float().amax()
        for i in range(beams):  # of a sum of at least 1: e^-18 = 1.5e-8 for each step
            x[b, i, 17] = (top - 17 - (i * 3 + b) % beams).to(dtype)
    order = [3, 0, 6, 2, 5, 1, 4]
    s = torch.tensor([[0.5 + k * 2.0 ** -24 for k in order]], device="cuda").expand(3, beams).contiguous()
    s[1] = 0.5
    compare(x, s, 9)


@pytest.mark.gpu
def test_more_candidates_than_are_put_in_order_by_counting():
    """64 equal beams, 64 wanted: every beam's best tie."""
    x, _ = made(2, 1, 300, torch.float32, 14)
    compare(x.expand(2, 64, 300).contiguous(), torch.full((2, 64), -0.75, device="cuda"), 64)
    x, s = made(2, 64, 300, torch.float32, 15, spread=0.01)
    compare(x, s * 1e-3, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows", [4, 592])
def test_vocabularies_masked_with_the_lowest_value(dtype, rows):
    """Fewer tokens allowed than wanted, the others at the type's lowest value: a tie as long as the row."""
    from voom_b200.runtime.beam import beam_select

    V, width = 128000, 16
    r = torch.Generator().manual_seed(3)
    row = torch.full((V,), torch.finfo(dtype).min, dtype=dtype)
    allowed = torch.randperm(V, generator=r)[:5]
    row[allowed] = torch.randn(5, generator=r).to(dtype)
    want, parents, tokens = od.beam_select(row[None, None], torch.zeros((1, 1)), width)
    got = beam_select(row.cuda().expand(rows, 1, V), torch.zeros((rows, 1), device="cuda"), width)
    assert torch.equal(got.tokens.cpu(), tokens.expand(rows, width))
    err = (got.scores.cpu().double() - want).abs() - STEP * want.abs()
    assert bool((err <= 6e-7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("width", [1, 17, 64])
def test_best_values_under_one_thread(width):
    """More of a row's best than a block holds lie 256 apart: the last resort, one after another."""
    from voom_b200.runtime.beam import beam_select

    V = 400000
    row = torch.zeros(V, dtype=torch.float32)
    at = torch.arange(5, V, 256)
    row[at] = 1.0 + torch.arange(at.numel()).float() / 2048
    x = torch.stack((row, row.flip(0)))[:, None].contiguous().cuda()
    compare(x, torch.full((2, 1), -0.5, device="cuda"), width)
    big = row.cuda().expand(600, 1, V)  # a block to each row
    got = beam_select(big, torch.zeros((600, 1), device="cuda"), width)
    want = at.flip(0)[:width].to(torch.int32)
    assert torch.equal(got.tokens.cpu(), want.expand(600, width))


@pytest.mark.gpu
def test_streams_graphs_and_repeats():
    from voom_b200.runtime.beam import beam_select

    x, s = made(3, 4, 9001, torch.bfloat16, 7)
    first = compare(x, s, 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = beam_select(x, s, 8, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = beam_select(x, s, 8)
        other = beam_select(x[:1], s[:1], 3)
    y, t = made(3, 4, 9001, torch.bfloat16, 8)
    x.copy_(y)
    s.copy_(t)
    graph.replay()
    torch.cuda.synchronize()
    want = beam_select(y, t, 8)
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert all(torch.equal(a, b[:1, :3]) for a, b in zip(other, want))
    assert beam_select(x[:0], s[:0], 4).scores.shape == (0, 4)


@pytest.mark.gpu
def test_refusals():
    from voom_b200.runtime.beam import beam_select

    x, s = made(2, 3, 100, torch.float32)
    for bad in (x[0], x.double(), x.transpose(1, 2), x[:, :, ::2]):
        with pytest.raises(ValueError, match="logits"):
            beam_select(bad, s, 2)
    for bad in (s[0], s.cpu(), s.double(), s.half(), torch.zeros((3, 2), device="cuda").T, s[:, :2]):
        with pytest.raises(ValueError, match="scores"):
            beam_select(x, bad, 2)
    for width in (0, -1, 65):
        with pytest.raises(ValueError, match="continuations"):
            beam_select(x, s, width)
    with pytest.raises(ValueError, match="continuations"):
        beam_select(torch.zeros((1, 65, 8), device="cuda"), torch.zeros((1, 65), device="cuda"), 2)
    with pytest.raises(ValueError, match="continuations"):
        beam_select(x[:, :, :0], s, 2)


@pytest.mark.gpu
def test_sizes_past_the_limits_are_refused_in_words():
    from voom_b200.runtime.beam import beam_select

    x = torch.zeros((1, 1, 1), dtype=torch.bfloat16, device="cuda")
    for shape in ((2 ** 27, 1, 1), (2 ** 21, 64, 1)):
        y = x.expand(shape)
        with pytest.raises(ValueError, match="2\\^31|2\\^27"):
            beam_select(y, torch.zeros((1, 1), device="cuda").expand(shape[:2]).contiguous(), 1)


def test_refusals_without_a_device(built_lib):
    from voom_b200._lib import VOOM_E_CAPACITY, VOOM_E_INVALID_ARG, VOOM_E_UNSUPPORTED, BeamSelectArgs
    from voom_b200.runtime.beam import beam_select

    with pytest.raises(ValueError, match="CUDA"):
        beam_select(torch.zeros((1, 2, 8)), torch.zeros((1, 2)), 2)

    def call(scratch=1 << 28, **kw):
        a = BeamSelectArgs()
        a.logits, a.scores, a.scores_out, a.parents, a.tokens = (1 << x for x in range(20, 25))
        a.l_b, a.l_i, a.B, a.beams, a.V, a.width, a.type = 400, 100, 2, 4, 100, 8, 0
        for x, y in kw.items():
            setattr(a, x, y)
        return built_lib.voom_beam_select(ctypes.byref(a), scratch, 0, None)

    assert call() == VOOM_E_CAPACITY and call(B=0) == 0
    for bad in (dict(logits=None), dict(scores=None), dict(tokens=None), dict(beams=0), dict(V=0), dict(width=0), dict(type=3),
                dict(logits=(1 << 20) + 1), dict(scratch=8), dict(scratch=None)):
        assert call(**bad) == VOOM_E_INVALID_ARG, bad
    for bad in (dict(beams=65), dict(width=65), dict(V=1 << 30)):
        assert call(**bad) == VOOM_E_UNSUPPORTED, bad
    assert built_lib.voom_beam_select(None, 1 << 28, 0, None) == VOOM_E_INVALID_ARG

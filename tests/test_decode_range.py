"""Linear attention of large and small states, values and keys whose decays span more than 32-bit
numbers do, against the definition in 64 bits.

With e = 2^-24, relative to the same sums of absolute values, as tests/test_decode_ops.py derives
them: (8 + 6 sqrt(2 L + dk)) e.  A factor is a mantissa and a power of two, whose product with a
number rounds once more than a factor's: 1 e for each token at most, which the sum's 2 L
independent roundings (two per token: a decay's product and the addition) have room for, since a
token's decay is one factor.  Nothing that is checked here is below 2^-100, where digits end.
"""
import math

import pytest
import torch

from test_decode_ops import EPS, _close, _linear64, _linear_run
from test_decode_ops import ctx, om  # noqa: F401  (fixtures)

SHAPES = [(2, 128, 128), (2, 33, 47), (1, 256, 72), (2, 64, 64), (3, 96, 80)]
BIG = 2.0 ** 100


def _burst(g, L, H, at, width, log2):
    """No decays but for `width` tokens from `at` on, whose factors' product is 2^-log2."""
    d = torch.zeros(L, H)
    x = 0.5 + torch.rand(width, H, generator=g)
    d[at:at + width] = -log2 * math.log(2) * x / x.sum(0)
    return d


def _check(om, ctx, lens, H, dk, dv, q, k, v, decay, S, steps=False, complement=False):
    B = len(lens)
    starts = [sum(lens[:i]) for i in range(B + 1)]
    want, bound, ends, eb = _linear64(q, k, v, decay, starts, S, dk ** -0.5, complement)
    c = (8 + 6 * math.sqrt(2 * max(lens) + dk)) * EPS
    o, S1 = _linear_run(om, ctx, lens, H, q.shape[1], k.shape[1], v.shape[1], dk, dv, q, k, v, decay, S,
                        list(range(B)), list(range(B)), steps=steps, in_place=True, complement=complement)
    _close(o, want, bound * c)
    _close(S1, ends, eb * c)


def _inputs(lens, H, dk, dv, seed):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens)
    q, k, v = (torch.randn(T, H, d, generator=g) for d in (dk, dk, dv))
    return g, q, k * dk ** -0.5, v, torch.randn(len(lens), H, dk, dv, generator=g)


@pytest.mark.gpu
@pytest.mark.parametrize("log2", [100, 130, 180])
@pytest.mark.parametrize("L,at,width", [(20, 3, 1), (20, 3, 12), (70, 20, 30), (200, 5, 64), (200, 64, 1),
                                        (600, 130, 64), (1500, 700, 400)])
@pytest.mark.parametrize("H,dk,dv", SHAPES)
def test_large_states_that_decay(om, ctx, H, dk, dv, L, at, width, log2):
    """A state of 2^100, and what a burst of decays leaves of it beside the tokens behind."""
    lens = [L, 40]
    g, q, k, v, S = _inputs(lens, H, dk, dv, L + log2)
    decay = torch.cat([_burst(g, L, H, at, width, log2), _burst(g, 40, H, 7, 3, log2)])
    _check(om, ctx, lens, H, dk, dv, q, k, v * (BIG * 2.0 ** -log2), decay, S * BIG)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["v", "k", "both"])
@pytest.mark.parametrize("L,at,width", [(20, 3, 1), (70, 20, 30), (70, 31, 2), (600, 130, 64), (1500, 700, 300)])
@pytest.mark.parametrize("H,dk,dv", SHAPES)
def test_large_tokens_that_decay(om, ctx, H, dk, dv, L, at, width, which):
    """Tokens of 2^100 before a burst of decays, of about what is left of them behind it."""
    lens = [L, 40]
    g, q, k, v, S = _inputs(lens, H, dk, dv, L + at)
    decay = torch.cat([_burst(g, L, H, at, width, 140), _burst(g, 40, H, 7, 3, 140)])
    behind = torch.cat([torch.arange(L) >= at, torch.arange(40) >= 7])[:, None, None]
    size = torch.where(behind, 2.0 ** -40, BIG)
    if which != "v":
        k = k * (size if which == "k" else size.sqrt())
    if which != "k":
        v = v * (size if which == "v" else size.sqrt())
    _check(om, ctx, lens, H, dk, dv, q, k, v, decay, S)


@pytest.mark.gpu
@pytest.mark.parametrize("H,dk,dv", SHAPES + [(2, 200, 130), (64, 64, 64)])
def test_single_tokens_of_large_states(om, ctx, H, dk, dv):
    """A token's own decay below the least normal number, and below the least of all."""
    for log2 in (100, 126, 140, 149, 152, 190):
        lens = [1] * 8
        g, q, k, v, S = _inputs(lens, H, dk, dv, log2)
        decay = torch.full((8, H), -log2 * math.log(2))
        for complement in (False, True):
            _check(om, ctx, lens, H, dk, dv, q, k, v * (BIG * 2.0 ** -log2), decay, S * BIG, steps=True,
                   complement=complement)


@pytest.mark.gpu
@pytest.mark.parametrize("H,dk,dv", SHAPES)
def test_states_that_grow_and_decay(om, ctx, H, dk, dv):
    """Decays above 0 and below in one chunk, whose sum hides how far its parts reach.  A burst
    takes a state of 1 to 2^80, 2^-50 and 2^-5; factors' products reach 2^125 (45 + 80 behind a
    token right before a burst's last decay), so tokens are of 2^-60."""
    lens = [90, 33]
    g, q, k, v, S = _inputs(lens, H, dk, dv, 5)
    decay = torch.zeros(sum(lens), H)
    for t0, n in ((0, 90), (90, 33)):
        for at in (4, 12, 20, 28, 60):
            if at + 8 <= n:
                decay[t0 + at:t0 + at + 4] = 20 * math.log(2)
                decay[t0 + at + 4] = -130 * math.log(2)
                decay[t0 + at + 6] = 45 * math.log(2)
    _check(om, ctx, lens, H, dk, dv, q, k, v * 2.0 ** -60, decay, S)


@pytest.mark.gpu
@pytest.mark.parametrize("H,dk,dv", SHAPES)
def test_large_states_beside_what_is_not_finite(om, ctx, H, dk, dv):
    """The same where a token's infinity and NaN have the sequence done with other instructions."""
    lens, at = [70, 40], 35
    g, q, k, v, S = _inputs(lens, H, dk, dv, 6)
    decay = torch.cat([_burst(g, 70, H, 20, 30, 140), _burst(g, 40, H, 7, 3, 140)])
    v, S = v * (BIG * 2.0 ** -140), S * BIG
    want, bound, ends, eb = _linear64(q, k, v, decay, [0, 70, 110], S, dk ** -0.5, False)
    v[at, 0, 3], v[at + 1, 0, 5] = math.inf, math.nan
    o, S1 = _linear_run(om, ctx, lens, H, H, H, H, dk, dv, q, k, v, decay, S, [0, 1], [0, 1], in_place=True)
    bad = torch.zeros(o.shape, dtype=torch.bool)
    bad[at:70, 0, 3] = bad[at + 1:70, 0, 5] = True
    assert not torch.isfinite(o[bad]).any()
    c = (8 + 6 * math.sqrt(140 + dk)) * EPS
    _close(o[~bad], want[~bad], bound[~bad] * c)
    S1[0, 0][:, [3, 5]] = ends[0, 0][:, [3, 5]] = 0.0
    _close(S1, ends, eb * c)


@pytest.mark.gpu
@pytest.mark.parametrize("H,dk,dv", SHAPES)
def test_strong_decays_of_ordinary_values(om, ctx, H, dk, dv):
    """Every chunk's decays span more than numbers do, of values that need no second pass."""
    lens = [333, 40]
    g, q, k, v, S = _inputs(lens, H, dk, dv, 7)
    _check(om, ctx, lens, H, dk, dv, q, k, v, -40 * torch.rand(373, H, generator=g), S)
    _check(om, ctx, lens, H, dk, dv, q, k, v * 2.0 ** 30, -8 * torch.rand(373, H, generator=g), S * 2.0 ** 30)

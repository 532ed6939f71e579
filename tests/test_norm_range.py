"""Norms of heads (gpu_norm_rope_axes, gpu_norm_kv_append) whose squares pass what 32 bits hold,
against the definition in 64 bits.

The bound is that of tests/test_decode_ops.py, (D / 64 + 16) / 2 + 6 of e = 2^-24: such a row's sum is
one of the row times a power of two, which rounds nothing but squares that are less than 2^-100 of
the sum.  Results below the least normal number are off by half its last step, 2^-150, more.
"""
import math

import pytest
import torch

from test_decode_ops import EPS, _close, _down, _norm64, _rope64, _up
from test_decode_ops import ctx, om  # noqa: F401  (fixtures)


def _rows(T, H, D, seed, eps0):
    """Ordinary rows between those of large and (without eps) of small numbers."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, D, generator=g)
    sizes = [1.0, 2.0 ** 63, 2.0 ** 64, 2.0 ** 90, 2.0 ** 125] + [2.0 ** -52, 2.0 ** -64, 2.0 ** -100, 2.0 ** -126, 2.0 ** -140] * eps0
    for t in range(T):
        for h in range(H):
            x[t, h] *= sizes[(t * H + h) % len(sizes)]
            if (t + h) % 7 == 3:
                x[t, h, 1:] *= 2.0 ** -40  # one number far above the others
    return x.clamp(-torch.finfo(torch.float32).max, torch.finfo(torch.float32).max)


CASES = [  # T, heads, kv, D, pairs, halves
    (20, 3, 2, 128, [16, 24, 24], True), (20, 2, 1, 256, [32], False), (11, 5, 5, 64, [], True),
    (13, 2, 2, 33, [16], True), (13, 3, 1, 66, [33], True), (11, 1, 1, 1000, [64], False),
    (9, 2, 1, 4, [2], False), (11, 2, 1, 4096, [100, 156], True), (11, 1, 2, 7, [2], False)]


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,kv,D,pairs,halves", CASES)
@pytest.mark.parametrize("kind", ["rms", "l2"])
@pytest.mark.parametrize("eps", [0.0, 1e-6, 1e38])
def test_norms_of_large_and_small_rows(om, ctx, T, H, kv, D, pairs, halves, kind, eps):
    q, k = _rows(T, H, D, D, eps == 0.0), _rows(T, kv, D, D + 1, eps == 0.0)
    g = torch.Generator().manual_seed(1)
    w = 1.0 + 0.5 * torch.randn(1, D, generator=g)
    pos = torch.randint(0, 100000, (len(pairs) or 1, T), generator=g, dtype=torch.int32)
    qb, kb, wb, pb = _up(ctx, q, k, w, pos)
    qo, ko = ctx.alloc(q.numel() * 4), ctx.alloc(k.numel() * 4)
    rope = om.rope_axes(pairs, 1e4, halves=halves) if pairs else None
    om.norm_rope_axes(ctx, qo, ko, qb, kb, T, H, kv, D, om.head_norm(kind, eps, wb), pb if pairs else None, rope)
    tol = (D / 64 + 16) / 2 + 6
    for out, x, weight in ((qo, q, w), (ko, k, None)):
        want, bound = _rope64(_norm64(x, weight, kind, float(torch.tensor(eps))), pairs, 1e4, halves, pos, tol)
        _close(_down(ctx, out, x.shape), want, bound + 4 * 2.0 ** -150 * D)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 33])
def test_norm_append_of_large_rows(om, ctx, D):
    """Into the cache; values, which have no norm, as they are."""
    T, H, kv, page = 18, 2, 2, 8
    q, k = _rows(T, H, D, 5, True), _rows(T, kv, D, 6, True)
    v = _rows(T, kv, D, 7, True)
    slots = torch.randperm(24, generator=torch.Generator().manual_seed(2))[:T].to(torch.int32)
    pool = torch.zeros(3, kv, page, D)
    qb, kb, vb, sb, kp, vp = _up(ctx, q, k, v, slots, pool, pool)
    qo = ctx.alloc(q.numel() * 4)
    om.norm_kv_append(ctx, om.kv_pages(kp, vp, "f32", 3, page, kv, D), kb, vb, T, sb, qo, qb, H, om.head_norm("rms", 0.0))
    tol = ((D / 64 + 16) / 2 + 6) * EPS
    for got, x in ((_down(ctx, qo, q.shape), q),
                   (_down(ctx, kp, pool.shape).permute(0, 2, 1, 3).reshape(24, kv, D)[slots.long()], k)):
        want = _norm64(x, None, "rms", 0.0)
        _close(got, want, want.abs() * tol + 2.0 ** -148)
    assert torch.equal(_down(ctx, vp, pool.shape).permute(0, 2, 1, 3).reshape(24, kv, D)[slots.long()], v)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 33])
def test_norms_of_rows_that_are_not_finite(om, ctx, D):
    """An infinity among numbers: they become 0, it is NaN; zeros without eps are NaN, with it 0."""
    x = torch.randn(4, 1, D, generator=torch.Generator().manual_seed(3)) * 2.0 ** 80
    x[0, 0, 3], x[1, 0, 3], x[2] = math.inf, math.nan, 0.0
    xb = _up(ctx, x)[0]
    for eps in (0.0, 1e-6):
        out = ctx.alloc(x.numel() * 4)
        om.norm_rope_axes(ctx, out, None, xb, None, 4, 1, 0, D, om.head_norm("l2", eps))
        got = _down(ctx, out, x.shape)[:, 0]
        rest = [i for i in range(D) if i != 3]
        assert (got[0, rest] == 0).all() and torch.isnan(got[0, 3]) and torch.isnan(got[1]).all()
        assert torch.isnan(got[2]).all() if eps == 0 else (got[2] == 0).all()
        want = _norm64(x[3], None, "l2", eps)
        _close(got[3:], want, want.abs() * ((D / 64 + 16) / 2 + 6) * EPS)

"""Linear attention and sampling at the sizes that choose the kernels' other instances: many
heads and sequences, wide heads, cut and whole; rows of the largest vocabularies in slices of
every length.

CPU: which instance a size chooses, by the kernels' own host side.
GPU: against the definition in 64 bits, as tests/test_decode_ops.py, whose bounds hold here:
  linear  the bound there counts roundings by the longest sequence and the key's dimensions,
          whatever instance does them.
  sample  with 2^-b the step of a weight (b = 51, less where n tokens' sum would pass 62 bits:
          42 at 2^20), each is off by half a step, a sum by n 2^-(b + 1), and where two sums are
          compared (a border, a share of one) by twice that: n 2^-b of the largest weight.
"""
import math
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import test_decode_ops as ops
from test_decode_ops import EPS, REQUESTS, _check_linear, _close, _linear64, _linear_inputs, _linear_run, _sample
from test_decode_ops import ctx, om  # noqa: F401  (fixtures)

HERE = os.path.dirname(os.path.abspath(__file__))


def _short(n, *first):
    """n lengths up to 100, some of them 0, behind those given."""
    return list(first) + [(37 * b) % 101 for b in range(n - len(first))]


# name: what the launches' kernels are, the sequences' lengths (0: single tokens, that many),
# heads, key and value dimensions
LINEAR = {
    "steps of a batch": (["step 4 32"], 64, 8, 128, 128),
    "steps, two rounds of rows": (["step 4 32"], 65, 8, 256, 64),
    "steps, a last vector within a group": (["step 4 32"], 130, 4, 136, 132),
    "steps of odd columns, two rounds": (["step 1 32"], 3, 2, 200, 130),
    "steps of few heads, two rounds": (["step 4 8"], 2, 3, 250, 36),
    "two blocks, whole": (["chunks 8 2 1 0"], _short(130), 2, 128, 128),
    "two blocks, parts that join by themselves": (["chunks 8 2 1 1", "chunks 8 2 1 0"], _short(64, 300, 256, 65), 2, 128, 128),
    "two blocks, parts joined by a launch": (["chunks 8 2 1 1", "join", "chunks 8 2 1 0"], _short(16, 1500, 500), 1, 128, 128),
    "two blocks, columns past the last": (["chunks 8 2 1 0"], _short(130), 2, 96, 200),
    "two blocks, odd rows, whole": (["chunks 8 2 0 0"], _short(130), 2, 99, 131),
    "two blocks, odd rows, joined": (["chunks 8 2 0 1", "join", "chunks 8 2 0 0"], _short(16, 1500, 400), 1, 127, 70),
    "two blocks of few dimensions": (["chunks 4 2 1 0"], _short(130), 2, 64, 128),
    "two blocks of few dimensions, odd": (["chunks 4 2 0 0"], _short(130), 2, 50, 131),
    "two blocks of few dimensions, odd, joined": (["chunks 4 2 0 1", "join", "chunks 4 2 0 0"], _short(16, 1500, 200), 1, 33, 67),
    "one block, odd": (["chunks 8 1 0 1", "chunks 8 1 0 0"], [150, 3, 97], 2, 99, 47),
    "one block, odd, joined": (["chunks 8 1 0 1", "join", "chunks 8 1 0 0"], [1000], 1, 97, 33),
    "wide keys, joined": (["chunks 16 1 1 1", "join", "chunks 16 1 1 0"], [1100, 64], 1, 256, 72),
    "wide keys, odd, joined": (["chunks 16 1 0 1", "join", "chunks 16 1 0 0"], [700], 1, 253, 65),
    "wide keys, whole": (["chunks 16 1 1 0"], _short(130), 4, 132, 24),
}


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    """Each call's launches as (kernel, x, y, z, bytes of the workspace)."""
    hipcc = "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    root = os.path.dirname(HERE)
    d = tmp_path_factory.mktemp("grids")
    flags = ["-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I" + os.path.join(root, "include")]
    for f in ("linear", "sample"):
        subprocess.run([hipcc, "--offload-host-only", "-O1", "--offload-arch=gfx950", "-std=c++17", flags[2],
                        "-c", os.path.join(root, "ornith-flight_amd", "csrc", "kernels", f + ".hip"),
                        "-o", str(d / (f + ".o"))], check=True)
    subprocess.run(["gcc", "-std=gnu99", *flags, "-c", os.path.join(HERE, "decode_grids.c"), "-o", str(d / "main.o")],
                   check=True)
    subprocess.run(["g++", "-no-pie", "-Wl,--unresolved-symbols=ignore-all", "-o", str(d / "grids"),
                    *[str(d / (f + ".o")) for f in ("main", "linear", "sample")]], check=True)

    def run(cases):
        text = "\n".join(" ".join(map(str, c)) for c in cases)
        out = subprocess.run([str(d / "grids")], input=text, capture_output=True, text=True, check=True,
                             timeout=300).stdout.splitlines()
        assert len(out) == len(cases)
        calls = []
        for words in (line.split() for line in out):
            call = []
            for i in range(0, len(words), 5):
                m = re.search(r"k_(?:linear|sample)_([a-z]+)(?:I((?:L[ib]\d+E)+)E)?", words[i])
                call.append((" ".join([m.group(1)] + re.findall(r"L[ib](\d+)E", m.group(2) or "")),
                             *map(int, words[i + 1:i + 5])))
            calls.append(call)
        return calls
    return run


def test_the_instances_of_linear_attention(launches):
    cases = [("l", *((lens, H, dk, dv, 1) if isinstance(lens, int) else (len(lens), H, dk, dv, max(lens))))
             for _, lens, H, dk, dv in LINEAR.values()]
    for name, call in zip(LINEAR, launches(cases)):
        assert [k[0] for k in call] == LINEAR[name][0], name


def test_the_launches_fit(launches):
    """A dimension has fewer than 2^32 threads, and y and z at most 65535 groups; the work
    buffers stay within the parts of 512 groups."""
    cases = [("l", n, H, dk, dv, L) for n in (1, 7, 65535) for H in (1, 32, 65535)
             for dk, dv in ((1, 1), (128, 128), (256, 256)) for L in (0, 1, 2, 64, 8192, 0x7fff0000)]
    cases += [("s", rows, n, 0, 0, 0) for rows in (1, 63, 65535) for n in (1, 32768, 32769, 248320, (1 << 20) - 1, 1 << 20)]
    for c, call in zip(cases, launches(cases)):
        assert call, c
        for kernel, x, y, z, room in call:
            assert x >= 1 and x * 1024 < 1 << 32 and 1 <= y <= 65535 and 1 <= z <= 65535, (c, kernel)
            if c[0] == "l":
                assert room <= 512 * (c[3] * c[4] + 2) * 4 + 4096, c


def test_the_slices_of_rows(launches):
    """Their number, for slices of 4096 tokens and of more."""
    cases = {(4, 1 << 20): 4096, (4, (1 << 20) - 1): 4096, (4, 524289): 4096, (70, 200000): 10240, (64, 150001): 8192,
             (64, 248320): 12288, (128, 248320): 22528, (2, 32769): 4096}
    for ((_, n), length), call in zip(cases.items(), launches([("s", *c, 0, 0, 0) for c in cases])):
        assert call[0][1] == -(-n // length)


@pytest.mark.gpu
@pytest.mark.parametrize("gates,complement", [("token", False), ("strong", True)])
@pytest.mark.parametrize("name", list(LINEAR))
def test_linear_instances(om, ctx, name, gates, complement):
    _, lens, H, dk, dv = LINEAR[name]
    steps = isinstance(lens, int)
    _check_linear(om, ctx, [1] * lens if steps else lens, H, 1, H, H, dk, dv, gates, complement,
                  seed=len(name), steps=steps)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["two blocks, whole", "two blocks, parts that join by themselves",
                                  "two blocks, parts joined by a launch", "two blocks, odd rows, joined"])
def test_linear_instances_that_are_not_finite(om, ctx, name):
    """What is finite is right beside what is not, in place."""
    _, lens, H, dk, dv = LINEAR[name]
    B, b = len(lens), max(range(len(lens)), key=lambda i: lens[i])
    t0, t1 = sum(lens[:b]), sum(lens[:b + 1])
    g, q, k, v, decay = _linear_inputs(lens, H, 1, H, H, dk, dv, "token", 31)
    S = torch.randn(B, H, dk, dv, generator=g)
    want, bound, ends, eb = _linear64(q, k, v, decay, [sum(lens[:i]) for i in range(B + 1)], S, dk ** -0.5, False)
    c = (8 + 6 * math.sqrt(2 * max(lens) + dk)) * EPS
    at = t0 + lens[b] // 3
    v[at, 0, 3], v[at + 1, 0, dv - 1] = math.inf, math.nan
    o, S1 = _linear_run(om, ctx, lens, H, 1, H, H, dk, dv, q, k, v, decay, S, list(range(B)), list(range(B)), in_place=True)
    bad = torch.zeros(o.shape, dtype=torch.bool)
    bad[at:t1, 0, 3] = bad[at + 1:t1, 0, dv - 1] = True
    assert not torch.isfinite(o[bad]).any() and not torch.isfinite(S1[b, 0][:, [3, dv - 1]]).any()
    _close(o[~bad], want[~bad], bound[~bad] * c + 1e-37)
    S1[b, 0][:, [3, dv - 1]] = 0.0
    ends[b, 0][:, [3, dv - 1]] = 0.0
    _close(S1, ends, eb * c + 1e-37)


# ---------------------------------------- sampling
def _choices(order, x, temperature, top_k, top_p, min_p, u, off):
    """As test_decode_ops._choices, of a row whose order is known, sums off by `off`."""
    on = int((x > -np.inf).sum())
    if temperature == 0:
        return {int(order[0]): [1.0]}
    top = x[order[0]]
    w = np.exp((x[order[:on]] - top) / float(np.float32(temperature)))
    if 0 < top_k < on:
        w = w[:top_k]
    before = np.cumsum(w) - w
    found = {}
    for sign in (-1.0, 1.0):
        last = before < float(np.float32(top_p)) * w.sum() + sign * off
        last &= w >= float(np.float32(min_p)) * (1.0 - sign * 1e-15)
        last[0] = True
        kept = w[last]
        c = np.cumsum(kept)
        for s in (-1.0, 1.0):
            i = min(int(np.searchsorted(c, float(np.float32(u)) * c[-1] + s * off, side="right")), len(kept) - 1)
            found.setdefault(int(order[i]), []).append(kept[i] / c[-1])
    return found


def _check_rows(om, ctx, x, requests, u):
    n = x.shape[1]
    bits = 51
    while n > 1 << (62 - bits):
        bits -= 1
    t, p, err = _sample(om, ctx, x, requests, u)
    assert err is None
    several = 0
    for i, q in enumerate(requests):
        x64 = x[i].astype(np.float64)
        order = np.argsort(-x64, kind="stable")
        ok = _choices(order, x64, *q, u[i], n * 2.0 ** -bits)
        several += len(ok) > 1
        assert int(t[i]) in ok, (i, q, u[i], int(t[i]), ok)
        want = min(ok[int(t[i])], key=lambda w: abs(p[i] - w))
        # a share: its weight and the sum (at least the largest weight) each off, and a rounding
        assert abs(p[i] - want) <= want * (EPS + n * 2.0 ** -bits) + 2.0 ** -bits, (i, q, p[i], want)
    assert several <= len(requests) // 8


LARGE = [(1.0, 0, 0.95, 0.0), (0.7, 50, 0.8, 0.0), (1.2, 1000, 1.0, 0.0), (1.0, 6000, 0.9, 0.0), (0.0, 0, 1.0, 0.0),
         (1.0, 0, 1.0, 0.01), (2.0, 0, 1.0, 0.0), (0.8, 2048, 0.99, 0.001)]


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1 << 20, (1 << 20) - 1, 524289, 248320])
@pytest.mark.parametrize("what", ["spread", "equal", "grid", "tail", "flat"])
def test_sample_of_large_vocabularies(om, ctx, n, what):
    g = np.random.default_rng(n + len(what))
    x = g.standard_normal((len(LARGE), n)) * {"flat": 0.05}.get(what, 3.0)
    if what == "equal":
        x[:] = 1.25
    elif what == "grid":
        x = np.round(x * 4) / 4
    x = x.astype(np.float32)
    u = (g.random(len(x)) * 0.999).astype(np.float32)
    if what == "tail":  # nothing but the last 200
        x[:, :n - 200] = -np.inf
    elif what == "equal":
        u[0] = u[5] = u[6] = 1 - 2.0 ** -24
    _check_rows(om, ctx, x, LARGE, u)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(64, 150001), (64, 248320), (2, 32769)])
def test_sample_of_slices_of_other_lengths(om, ctx, rows, n):
    g = np.random.default_rng(rows)
    x = (g.standard_normal((rows, n), np.float32) * np.float32(2.5))
    x[1::5] = np.round(x[1::5] * 4) / 4
    x[2::5, : n - 300] = -np.inf
    requests = [(LARGE + REQUESTS)[i % (len(LARGE) + len(REQUESTS))] for i in range(rows)]
    _check_rows(om, ctx, x, requests, (g.random(rows) * 0.999).astype(np.float32))


@pytest.mark.gpu
def test_sample_greedily(om, ctx):
    """A batch of greedy rows in slices: the first of the largest, wherever it lies."""
    n = 200000
    x = np.random.default_rng(2).standard_normal((70, n)).astype(np.float32)
    at = [0, 1, 4095, 4096, 8191, n - 1, n - 2] * 10
    for i, a in enumerate(at):
        x[i, a] = 9.0
        x[i, a + (n - a) // 2:n:max(1, n // 50)] = 9.0
        x[i, a] = 9.0
    t, p, err = _sample(om, ctx, x, [(0.0, 3, 0.5, 0.5)] * 70, np.full(70, 0.5, np.float32))
    assert err is None and (p == 1.0).all()
    assert t.tolist() == [int(np.argmax(r)) for r in x]


@pytest.mark.gpu
def test_sample_special_rows_in_slices(om, ctx):
    """Rows in slices: infinities, NaN, nothing at all, requests that are refused, a stride."""
    n, stride = 40000, 40013
    g = np.random.default_rng(9)
    x = g.standard_normal((9, stride)).astype(np.float32)
    x[:, n:] = 80.0  # not the rows'
    x[0, :n], x[1, :n] = -np.inf, np.nan
    x[2, [17, 30000]] = np.inf
    x[3, :n] = -np.inf
    x[3, n - 1] = -1e38
    x[4, 1:n] = np.nan
    requests = [(1.0, 0, 0.9, 0.0)] * 5 + [(-1.0, 0, 0.9, 0.0), (0.0, 9, 1.5, 0.0), (1.0, 0, 0.9, 0.0), (0.7, 20, 0.8, 0.0)]
    u = np.array([0.6] * 7 + [1.0, 0.6], np.float32)
    rb, ub = ctx.upload(np.array(requests, om.SAMPLE_REQUEST)), ctx.upload(u)
    xb, tb, pb = ctx.upload(x), ctx.upload(np.full(10, 77, np.int32)), ctx.upload(np.full(10, 7.5, np.float32))
    with pytest.raises(RuntimeError, match="row"):
        om.sample(ctx, tb, pb, xb, 9, n, rb, ub, stride=stride)
    t, p = ctx.download(tb, np.int32, (10,)), ctx.download(pb, np.float32, (10,))
    assert t[:8].tolist() == [-1, -1, 30000, n - 1, 0, -1, -1, -1] and t[9] == 77
    assert p[:8].tolist() == [0, 0, 0.5, 1, 1, 0, 0, 0] and p[9] == 7.5
    x64 = x[8, :n].astype(np.float64)
    assert int(t[8]) in _choices(np.argsort(-x64, kind="stable"), x64, *requests[8], u[8], n * 2.0 ** -46)
    assert om.lib().gpu_kv_check(ctx.ptr) == 0


# ---------------------------------------- calls with one side only
@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[1] * 3, [40, 3, 0], [700, 1, 90]])
def test_linear_from_zeros_to_slots(om, ctx, lens):
    """No slots to start from, states left behind; and the other way round."""
    H, dk, dv = 2, 32, 48
    g, q, k, v, decay = _linear_inputs(lens, H, 1, 2, 1, dk, dv, "head", 4)
    S = torch.randn(4, H, dk, dv, generator=g)
    starts = [sum(lens[:i]) for i in range(4)]
    bufs = ops._up(ctx, q, k, v, decay)
    slots, tb = ops._up(ctx, torch.tensor([3, 0, 1], dtype=torch.int32), torch.tensor(starts, dtype=torch.int32))
    c = (8 + 6 * math.sqrt(2 * max(lens) + dk)) * EPS
    for ins, outs in ((None, slots), (slots, None)):
        sb, out = ops._up(ctx, S)[0], ctx.alloc(sum(lens) * H * dv * 4)
        om.linear_attend(ctx, om.linear_states(sb, 4, H, dk, dv), out, *bufs[:3], 1, 2, 1, sum(lens), bufs[3], 3,
                         None if max(lens) == 1 else tb, ins, outs, None)
        S0 = S[[3, 0, 1]] if ins else torch.zeros(3, H, dk, dv)
        want, bound, ends, eb = _linear64(q, k, v, decay, starts, S0, dk ** -0.5, False)
        _close(ops._down(ctx, out, want.shape), want, bound * c + 1e-37)
        got = ops._down(ctx, sb, S.shape)
        if outs:
            _close(got[[3, 0, 1]], ends, eb * c + 1e-37)
        assert torch.equal(got[2], S[2]) and (outs is not None or torch.equal(got, S))


@pytest.mark.gpu
@pytest.mark.parametrize("D,halves", [(128, True), (33, False)])
def test_norms_of_one_side(om, ctx, D, halves):
    """Keys alone, queries alone, and an append without queries."""
    T, kv, page = 9, 2, 8
    k = torch.randn(T, kv, D, generator=torch.Generator().manual_seed(D))
    want, tol = ops._norm64(k, None, "rms", 1e-6), (D / 64 + 16) * EPS
    kb, sb = ops._up(ctx, k, torch.arange(T, dtype=torch.int32) + 3)
    out = [ctx.alloc(k.numel() * 4) for _ in range(2)]
    om.norm_rope_axes(ctx, None, out[0], None, kb, T, 0, kv, D, om.head_norm("rms"))
    om.norm_rope_axes(ctx, out[1], None, kb, None, T, kv, 0, D, om.head_norm("rms"))
    for o in out:
        _close(ops._down(ctx, o, k.shape), want, want.abs() * tol)
    kp, vp = ops._up(ctx, torch.zeros(2, kv, page, D), torch.zeros(2, kv, page, D))
    om.norm_kv_append(ctx, om.kv_pages(kp, vp, "f32", 2, page, kv, D), kb, kb, T, sb, None, None, 0, om.head_norm("rms"))
    rows = [ops._down(ctx, b, (2, kv, page, D)).permute(0, 2, 1, 3).reshape(16, kv, D) for b in (kp, vp)]
    _close(rows[0][3:3 + T], want, want.abs() * tol)
    assert torch.equal(rows[1][3:3 + T], k) and (rows[0][:3] == 0).all() and (rows[0][3 + T:] == 0).all()

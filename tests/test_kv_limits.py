"""The paged key-value cache's calls where numbers end: values near the largest
of 32 bits, scales of the 8-bit type, sizes of a launch, bits of a product, a
workspace that grows.  Definitions and tolerances are those of test_kv_ops.py.
"""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest
import torch

from test_kv_ops import (DTYPE, HERE, Cache, Call, attend, attend64, ctx, host, i32, om, tables, value)  # noqa: F401


# ------------------------------------------------------------ values near the largest
def large_values(c, biggest, seed):
    """Every value of V between half of +-biggest and all of it, one sign per dimension."""
    g = torch.Generator().manual_seed(seed)
    sign = torch.where(torch.rand(c.v.shape[3], generator=g) < 0.5, -1.0, 1.0)
    x = (0.5 + 0.5 * torch.rand(c.v.shape, generator=g)) * sign * biggest
    c.v.copy_(x.to(c.v.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv,D,page,lens", [
    (8, 2, 64, 16, [700, 0, 3]), (4, 1, 128, 64, [9000, 5]), (3, 3, 33, 8, [300]), (3, 1, 33, 64, [6000]),
    (20, 4, 80, 16, [500, 3]), (16, 2, 256, 64, [4100]), (2, 1, 250, 64, [2500]), (40, 1, 192, 64, [1500])])
def test_attend_values_near_the_largest(om, ctx, type, heads, kv, D, page, lens):
    """A mean of finite values is finite, however many they are: a pair in one group, and cut
    between groups."""
    rng = np.random.default_rng(D)
    n_pages = sum(-(-n // page) for n in lens)
    c = Cache(om, ctx, type, n_pages, page, kv, D, seed=D)
    large_values(c, 3e38, D)
    c.write()
    table = tables(rng, lens, page, n_pages, -(-max(lens) // page))
    q = rng.standard_normal((len(lens), heads, D)).astype(np.float32)
    score = rng.uniform(0, 2, (len(lens), kv, max(lens))).astype(np.float32)
    for factor in (1.0, 0.0):  # 0: every weight is 1 / n
        out, sc = attend(om, ctx, c, q * factor, lens, table, score=score, max_len=max(lens))
        assert np.isfinite(out).sum() == out.size
        for b, n in enumerate(lens):
            k, v = c.rows(table[b], n) if n else (np.zeros((kv, 0, D)),) * 2
            want, w, tol, tw = attend64((q * factor)[b], k, v, 1 / math.sqrt(D))
            assert np.abs(out[b] - want).max() <= tol, (b, factor)
            add = w.reshape(kv, heads // kv, n).sum(1)
            ws = score[b, :, :n].astype(np.float64) + add
            assert (np.abs(sc[b, :, :n] - ws) <= (tw + 2.0 ** -24 * heads // kv) * add +
                    4 * 2.0 ** -24 * np.abs(ws)).all(), (b, factor)
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 100, 128, 256])
def test_attend_large_values_behind_a_growing_score(om, ctx, type, D):
    """Scores that step up and down by less than a factor of 2^6 within a stretch of one group:
    a weight relative to an earlier maximum is up to 64, and 64 such values are past 32 bits."""
    B, n, page = 150, 4096, 1024
    c = Cache(om, ctx, type, 4, page, 1, D, seed=D)
    large_values(c, 3e37, D)
    c.k[:] = 0.0
    step = torch.arange(n).reshape(4, 1, page) // 256 % 2 == 1
    c.k[..., 0] = torch.where(step, 4.0625, 0.0).to(c.k.dtype)  # 4.0625 log2 e = 5.86
    c.write()
    q = np.zeros((B, 4, D), np.float32)
    q[..., 0] = 1.0
    table = i32(np.tile(np.arange(4), (B, 1)))
    out = attend(om, ctx, c, q, [n] * B, table, scale=1.0)
    k, v = c.rows(table[0], n)
    want, _, tol, _ = attend64(q[0], k, v, 1.0)
    assert np.isfinite(out).sum() == out.size
    assert np.abs(out - want).max() <= tol
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("D,n", [(64, 9000), (128, 200), (33, 700)])
def test_attend_large_values_beside_what_is_not_finite(om, ctx, type, D, n):
    """An infinite value makes its dimension infinite, and the others stay what they are: large
    ones, and ones that would end below the smallest if they were scaled down."""
    rng = np.random.default_rng(n)
    n_pages = -(-n // 64)
    c = Cache(om, ctx, type, n_pages, 64, 1, D, seed=D)
    large_values(c, 3e38, D)
    c.v[..., 3] = (torch.rand(c.v.shape[:3], generator=torch.Generator().manual_seed(1)) * 1e-36).to(c.v.dtype)
    table = tables(rng, [n], 64, n_pages, n_pages)
    c.v[table[0, (n // 2) // 64], 0, n // 2 % 64, 4] = math.inf
    c.write()
    q = rng.standard_normal((1, 4, D)).astype(np.float32)
    out = attend(om, ctx, c, q, [n], table)
    k, v = c.rows(table[0], n)
    assert np.isposinf(out[0][:, 4]).sum() == 4
    for d in [d for d in range(D) if d != 4]:  # every dimension by its own size
        want, _, tol, _ = attend64(q[0], k, v[..., d:d + 1], 1 / math.sqrt(D))
        assert np.abs(out[0][:, d:d + 1] - want).max() <= tol, d
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,n", [(64, 1), (64, 40), (128, 6000), (33, 40), (33, 6000)])
def test_attend_no_weight_at_all_is_zero(om, ctx, type, D, n):
    """A head whose scores are all -infinity gives zeros, whatever the values are; the sequence
    beside it is as ever."""
    rng = np.random.default_rng(n)
    n_pages = 2 * -(-n // 64)
    c = Cache(om, ctx, type, n_pages, 64, 1, D, seed=D)
    table = tables(rng, [n, n], 64, n_pages, n_pages // 2)
    dead = torch.as_tensor(table[0].astype(np.int64))
    c.k[dead] = -math.inf
    c.v[dead[::2]] = math.inf
    c.v[dead[0], 0, 0, 1] = math.nan
    c.write()
    q = np.abs(rng.standard_normal((2, 4, D))).astype(np.float32) + 0.25
    out = attend(om, ctx, c, q, [n, n], table)
    assert (out[0] == 0).sum() == out[0].size
    k, v = c.rows(table[1], n)
    want, _, tol, _ = attend64(q[1], k, v, 1 / math.sqrt(D))
    assert np.abs(out[1] - want).max() <= tol
    c.free()


# ------------------------------------------------------------ scales of the 8-bit type
@pytest.mark.parametrize("what", ["append", "attend", "evict"])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_host_takes_scales_with_a_reciprocal(host, what, which):
    c = Call(host, what)
    c.pages.type = host.om.KV_TYPES["e4m3"]
    for scale in (2.0 ** -126, 1e-20, 0.3, 1e20, 2.0 ** 126):
        setattr(c.pages, which, scale)
        assert c() == (0, 1), scale
    for scale in (1e-45, 1e-39, float(np.nextafter(np.float32(2.0 ** -126), np.float32(0))),
                  float(np.nextafter(np.float32(2.0 ** 126), np.float32(np.inf))), 3e38):
        setattr(c.pages, which, scale)
        assert c() == (-1, 0), scale
    c.pages.type = host.om.KV_TYPES["f16"]  # has no scales
    assert c() == (0, 1)



# ------------------------------------------------------------ calls with nothing to do
@pytest.mark.parametrize("what", ["rope", "append", "attend", "evict"])
def test_host_an_empty_call_waits_and_reports(host, what):
    """A synchronous call ends what was queued before it and reports what it met, also where it has
    no tokens or sequences itself; an asynchronous one does neither."""
    def empty(flags):
        c = Call(host, what)
        c.args["T" if "T" in c.args else "B"] = 0
        if "flags" in c.args:
            c.args["flags"] = flags
        else:
            c.opts.flags = flags
        return c()
    syncs = C.c_int.in_dll(host.L, "kv_syncs")
    host.L.kv_test_mark(host.ctx, 0, 2)
    n = syncs.value
    assert empty(host.om.KV_ASYNC) == (0, 0) and syncs.value == n
    assert empty(0) == (-1, 0) and syncs.value == n + 1 and "row 2" in host.error()
    assert empty(0) == (0, 0)


E4M3 = np.arange(256, dtype=np.uint8)
E4M3 = torch.from_numpy(E4M3).view(torch.float8_e4m3fn).float().numpy()
E4M3 = np.sort(E4M3[np.isfinite(E4M3) & (E4M3 >= 0)])  # 0 twice


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore::RuntimeWarning")  # 449 x 2^126
@pytest.mark.parametrize("scale", [0.3, 1.0, 3.0, 0.0123, 1e-20, 7e15, 2.0 ** -126, 2.0 ** 126, 3.3e-38])
@pytest.mark.parametrize("rotated", [False, True])
def test_append_rounds_the_quotient(om, ctx, scale, rotated):
    """x is stored as x / scale of 32 bits, rounded to nearest: at the middles between two
    values of the type and beside them, at zeros, and past the largest."""
    scale = float(np.float32(scale))
    mid = ((E4M3[1:].astype(np.float64) + E4M3[:-1]) / 2 * scale).astype(np.float32)
    x, d = [mid], mid
    for _ in range(4):
        d = np.nextafter(d, np.float32(np.inf))
        x.append(d)
    d = mid
    for _ in range(4):
        d = np.nextafter(d, np.float32(0))
        x.append(d)
    x = np.concatenate(x + [np.zeros(64, np.float32), (E4M3 * np.float64(scale)).astype(np.float32),
                            np.array([449, 480, 600, 1e6], np.float64).astype(np.float32) * np.float32(scale)])
    x = np.concatenate([x, -x])
    D = 64 if not rotated else 66  # 66: rows that are no whole float4s
    T = -(-x.size // D)
    x = np.concatenate([x, np.zeros(T * D - x.size, np.float32)]).reshape(T, 1, D)
    n_pages = -(-T // 16)
    c = Cache(om, ctx, "e4m3", n_pages, 16, 1, D, seed=1, ks=scale, vs=scale)
    bufs = [ctx.upload(y) for y in (x, i32(np.arange(T)), i32(np.zeros(T)))]
    rope = om.rope_axes([8], 1e4) if rotated else None  # at position 0: nothing turns
    om.kv_append(ctx, c.pages, bufs[0], bufs[0], T, bufs[1], None, None, 0, bufs[2] if rope else None, rope)
    for got, turned in zip(c.read(), (rotated, False)):
        y = x[:, 0].copy()
        if turned:  # cos 1, sin 0; an infinity (past the largest 2^126) makes its pair NaN
            u, v = x[:, 0, 0:16:2], x[:, 0, 1:16:2]
            with np.errstate(invalid="ignore"):
                y[:, 0:16:2], y[:, 1:16:2] = u - v * np.float32(0), u * np.float32(0) + v
        y = torch.from_numpy((y / np.float32(scale)).clip(-448, 448)).to(torch.float8_e4m3fn).float()
        got = got.float().transpose(1, 2).reshape(-1, D)[:T]
        assert torch.isnan(got).sum() == (torch.isnan(got) & torch.isnan(y)).sum() == torch.isnan(y).sum()
        assert torch.isnan(y).sum() == 0 or scale > 1e37
        assert ((got != y) & ~torch.isnan(y)).sum() == 0
    for b in bufs:
        b.free()
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("vs", [2.0 ** -126, 1e-30, 0.3, 1e30])
@pytest.mark.parametrize("n", [40, 5000])
def test_attend_scales_keep_their_digits(om, ctx, vs, n):
    """out is v_scale times the mean of what is stored, to fp32's rounding, at the ends of the
    scales, too: 1 / sum and v_scale are not formed as one small number."""
    rng = np.random.default_rng(n)
    n_pages = -(-n // 64)
    vs = float(np.float32(vs))
    c = Cache(om, ctx, "e4m3", n_pages, 64, 1, 128, seed=n, vs=vs, ks=0.3)
    c.k[:] = 0  # the scores are exact: what is left is the sum's rounding
    c.v.copy_((c.v.float().abs() * 16 + 64).clamp(max=448).to(c.v.dtype))
    c.write()
    table = tables(rng, [n], 64, n_pages, n_pages)
    q = rng.standard_normal((1, 4, 128)).astype(np.float32)
    out = attend(om, ctx, c, q, [n], table)
    k, v = c.rows(table[0], n)
    want, _, tol, _ = attend64(q[0], k, v, 1 / math.sqrt(128))
    assert np.abs(out[0] - want).max() <= tol + 2.0 ** -24 * np.abs(want).max()
    c.free()


# ------------------------------------------------------------ sizes of the launches
@pytest.fixture(scope="module")
def grids(tmp_path_factory):
    """The launches (x, y, z, threads) of calls, by the kernels' own host side."""
    hipcc = "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    root = os.path.dirname(HERE)
    d = tmp_path_factory.mktemp("grids")
    flags = ["-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I" + os.path.join(root, "include")]
    kernels = os.path.join(root, "ornith-flight_amd", "csrc", "kernels")
    for f in ("kv", "kv_attend", "kv_evict"):
        subprocess.run([hipcc, "--offload-host-only", "-O1", "--offload-arch=gfx950", "-std=c++17", *flags[2:],
                        "-c", os.path.join(kernels, f + ".hip"), "-o", str(d / (f + ".o"))], check=True)
    subprocess.run(["gcc", "-std=gnu99", *flags, "-c", os.path.join(HERE, "kv_grids.c"), "-o", str(d / "main.o")],
                   check=True)
    subprocess.run(["g++", "-no-pie", "-Wl,--unresolved-symbols=ignore-all", "-o", str(d / "grids"),
                    *[str(d / (f + ".o")) for f in ("main", "kv", "kv_attend", "kv_evict")]], check=True)

    def run(cases):
        text = "\n".join(" ".join(map(str, c)) for c in cases)
        out = subprocess.run([str(d / "grids")], input=text, capture_output=True, text=True, check=True,
                             timeout=300).stdout.splitlines()
        assert len(out) == len(cases)
        return [np.array(line.split(), np.int64).reshape(-1, 4) for line in out]
    return run


def within_the_limits(cases, launches):
    """A dimension has fewer than 2^32 threads, and y and z at most 65535 groups."""
    for c, g in zip(cases, launches):
        assert len(g) >= 1 and (g >= 1).all(), c
        assert (g[:, 0] * g[:, 3] < 1 << 32).all() and (g[:, 1:3] <= 65535).all(), (c, g.tolist())


@pytest.mark.parametrize("in_place", [0, 1])
@pytest.mark.parametrize("type", [0, 1, 2, 3])
def test_an_evictions_launches_fit(grids, type, in_place):
    """Up to the most that a call may keep, whatever words the rows are moved in."""
    most = 1 << 27
    cases = [("e", hd, type, kv, n, length, keep, in_place) for hd in (1, 8, 33, 64, 129, 130, 192, 250, 255, 256)
             for kv, n in ((1, 1), (8, 3), (32767, 65535))
             for length, keep in ((most, most), (2 ** 31 - 2 ** 16, most), (most, 2 ** 31 - 1), (1 << 26, 1 << 26),
                                  (5000, 700), (1, 1), (0, 1))]
    within_the_limits(cases, grids(cases))


def test_an_attentions_and_a_rotations_launches_fit(grids):
    cases = [("a", hd, type, kv, n, length, heads, score) for hd in (1, 64, 100, 256) for type in range(4)
             for kv, n, heads in ((1, 1, 65535), (32, 65535, 32), (1, 65535, 512), (32767, 64, 32767))
             for length in (1, 5000, 2 ** 31 - 2 ** 16) for score in (0, 1)]
    cases += [("r", hd, R, halves, kv, T, heads, slots) for hd, R in ((1, 0), (64, 32), (66, 33), (4096, 256))
              for halves in (0, 1) for kv, heads in ((1, 0), (8, 64), (65535, 65535))
              for T in (1, 4097, 2 ** 31 - 1) for slots in (0, 1)]
    within_the_limits(cases, grids(cases))


@pytest.mark.gpu
def test_evict_more_stretches_than_a_launch_takes(om, ctx):
    """Rows of 129 bytes are moved by stretches of 4, and more than 2^20 stretches by more than one
    launch.  Equal scores keep the first tokens, in order."""
    D, page, n, keep = 129, 1024, 4_400_000, 4_300_000
    new, old = -(-keep // page), -(-n // page)
    rng = np.random.default_rng(2)
    nbytes = (new + old) * page * D
    K, V = ctx.alloc(nbytes), ctx.alloc(nbytes)
    pages = om.kv_pages(K, V, "e4m3", new + old, page, 1, D)
    x = rng.integers(0, 256, nbytes, np.uint8)
    for b in (K, V):
        om.lib().gpu_copy_to_device(ctx.ptr, b.ptr, om._p(x), nbytes)
        x = x[::-1].copy()
    table, dst = i32(new + np.arange(old))[None], i32(rng.permutation(new))[None]
    bufs = [ctx.upload(a) for a in (table, i32([n]), np.zeros(n, np.float32), dst, i32([0]), np.zeros(keep, np.int32))]
    tb, lb, sb, db, dl, kb = bufs
    om.kv_evict(ctx, pages, 1, tb, old, lb, sb, n, db, new, dl, None, 0, kb, om.evict_opts(keep, max_len=n))
    assert ctx.download(dl, np.int32, (1,))[0] == keep
    assert np.array_equal(ctx.download(kb, np.int32, (keep,)), np.arange(keep))
    for b in (K, V):
        got = ctx.download(b, np.uint8, (new, page, D))[dst[0]].reshape(-1, D)
        src = x.reshape(-1, page, D)
        assert np.array_equal(got[:keep], src[new:].reshape(-1, D)[:keep])
        last = src[:new][dst[0]].reshape(-1, D)
        assert np.array_equal(got[keep:], last[keep:])  # places past the last are as they were
        x = x[::-1].copy()
    for b in bufs + [K, V]:
        b.free()


# ------------------------------------------------------------ bits of the products
def sharp(type, D, seed, bits=24):
    """Queries of a few dimensions and keys whose scores lie up to 40 apart (three heads) and up
    to 0.8 (three more), V's column j the indicator of token j (so out_j is its weight) and its
    last column 1.  Returns q, k, v, the weights in 64 bits and what each may be off, relative
    to itself.

    A score is the sum of 4 products of positive numbers: 12 products of parts and their sums,
    each rounded once, and the scale's two roundings in the query: 16 e of itself, for the
    token's score and for the largest; the exponential and the share 8 e, the sum's chain
    6 sqrt(n) e.  With bits = 16 the query and the weights are cut to 16 bits, as two parts of
    8 would hold them."""
    rng = np.random.default_rng(seed)
    n = 12
    q = np.zeros((6, D), np.float32)
    dims = rng.permutation(D)[:4]
    q[:, dims] = rng.uniform(2, 4, (6, 4)).astype(np.float32) * math.sqrt(D)
    q[3:] *= 0.02
    k = torch.zeros(n, D)
    level = torch.linspace(-1.5, 1.5, n)[torch.from_numpy(rng.permutation(n))]
    k[:, dims] = level[:, None] * torch.from_numpy(rng.uniform(0.9, 1.1, (n, 4)).astype(np.float32))
    v = torch.zeros(n, D)
    v[torch.arange(n), torch.arange(n)] = 1.0
    v[:, D - 1] = 1.0
    k, v = k.to(DTYPE[type]), v.to(DTYPE[type])

    def cut(x):
        return (x.astype(np.float32).view(np.uint32) & np.uint32(2 ** 32 - 2 ** (24 - bits))).view(np.float32)
    qs = cut(q) if bits < 24 else q
    s = qs.astype(np.float64) @ value(k).T / math.sqrt(D)
    e = np.exp(s - s.max(1, keepdims=True))
    w = (cut(e).astype(np.float64) if bits < 24 else e) / e.sum(1, keepdims=True)
    size = np.abs(s) + np.abs(s).max(1, keepdims=True)
    tol = (16 * size + 8 + 6 * math.sqrt(n)) * 2.0 ** -24
    one = (8 + 6 * math.sqrt(n)) * 2.0 ** -24  # the column of ones: scores do not count
    return q, k, v, w, tol, one


SHARP = [(type, D) for type in DTYPE for D in (64, 80, 128, 250, 256)]


@pytest.mark.parametrize("type,D", SHARP)
def test_16_bits_are_too_few_for_the_next_test(type, D):
    for seed in range(4):
        _, _, _, w, tol, one = sharp(type, D, seed)
        _, _, _, w16, _, _ = sharp(type, D, seed, bits=16)
        assert (np.abs(w16 - w) > 2 * tol * w)[:3].any()
        assert (np.abs(w16.sum(1) - 1) > 2 * one)[3:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("type,D", SHARP)
def test_attend_keeps_24_bits(om, ctx, type, D):
    for seed in range(4):
        q, k, v, w, tol, one = sharp(type, D, seed)
        n = k.shape[0]
        c = Cache(om, ctx, type, 1, 16, 1, D)
        c.k[0, 0, :n], c.v[0, 0, :n] = k, v
        c.write()
        score = np.zeros((1, 1, 16), np.float32)
        out, sc = attend(om, ctx, c, q[None], [n], i32([[0]]), score=score)
        assert (np.abs(out[0, :, :n] - w) <= tol * w).all()
        assert (np.abs(out[0, :, D - 1] - 1) <= one).all()
        assert (np.abs(sc[0, 0, :n] - w.sum(0)) <= (tol * w).sum(0) + 4 * 2.0 ** -24 * w.sum(0)).all()
        c.free()


# ------------------------------------------------------------ a workspace that grows
def test_a_growing_workspace_waits_before_it_frees(tmp_path):
    exe = tmp_path / "kv_growth"
    r = subprocess.run(["gcc", "-std=gnu99", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-no-pie",
                        "-Wl,--unresolved-symbols=ignore-all", "-o", str(exe), os.path.join(HERE, "kv_growth.c"),
                        "-lm"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    out = subprocess.run([str(exe), "100", "50", "100", "1000", "999", "1", "100000"], capture_output=True,
                         text=True, timeout=60, check=True).stdout.split("\n")
    assert out[0] in ("m", "wm") and out[1:7] == ["", "", "wfm", "", "", "wfm"]


@pytest.mark.gpu
def test_calls_in_a_row_on_a_growing_workspace(om):
    """Asynchronous calls of a fresh context, each asking for more room than the ones before or
    for less, with an eviction between: each gives what it gives alone."""
    rng = np.random.default_rng(19)
    one, two = om.Context(), om.Context()
    c = Cache(om, one, "bf16", 600, 16, 2, 128, seed=10)
    jobs, want = [], []
    for B, n, score in ((1, 40, False), (2, 900, True), (1, 4000, False), (3, 30, True), (2, 4000, True),
                        (1, 300, True), (9, 600, False), (4, 2000, True), (1, 5, False)):
        lens = [n] + [int(x) for x in rng.integers(0, n + 1, B - 1)]
        table = i32(rng.integers(0, 300, (B, 250)))  # of the first half: pages that only the attention reads
        q = rng.standard_normal((B, 8, 128)).astype(np.float32)
        s = rng.uniform(0, 1, (B, 2, n)).astype(np.float32) if score else None
        want.append(attend(om, two, c, q, lens, table, score=s, max_len=n))
        b = [one.upload(x) for x in (q, np.zeros_like(q), table, i32(lens))]
        o = dict(max_len=n, flags=om.KV_ASYNC)
        if score:
            b += [one.upload(s), one.upload(np.full_like(s, -9.0))]
            o.update(score_in=b[4], score_out=b[5], score_stride=n)
        jobs.append((B, b, om.attend_opts(**o)))
    # an eviction of many sequences of two tokens each, in the second half's pages
    N = 300
    ev = [one.upload(x) for x in (i32(300 + np.arange(N))[:, None], i32([2] * N),
                                  rng.uniform(0, 1, (N, 2, 16)).astype(np.float32), np.zeros((N, 2, 1), np.int32))]
    score = one.download(ev[2], np.float32, (N, 2, 16))
    for i, (B, b, o) in enumerate(jobs):
        om.kv_attend(one, c.pages, b[1], b[0], B, 8, b[2], 250, b[3], o)
        if i == 4:
            om.kv_evict(one, c.pages, N, ev[0], 1, ev[1], ev[2], 16, ev[0], 1, ev[1], None, 0, ev[3],
                        om.evict_opts(1, flags=om.KV_ASYNC))
    assert om.lib().gpu_kv_check(one.ptr) == 0
    for (B, b, _), w in zip(jobs, want):
        out, sc = w if isinstance(w, tuple) else (w, None)
        assert np.array_equal(one.download(b[1], np.float32, out.shape), out)
        if sc is not None:
            assert np.array_equal(one.download(b[5], np.float32, sc.shape), sc)
    assert np.array_equal(one.download(ev[3], np.int32, (N, 2, 1))[..., 0], score[:, :, :2].argmax(2))
    assert (one.download(ev[1], np.int32, (N,)) == 1).sum() == N
    c.free()
    for x in (one, two):
        x.close()

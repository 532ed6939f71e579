"""The paged key-value cache (gpu_kv_append, gpu_kv_attend, gpu_kv_evict) and
gpu_rope_axes.

CPU: what the host refuses, and what it hands to the kernels, with
csrc/host/kv.c compiled over counting launches (tests/kv_host.c).

GPU: each call against its definition in 64 bits over the values the cache
holds.  With e = 2^-24 (half a step of fp32):
  rope    an output is u c - v s.  The turn is rounded to fp32 at up to half a
          turn (error 2^-25 half turns, pi 2^-25 of angle), sin and cos are
          within two ulp (2 x 2^-24), the two products and the sum round by e
          each: at most (|u| + |v|) (pi / 2 + 2 + 2) e < 6 e (|u| + |v|).
  append  the same, and half a step of the cache's type.
  attend  a score of D products is off by rounding errors that are independent
          for random inputs: 6 standard deviations are below
          ds = 6 sqrt(2 D) e scale max_t sum_d |q_d k_td|.  A weight is then off
          by 2 ds + 8 e of itself (its exponential and its share of the sum,
          the sum's own chain of n terms by 6 sqrt(n) e), and so is an output,
          relative to the largest |v|.
  evict   copies and whole numbers: equal.
"""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
EPS = 2.0 ** -24
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
         "e4m3": torch.float8_e4m3fn}
# half a step of a normal value, relative to it, and of the smallest values
STEP = {"f32": (2.0 ** -24, 2.0 ** -150), "f16": (2.0 ** -11, 2.0 ** -25),
        "bf16": (2.0 ** -8, 2.0 ** -134), "e4m3": (2.0 ** -4, 2.0 ** -10)}


@pytest.fixture(scope="module")
def om():
    import ornith_moe
    ornith_moe.lib()
    return ornith_moe


# ------------------------------------------------------------ the host, on the CPU
class Host:
    """kv.c over counting launches; every call is one of its entry points."""

    def __init__(self, om, so):
        self.om, self.L = om, C.CDLL(so)
        for n in ("kv_test_context", "kv_test_buffer"):
            getattr(self.L, n).restype = C.c_void_p
        self.L.kv_test_buffer.argtypes = [C.c_size_t]
        self.L.kv_test_error.restype = C.c_char_p
        self.L.kv_test_error.argtypes = [C.c_void_p]
        self.L.kv_test_mark.argtypes = [C.c_void_p, C.c_int, C.c_int]
        self.L.kv_test_workspace.argtypes = [C.c_void_p]
        self.L.kv_test_turns.restype = C.c_double
        real = om.lib()
        for n in ("gpu_rope_axes", "gpu_kv_append", "gpu_kv_attend", "gpu_kv_evict", "gpu_kv_check"):
            getattr(self.L, n).argtypes = getattr(real, n).argtypes
        self.ctx = self.L.kv_test_context(0)

    def launches(self):
        return C.c_int.in_dll(self.L, "kv_launches").value

    def buf(self, n):
        return self.L.kv_test_buffer(n)

    def error(self):
        return self.L.kv_test_error(self.ctx).decode()


@pytest.fixture(scope="module")
def host(om, tmp_path_factory):
    so = str(tmp_path_factory.mktemp("kv") / "kv_host.so")
    r = subprocess.run(["gcc", "-std=gnu99", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                        "-shared", "-fPIC", "-o", so, os.path.join(HERE, "kv_host.c"), "-lm"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    return Host(om, so)


class Call:
    """A right call of each entry point (3 sequences of up to 40 tokens, 4 heads over 2 kv
    heads of 32, pages of 16); `args` are changed by the tests."""

    def __init__(self, h, what):
        self.h, self.what, om = h, what, h.om
        B, H, kv, D, n_pages, width, T = 3, 4, 2, 32, 9, 3, 5
        page = n_pages * kv * 16 * D * 2
        self.pages = om.KVPages(h.buf(page), h.buf(page), om.KV_TYPES["f16"], n_pages, 16, kv, D, 0, 0)
        self.rope = om.rope_axes([4, 6, 2], 1e4)
        if what == "rope":
            self.args = dict(q_out=h.buf(T * H * D * 4), k_out=h.buf(T * kv * D * 4),
                             Q=h.buf(T * H * D * 4), K=h.buf(T * kv * D * 4), T=T, heads=H, kv=kv,
                             D=D, pos=h.buf(3 * T * 4), rope=self.rope, flags=0)
        elif what == "append":
            self.args = dict(pages=self.pages, K=h.buf(T * kv * D * 4), V=h.buf(T * kv * D * 4), T=T,
                             slots=h.buf(T * 4), q_out=h.buf(T * H * D * 4), Q=h.buf(T * H * D * 4),
                             heads=H, pos=h.buf(3 * T * 4), rope=self.rope, flags=0)
        elif what == "attend":
            self.opts = om.AttendOpts(0, 40, 0, h.buf(B * kv * 40 * 4), h.buf(B * kv * 40 * 4), 40, 1)
            self.args = dict(pages=self.pages, out=h.buf(B * H * D * 4), Q=h.buf(B * H * D * 4), B=B,
                             heads=H, table=h.buf(B * width * 4), width=width, lens=h.buf(B * 4),
                             opts=self.opts)
        else:
            self.opts = om.EvictOpts(20, 2, 3, 40, 0)
            self.args = dict(pages=self.pages, B=B, table=h.buf(B * width * 4), width=width,
                             lens=h.buf(B * 4), score=h.buf(B * kv * 40 * 4), stride=40,
                             dst=h.buf(B * 2 * 4), dst_pages=2, dst_lens=h.buf(B * 4),
                             dst_score=h.buf(B * kv * 20 * 4), dst_stride=20,
                             kept=h.buf(B * kv * 20 * 4), opts=self.opts)

    def __call__(self):
        fn = getattr(self.h.L, {"rope": "gpu_rope_axes"}.get(self.what, "gpu_kv_" + self.what))
        a = [C.byref(v) if isinstance(v, C.Structure) else v for v in self.args.values()]
        n = self.h.launches()
        rc = fn(self.h.ctx, *a)
        return rc, self.h.launches() - n


@pytest.mark.parametrize("what", ["rope", "append", "attend", "evict"])
def test_host_takes_a_right_call(host, what):
    assert Call(host, what)() == (0, 1)
    c = Call(host, what)
    for a in ("T", "B"):
        if a in c.args:
            c.args[a] = 0
    assert c() == (0, 0)  # nothing to do


@pytest.mark.parametrize("what", ["append", "attend", "evict"])
@pytest.mark.parametrize("field,value", [
    ("K", None), ("V", None), ("type", 4), ("type", -1), ("n_pages", 0), ("n_pages", 10),
    ("n_pages", 1 << 28), ("page_size", 0), ("page_size", 4), ("page_size", 24),
    ("page_size", 2048), ("n_kv_heads", 0), ("n_kv_heads", 3), ("n_kv_heads", 1 << 20),
    ("head_dim", 0), ("head_dim", 33), ("head_dim", 257)])
def test_host_refuses_pages(host, what, field, value):
    c = Call(host, what)
    setattr(c.pages, field, value)
    rc, n = c()
    assert rc < 0 and n == 0 and host.error().startswith("gpu_kv_" + what)


@pytest.mark.parametrize("what", ["append", "attend", "evict"])
@pytest.mark.parametrize("scale", [-1.0, math.inf, math.nan])
def test_host_refuses_scales_of_8_bits(host, what, scale):
    c = Call(host, what)
    c.pages.type = host.om.KV_TYPES["e4m3"]
    assert c() == (0, 1)
    c.pages.v_scale = scale
    assert c()[0] < 0


REFUSED = [
    ("rope", "pos", None), ("rope", "Q", None), ("rope", "k_out", None), ("rope", "heads", 0),
    ("rope", "T", -1), ("rope", "T", 6), ("rope", "heads", 5), ("rope", "kv", 3), ("rope", "D", 23),
    ("rope", "heads", 1 << 20),
    ("append", "K", None), ("append", "V", None), ("append", "slots", None), ("append", "T", 6),
    ("append", "T", -1), ("append", "heads", 5), ("append", "heads", 0), ("append", "q_out", None),
    ("append", "pos", None), ("append", "T", 1 << 30),
    ("attend", "out", None), ("attend", "Q", None), ("attend", "table", None),
    ("attend", "lens", None), ("attend", "B", 4), ("attend", "B", -1), ("attend", "heads", 3),
    ("attend", "heads", 6), ("attend", "heads", 0), ("attend", "width", 4), ("attend", "width", 2),
    ("attend", "width", -1), ("attend", "width", 1 << 30), ("attend", "B", 1 << 30),
    ("evict", "table", None), ("evict", "lens", None), ("evict", "score", None),
    ("evict", "dst", None), ("evict", "dst_lens", None), ("evict", "kept", None),
    ("evict", "opts", None), ("evict", "B", 4), ("evict", "width", 2), ("evict", "stride", 39),
    ("evict", "stride", 41), ("evict", "dst_pages", 1), ("evict", "dst_pages", 3),
    ("evict", "dst_stride", 19), ("evict", "dst_stride", 21), ("evict", "stride", -1)]


@pytest.mark.parametrize("what,arg,value", REFUSED)
def test_host_refuses_arguments(host, what, arg, value):
    c = Call(host, what)
    assert arg in c.args
    c.args[arg] = value
    rc, n = c()
    assert rc < 0 and n == 0 and host.error()


@pytest.mark.parametrize("what,out,others", [
    ("rope", "q_out", ["K", "pos", "k_out"]), ("rope", "k_out", ["Q", "pos"]),
    ("append", "q_out", ["slots", "pos"]),
    ("attend", "out", ["Q", "table", "lens"]),
    ("evict", "kept", ["table", "lens", "score", "dst"]), ("evict", "dst_lens", ["table"]),
    ("evict", "dst_score", ["kept"])])
def test_host_refuses_aliases(host, what, out, others):
    for o in others:
        c = Call(host, what)
        big = host.buf(1 << 20)
        c.args[out] = c.args[o] = big
        assert c() in [(-1, 0)], (out, o)


def test_host_refuses_rotated_queries_over_rows_still_to_be_read(host):
    """q_out may be Q, but not where K or V is that buffer, too."""
    for o in ("K", "V"):
        c = Call(host, "append")
        c.args["q_out"] = c.args["Q"] = c.args[o] = host.buf(1 << 20)
        assert c() == (-1, 0), o
    c = Call(host, "rope")
    c.args["q_out"] = c.args["Q"] = c.args["K"] = host.buf(1 << 20)
    assert c() == (-1, 0)


def test_host_takes_in_place_calls(host):
    c = Call(host, "rope")
    c.args["q_out"], c.args["k_out"] = c.args["Q"], c.args["K"]
    assert c() == (0, 1)
    c = Call(host, "append")
    c.args["q_out"] = c.args["Q"]
    assert c() == (0, 1)
    c = Call(host, "attend")
    c.opts.score_in = c.opts.score_out
    assert c() == (0, 1)
    c = Call(host, "evict")
    c.args.update(dst=c.args["table"], dst_pages=3, dst_lens=c.args["lens"],
                  dst_score=c.args["score"], dst_stride=40)
    assert c() == (0, 1)
    c.args["dst_pages"] = 2
    assert c() == (-1, 0)


def test_host_leaves_sides_out(host):
    c = Call(host, "rope")
    c.args.update(K=None, k_out=None, kv=0)
    assert c() == (0, 1)
    c = Call(host, "append")
    c.args.update(Q=None, q_out=None, heads=0)
    assert c() == (0, 1)
    c.args.update(pos=None, rope=None)
    assert c() == (0, 1)
    c.args.update(Q=host.buf(1 << 20), q_out=host.buf(1 << 20), heads=4)
    assert c() == (-1, 0)  # queries without a rotation
    c = Call(host, "attend")
    c.args["opts"] = None
    assert c() == (0, 1)
    c = Call(host, "evict")
    c.args.update(dst_score=None, dst_stride=0)
    assert c() == (0, 1)


@pytest.mark.parametrize("change", [
    dict(n_axes=0), dict(n_axes=5), dict(base=0.0), dict(base=-1.0), dict(base=math.inf),
    dict(base=math.nan), dict(pairs=(4, -1, 2, 0)), dict(pairs=(6, 6, 5, 0)),
    dict(pairs=(1 << 30, 1 << 30, 1 << 30, 0)), dict(n_axes=4),
    dict(base=5e-324, pairs=(16, 0, 0, 0))])
def test_host_refuses_rotations(host, change):
    for what in ("rope", "append"):
        c = Call(host, what)
        for k, v in change.items():
            setattr(c.rope, k, (C.c_int * 4)(*v) if k == "pairs" else v)
        assert c()[0] < 0, what


@pytest.mark.parametrize("change", [
    dict(scale=math.nan), dict(scale=math.inf), dict(max_len=49), dict(max_len=-1), dict(max_len=41),
    dict(max_len=0), dict(score_stride=39), dict(score_stride=41), dict(score_stride=-1),
    dict(score_out=None), dict(score_new=-1)])
def test_host_refuses_attend_options(host, change):
    c = Call(host, "attend")
    for k, v in change.items():
        setattr(c.opts, k, v)
    assert c() == (-1, 0)


@pytest.mark.parametrize("change", [
    dict(keep=0), dict(keep=4), dict(sink=-1), dict(recent=-1), dict(sink=2 ** 31 - 1),
    dict(max_len=49), dict(max_len=-1), dict(max_len=0), dict(keep=21), dict(keep=2 ** 31 - 1)])
def test_host_refuses_evict_options(host, change):
    c = Call(host, "evict")
    for k, v in change.items():
        setattr(c.opts, k, v)
    assert c() == (-1, 0)


def test_host_refuses_what_passes_its_limits(host):
    """Calls whose buffers would hold what they ask for."""
    def big(what, pages=(), args=(), opts=()):
        c = Call(host, what)
        for k, v in c.args.items():
            if isinstance(v, int) and v > 1 << 30:  # a buffer's handle
                c.args[k] = host.buf(1 << 60)
        c.pages.K, c.pages.V = host.buf(1 << 60), host.buf(1 << 60)
        c.args.update(args)
        for k, v in dict(pages).items():
            setattr(c.pages, k, v)
        for k, v in dict(opts).items():
            setattr(c.opts, k, v)
        return c()
    att = dict(score_in=None, score_out=None)
    assert big("attend", opts=att) == (0, 1)
    assert big("attend", args=dict(B=65535), opts=att) == (0, 1)
    assert big("attend", args=dict(B=65536), opts=att) == (-4, 0)
    assert big("attend", dict(n_kv_heads=32), dict(B=65535, heads=32), att) == (0, 1)
    assert big("attend", dict(n_kv_heads=33), dict(B=65535, heads=33), att) == (-4, 0)
    assert big("attend", dict(n_kv_heads=32), dict(B=65535, heads=32 * 17), att) == (-4, 0)
    assert big("attend", args=dict(heads=65536), opts=att)[0] < 0
    wide = dict(page_size=1024)
    assert big("attend", wide, dict(width=2 ** 21 - 64), dict(att, max_len=0)) == (0, 1)
    assert big("attend", wide, dict(width=2 ** 21 - 63), dict(att, max_len=0)) == (-1, 0)
    page = dict(page_size=1024, head_dim=256, type=0)
    assert big("append", dict(page, n_kv_heads=4095)) == (0, 1)
    assert big("append", dict(page, n_kv_heads=4096)) == (-4, 0)
    assert big("rope", args=dict(D=4096)) == (0, 1)
    assert big("rope", args=dict(D=4097)) == (-4, 0)
    assert big("rope", args=dict(heads=65536))[0] < 0
    far = dict(width=2 ** 18, stride=2 ** 28, dst_pages=2 ** 18, dst_stride=2 ** 28)
    assert big("evict", wide, far, dict(keep=1 << 27, max_len=0)) == (0, 1)
    assert big("evict", wide, far, dict(keep=(1 << 27) + 1, max_len=0)) == (-4, 0)
    assert big("evict", wide, far, dict(keep=2 ** 31 - 1, max_len=1 << 27)) == (0, 1)


def test_host_no_context(host):
    for what in ("rope", "append", "attend", "evict"):
        c = Call(host, what)
        ctx, host.ctx = host.ctx, None
        try:
            assert c() == (-1, 0)
        finally:
            host.ctx = ctx
    assert host.L.gpu_kv_check(None) < 0


def test_host_runs_on_the_contexts_device(host):
    dev = C.c_int.in_dll(host.L, "kv_device")
    dev.value = 3
    assert Call(host, "attend")() == (0, 1) and dev.value == 3
    dev.value = 0


def test_host_without_room(host):
    ctx, host.ctx = host.ctx, host.L.kv_test_context(0)
    no = C.c_int.in_dll(host.L, "kv_no_room")
    no.value = 1
    assert Call(host, "attend")() == (-2, 0) and "workspace" in host.error()
    assert Call(host, "evict")() == (-2, 0)
    no.value = 0
    assert Call(host, "attend")() == (0, 1) and host.L.kv_test_workspace(host.ctx)
    host.ctx = ctx


def test_host_reports_what_the_kernels_met(host):
    L = host.L
    for what, at, said in ((0, 2, "row 2"), (1, 7, "token 7"), (2, 0, "sequence 0")):
        L.kv_test_mark(host.ctx, what, at)
        syncs = C.c_int.in_dll(L, "kv_syncs").value
        c = Call(host, "rope")
        c.args["flags"] = host.om.KV_ASYNC  # neither waits nor looks
        assert c() == (0, 1) and C.c_int.in_dll(L, "kv_syncs").value == syncs
        assert L.gpu_kv_check(host.ctx) == -1 and said in host.error()
        assert L.gpu_kv_check(host.ctx) == 0  # once
        L.kv_test_mark(host.ctx, what, at)
        assert Call(host, "append")()[0] == -1 and said in host.error()


@pytest.mark.parametrize("pairs,interleaved,axes", [
    ([3, 0, 2], 0, [0, 0, 0, 2, 2]), ([3, 0, 2], 1, [0, 2, 0, 2, 0]), ([2, 4, 1], 1, [0, 1, 2, 0, 1, 1, 1]),
    ([16], 0, [0] * 16), ([16], 1, [0] * 16), ([0, 0], 0, [])])
def test_host_deals_out_the_axes(host, pairs, interleaved, axes):
    c = Call(host, "rope")
    c.args["rope"] = host.om.rope_axes(pairs, 1e6, interleaved=interleaved)
    assert c() == (0, 1)
    assert [host.L.kv_test_axis(p) for p in range(len(axes))] == axes
    R = len(axes)
    for p in range(R):
        want = 1e6 ** (-p / R) / (2 * math.pi)
        assert abs(host.L.kv_test_turns(p) - want) <= want * (p + 4) * 2.0 ** -52


# ------------------------------------------------------------ definitions in 64 bits
def stored(x, type, scale=1.0):
    """The value a cache of `type` holds for fp32 x."""
    x = torch.as_tensor(x, dtype=torch.float32)
    if type == "e4m3":
        x = x * (np.float32(1.0) / np.float32(scale))
        x = x.clamp(-448.0, 448.0)
    return x.to(DTYPE[type])


def value(x, scale=1.0):
    return x.to(torch.float64).numpy() * scale


def rope64(x, pos, pairs, base, halves, interleaved):
    """x [T][heads][D] rotated, and the largest rounding (|u| + |v|) * 6 e of every output."""
    R, left, axis = sum(pairs), list(pairs), []
    while len(axis) < R:
        for a in range(len(pairs)):
            n = min(left[a], 1) if interleaved else left[a]
            axis += [a] * n
            left[a] -= n
    x = x.astype(np.float64)
    y, tol = x.copy(), np.zeros_like(x)
    for p in range(R):
        i, j = (p, p + R) if halves else (2 * p, 2 * p + 1)
        ang = (pos[axis[p]].astype(np.float64) * base ** (-p / R))[:, None]
        u, v = x[..., i], x[..., j]
        y[..., i], y[..., j] = u * np.cos(ang) - v * np.sin(ang), u * np.sin(ang) + v * np.cos(ang)
        tol[..., i] = tol[..., j] = 6 * EPS * (np.abs(u) + np.abs(v))
        # the angle itself, in 64 bits, of pos turns at most
        tol[..., i] += (np.abs(u) + np.abs(v)) * np.abs(ang) * (p + 4) * 2.0 ** -52
        tol[..., j] = tol[..., i]
    return y, tol


def attend64(q, k, v, scale):
    """q [H][D], k and v [kv][n][D]: out [H][D], weights [H][n], and the tolerance of out and
    of a weight."""
    H, D = q.shape
    kv, n, _ = k.shape
    out, w = np.zeros((H, D)), np.zeros((H, n))
    if n == 0:
        return out, w, 0.0, 0.0
    big = 0.0
    with np.errstate(over="ignore", invalid="ignore"):
        for j in range(H):
            h = j // (H // kv)
            s = (k[h] @ q[j].astype(np.float64)) * scale
            big = max(big, scale * (np.abs(k[h]) @ np.abs(q[j].astype(np.float64))).max())
            e = np.exp(s - s.max())
            w[j] = e / e.sum()
            out[j] = w[j] @ v[h]
    ds = 6 * math.sqrt(2 * D) * EPS * big
    tw = 2 * ds + 8 * EPS + 6 * math.sqrt(n) * EPS
    return out, w, (tw + 6 * math.sqrt(n) * EPS) * np.abs(v).max(), tw


def choose(score, n, keep, sink, recent):
    """The kept tokens of one kv head, in order."""
    if n <= keep:
        return list(range(n))
    mid = range(sink, n - recent)
    key = [(-math.inf if math.isnan(s) else float(s)) for s in score]
    # a NaN is below everything, an infinity among the numbers
    mid = sorted(mid, key=lambda i: (math.isnan(score[i]), -key[i], i))
    return sorted(list(range(sink)) + mid[:keep - sink - recent] + list(range(n - recent, n)))


# ------------------------------------------------------------ on the GPU
@pytest.fixture(scope="module")
def ctx(om):
    c = om.Context()
    yield c
    c.close()


class Cache:
    """Pages on the device and what they hold, as tensors [page][kv][slot][D]."""

    def __init__(self, om, ctx, type, n_pages, page, kv, D, seed=0, ks=0.0, vs=0.0):
        g = torch.Generator().manual_seed(seed)
        self.type, self.page, self.om, self.ctx = type, page, om, ctx
        self.ks, self.vs = ks or 1.0, vs or 1.0
        shape = (n_pages, kv, page, D)
        self.k = stored(torch.randn(shape, generator=g) * self.ks, type, self.ks)
        self.v = stored(torch.randn(shape, generator=g) * self.vs, type, self.vs)
        self.K, self.V = ctx.alloc(self.bytes()), ctx.alloc(self.bytes())
        self.pages = om.kv_pages(self.K, self.V, type, n_pages, page, kv, D, ks, vs)
        self.write()

    def bytes(self):
        return self.k.numel() * self.k.element_size()

    def write(self):
        for b, x in ((self.K, self.k), (self.V, self.v)):
            a = x.contiguous().view(torch.uint8).numpy()
            self.om.lib().gpu_copy_to_device(self.ctx.ptr, b.ptr, self.om._p(a), a.nbytes)

    def read(self):
        return tuple(torch.from_numpy(self.ctx.download(b, np.uint8, (self.bytes(),)))
                     .view(self.k.dtype).view(self.k.shape) for b in (self.K, self.V))

    def rows(self, ids, n):
        """Values [kv][n][D] of K and V of a sequence."""
        out = []
        for x, s in ((self.k, self.ks), (self.v, self.vs)):
            x = value(x[torch.as_tensor(ids[:-(-n // self.page)], dtype=torch.int64)], s)
            out.append(x.transpose(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[3])[:, :n])
        return out

    def free(self):
        self.K.free()
        self.V.free()


def same(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def i32(a):
    return np.ascontiguousarray(a, np.int32)


ROPES = [(1, 2, 1, 8, [4], 0, 0), (1, 16, 2, 256, [32], 0, 0), (7, 3, 1, 6, [1, 1, 1], 0, 1),
         (33, 5, 0, 128, [24, 20, 20], 1, 1), (5, 0, 4, 80, [10, 0, 7, 3], 1, 1), (3, 4, 2, 33, [16], 0, 0),
         (129, 32, 8, 128, [16, 24, 24], 1, 0), (2, 1, 1, 512, [100, 100, 56], 0, 1),
         (4, 2, 2, 64, [0], 0, 0), (3, 2, 1, 100, [5, 8], 1, 0), (1000, 2, 1, 64, [11, 11, 10], 1, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("start", [0, 131071, -5, 2 ** 31 - 3000])
@pytest.mark.parametrize("T,heads,kv,D,pairs,halves,inter", ROPES)
def test_rope_axes(om, ctx, T, heads, kv, D, pairs, halves, inter, start):
    rng = np.random.default_rng(T + D)
    q = rng.standard_normal((T, heads, D)).astype(np.float32)
    k = rng.standard_normal((T, kv, D)).astype(np.float32)
    pos = i32(start + rng.integers(0, 2 * T + 1, (len(pairs), T)))
    rope = om.rope_axes(pairs, 1e6, halves, inter)
    qb, kb, pb = (ctx.upload(x) if x.size else None for x in (q, k, pos))
    for in_place in (False, True):
        qo = None if qb is None else qb if in_place else ctx.alloc(q.nbytes)
        ko = None if kb is None else kb if in_place else ctx.alloc(k.nbytes)
        om.rope_axes_apply(ctx, qo, ko, qb, kb, T, heads, kv, D, pb, rope)
        for x, b, o in ((q, qb, qo), (k, kb, ko)):
            if b is None:
                continue
            want, tol = rope64(x, pos, pairs, 1e6, halves, inter)
            got = ctx.download(o, np.float32, x.shape)
            assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()
            R2 = 2 * sum(pairs)
            assert np.array_equal(got[..., R2:].view(np.uint32), x[..., R2:].view(np.uint32))
            if not in_place:
                assert np.array_equal(ctx.download(b, np.float32, x.shape), x)
                o.free()
    for b in (qb, kb, pb):
        if b:
            b.free()


@pytest.mark.gpu
def test_rope_axes_of_one_axis_is_gpu_rope(om, ctx):
    """One axis of 32 pairs in adjacent order: gpu_rope's rotation (whose angle is rounded to
    fp32: pos * 2^-24 of angle)."""
    rng = np.random.default_rng(2)
    q, k = (rng.standard_normal((n, 256)).astype(np.float32) for n in (16, 2))
    for pos in (0, 1, 1000):
        b = [ctx.upload(x) for x in (q, k, q, k, i32([pos]))]
        om.lib().gpu_rope(ctx.ptr, b[0].ptr, b[1].ptr, 1, 256, 16, 2, C.c_float(1e7), pos)
        om.rope_axes_apply(ctx, b[2], b[3], b[2], b[3], 1, 16, 2, 256, b[4], om.rope_axes([32], 1e7))
        for i, x in ((0, q), (1, k)):
            u, v = ctx.download(b[i], np.float32, x.shape), ctx.download(b[i + 2], np.float32, x.shape)
            big = np.abs(x).max() * 2
            assert np.abs(u - v).max() <= big * (12 * EPS + 3 * pos * EPS)
            if pos == 0:
                assert np.array_equal(v, x)
        for x in b:
            x.free()


@pytest.mark.gpu
@pytest.mark.parametrize("type", list(DTYPE))
@pytest.mark.parametrize("T,heads,kv,D,page,pairs,halves", [
    (1, 4, 2, 256, 16, [32], 0), (19, 8, 1, 64, 8, [11, 11, 10], 1), (70, 0, 3, 80, 32, [20], 1),
    (9, 2, 2, 33, 8, [3, 4], 0), (5, 1, 1, 1, 8, [], 0), (40, 6, 3, 7, 16, [1], 0),
    (300, 12, 4, 128, 64, [24, 20, 20], 1)])
def test_append(om, ctx, type, T, heads, kv, D, page, pairs, halves):
    rng = np.random.default_rng(T * D)
    n_pages = -(-T // page) + 2
    c = Cache(om, ctx, type, n_pages, page, kv, D, seed=T, ks=0.5 if type == "e4m3" else 0,
              vs=2.0 if type == "e4m3" else 0)
    q = rng.standard_normal((T, heads, D)).astype(np.float32)
    k, v = ((rng.standard_normal((T, kv, D)) * 3).astype(np.float32) for _ in range(2))
    if T > 4:  # beyond the narrow types' range
        v[1, 0, 0], v[2, 0, 0], v[3, 0, 0] = 1e6, -np.inf, np.nan
    slots = i32(rng.permutation(n_pages * page)[:T])
    if T > 1:
        slots[T // 2] = -1
    pos = i32(rng.integers(0, 100000, (max(1, len(pairs)), T)))
    rope = om.rope_axes(pairs, 1e4, halves) if pairs else None
    bufs = [ctx.upload(x) for x in (k, v, slots, pos)]
    qb = ctx.upload(q) if heads and pairs else None
    qo = ctx.alloc(q.nbytes) if qb else None
    om.kv_append(ctx, c.pages, bufs[0], bufs[1], T, bufs[2], qo, qb, heads if qb else 0,
                 bufs[3] if rope else None, rope)
    got_k, got_v = c.read()
    want_k, tol = rope64(k, pos, pairs, 1e4, halves, 0) if pairs else (k.astype(np.float64),
                                                                      np.zeros(k.shape))
    on = slots >= 0
    at = torch.as_tensor(slots[on].astype(np.int64))
    # V is the conversion itself, and every other slot is as it was
    c.v[at // page, :, at % page] = stored(v[on], type, c.vs)
    if type == "e4m3" and T > 4:  # torch's clamp keeps the NaN, as the cache does
        assert np.isnan(value(c.v)).sum() == np.isnan(v[on]).sum()
    nan = torch.isnan(c.v.float())
    assert torch.equal(torch.isnan(got_v.float()), nan)
    assert same(torch.where(nan, torch.zeros(()), got_v.float()),
                torch.where(nan, torch.zeros(()), c.v.float()))
    half, small = STEP[type]
    err = np.abs(value(got_k[at // page, :, at % page], c.ks) - want_k[on])
    assert (err <= tol[on] * (1 + 2 * half) + np.maximum(np.abs(want_k[on]) * half, small * c.ks)).all()
    got_k[at // page, :, at % page] = c.k[at // page, :, at % page]
    assert same(got_k, c.k)
    if qb:
        want, tol = rope64(q, pos, pairs, 1e4, halves, 0)
        assert (np.abs(ctx.download(qo, np.float32, q.shape) - want) <= tol).all()
        qb.free()
        qo.free()
    for b in bufs:
        b.free()
    c.free()


def tables(rng, lens, page, n_pages, width, junk=-7):
    """Pages drawn without repetition; entries past a length are junk."""
    ids = rng.permutation(n_pages)
    t = np.full((len(lens), width), junk, np.int32)
    n = 0
    for b, length in enumerate(lens):
        m = -(-length // page)
        t[b, :m] = ids[n:n + m]
        n += m
    return t


def attend(om, ctx, c, q, lens, table, scale=0.0, score=None, decay=1.0, max_len=0, flags=0):
    """One call; returns out and, with score [B][kv][stride], the new scores."""
    B, H, D = q.shape
    bufs = [ctx.upload(q), ctx.alloc(q.nbytes), ctx.upload(i32(table) if table.size else i32([0])),
            ctx.upload(i32(lens))]
    o = om.attend_opts(scale=scale, max_len=max_len, flags=flags)
    if score is not None:
        si, so = ctx.upload(score), ctx.upload(np.full_like(score, -9.0))
        o = om.attend_opts(scale=scale, max_len=max_len, flags=flags, score_in=si, score_out=so,
                           score_stride=score.shape[2], decay=decay)
        bufs += [si, so]
    try:
        om.kv_attend(ctx, c.pages, bufs[1], bufs[0], B, H, bufs[2], table.shape[1], bufs[3], o)
        out = ctx.download(bufs[1], np.float32, q.shape)
        return (out, ctx.download(bufs[5], np.float32, score.shape)) if score is not None else out
    finally:
        for b in bufs:
            b.free()


def check_attend(om, ctx, c, q, lens, table, scale=0.0, with_score=True, decay=0.75, max_len=0):
    B, H, D = q.shape
    kv, width = c.k.shape[1], table.shape[1] * c.page
    rng = np.random.default_rng(1)
    score = rng.uniform(0, 2, (B, kv, width + 3)).astype(np.float32) if with_score else None
    got = attend(om, ctx, c, q, lens, table, scale, score, decay, max_len)
    out, sc = got if with_score else (got, None)
    for b, n in enumerate(lens):
        k, v = c.rows(table[b], n) if n else (np.zeros((kv, 0, D)),) * 2
        want, w, tol, tw = attend64(q[b], k, v, scale or 1 / math.sqrt(D))
        assert np.abs(out[b] - want).max() <= tol, (b, n, np.abs(out[b] - want).max(), tol)
        if with_score:
            add = w.reshape(kv, H // kv, n).sum(1)
            ws = decay * score[b, :, :n].astype(np.float64) + add
            assert (np.abs(sc[b, :, :n] - ws) <= (tw + EPS * H // kv) * add + 4 * EPS * np.abs(ws)).all(), (b, n)
            assert (sc[b, :, n:] == -9.0).all()
    return out


SHAPES = [  # heads, kv heads, D, page, lengths
    (16, 2, 256, 16, [37]), (16, 2, 256, 16, [1]), (8, 8, 64, 8, [0, 1, 7, 8, 9, 31, 32, 33]),
    (4, 1, 128, 32, [127, 128, 129, 0, 255, 257]), (20, 4, 80, 16, [500, 3, 64]),
    (32, 2, 96, 64, [65, 1000]), (17, 1, 192, 16, [100, 700]), (40, 1, 128, 16, [33, 300]),
    (3, 3, 33, 8, [50, 17]), (2, 1, 1, 8, [40]), (6, 2, 7, 16, [5, 90]), (5, 5, 100, 8, [130]),
    (128, 4, 64, 128, [400, 0, 129]), (12, 12, 64, 1024, [2047]), (2, 2, 250, 16, [77]),
    (4, 4, 8, 8, [3, 600]), (8, 2, 256, 16, [4100])]


@pytest.mark.gpu
@pytest.mark.parametrize("type", list(DTYPE))
@pytest.mark.parametrize("heads,kv,D,page,lens", SHAPES)
def test_attend(om, ctx, type, heads, kv, D, page, lens):
    rng = np.random.default_rng(heads * D + len(lens))
    n_pages = sum(-(-n // page) for n in lens) + 2
    ks, vs = (0.25, 1.5) if type == "e4m3" else (0, 0)
    c = Cache(om, ctx, type, n_pages, page, kv, D, seed=D, ks=ks, vs=vs)
    q = rng.standard_normal((len(lens), heads, D)).astype(np.float32)
    table = tables(rng, lens, page, n_pages, -(-max(lens) // page) + 1)
    check_attend(om, ctx, c, q, lens, table)
    check_attend(om, ctx, c, q * 4, lens, table, scale=0.3, with_score=False, max_len=max(lens))
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("type", list(DTYPE))
def test_attend_many_ragged_sequences(om, ctx, type):
    """Rows of every length, empty ones between them, more than a wave of them."""
    rng = np.random.default_rng(5)
    lens = [int(n) for n in rng.integers(0, 400, 150)]
    lens[3], lens[77], lens[149] = 0, 2500, 0
    n_pages = sum(-(-n // 16) for n in lens)
    c = Cache(om, ctx, type, n_pages, 16, 2, 64, seed=3)
    q = rng.standard_normal((150, 8, 64)).astype(np.float32)
    table = tables(rng, lens, 16, n_pages, -(-2500 // 16))
    check_attend(om, ctx, c, q, lens, table)
    check_attend(om, ctx, c, q, [0] * 150, table)
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("type", list(DTYPE))
@pytest.mark.parametrize("heads,D", [(8, 128), (3, 33), (8, 256)])
def test_attend_leaves_masked_slots_out(om, ctx, type, heads, D):
    """NaN and infinities behind a sequence's last token, in its last page and the others'."""
    lens = [1, 13, 40, 0, 160]
    rng = np.random.default_rng(7)
    c = Cache(om, ctx, type, 30, 16, 1, D, seed=1)
    table = tables(rng, lens, 16, 30, 11)
    used = torch.zeros(30, 16, dtype=torch.bool)
    for b, n in enumerate(lens):
        for t in range(n):
            used[table[b, t // 16], t % 16] = True
    junk = torch.tensor([math.nan, math.inf, -math.inf]) if type != "e4m3" else torch.tensor([math.nan])
    for x in (c.k, c.v):
        y = x.float()
        j = junk[torch.arange(y.numel()) % len(junk)].view(y.shape)
        x.copy_(torch.where(used[:, None, :, None], y, j).to(x.dtype))
    c.write()
    q = rng.standard_normal((5, heads, D)).astype(np.float32)
    check_attend(om, ctx, c, q, lens, table)
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,D", [(8, 128), (4, 33)])
def test_attend_values_that_are_not_finite(om, ctx, type, heads, D):
    """What 32-bit arithmetic gives: a key whose score is -inf has no weight, an infinite value
    makes its dimension infinite and no other, a NaN key makes its sequence NaN."""
    rng = np.random.default_rng(9)
    lens = [70, 70, 70, 70]
    c = Cache(om, ctx, type, 20, 16, 1, D, seed=2)
    table = tables(rng, lens, 16, 20, 5)
    q = np.abs(rng.standard_normal((4, heads, D))).astype(np.float32) + 0.5
    c.k[table[0, 1], 0, 3, 5] = -math.inf   # sequence 0: token 19
    c.v[table[0, 1], 0, 3] = 5.0
    c.v[table[1, 2], 0, 1, 4] = math.inf    # sequence 1: token 33, dimension 4
    c.k[table[2, 4], 0, 2, 0] = math.nan    # sequence 2: token 66
    c.write()
    out = attend(om, ctx, c, q, lens, table)
    for b in (0, 1, 3):
        k, v = c.rows(table[b], 70)
        if b == 0:
            k, v = np.delete(k, 19, 1), np.delete(v, 19, 1)
        fin = np.delete(np.arange(D), 4) if b == 1 else np.arange(D)
        want, _, tol, _ = attend64(q[b], k, v[..., fin] if b == 1 else v, 1 / math.sqrt(D)) \
            if b != 1 else attend64_cols(q[b], k, v, fin)
        assert np.abs(out[b][:, fin] - want).max() <= tol, b
    assert np.isposinf(out[1][:, 4]).all()
    assert np.isnan(out[2]).all()
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("type", list(DTYPE))
@pytest.mark.parametrize("n,bad", [(1, 0), (40, 17), (300, 299), (5000, 3)])
def test_attend_one_nan_key_makes_its_sequence_nan(om, ctx, type, n, bad):
    """Also where every score is one, and in a part that another group joins; a key of -inf
    alone leaves a sequence without weights: zeros."""
    rng = np.random.default_rng(n)
    lens = [n, n, 1]
    n_pages = sum(-(-m // 16) for m in lens)
    c = Cache(om, ctx, type, n_pages, 16, 1, 64, seed=2)
    table = tables(rng, lens, 16, n_pages, -(-n // 16))
    c.k[table[0, bad // 16], 0, bad % 16, 0] = math.nan
    if type != "e4m3":
        c.k[table[2, 0], 0, 0] = -math.inf
    c.write()
    q = np.abs(rng.standard_normal((3, 4, 64))).astype(np.float32) + 0.25
    out = attend(om, ctx, c, q, lens, table)
    assert np.isnan(out[0]).all()
    k, v = c.rows(table[1], n)
    want, _, tol, _ = attend64(q[1], k, v, 1 / 8)
    assert np.abs(out[1] - want).max() <= tol
    if type != "e4m3":
        assert (out[2] == 0).all()
    c.free()


def attend64_cols(q, k, v, cols):
    out, w, tol, tw = attend64(q, k, np.where(np.isfinite(v), v, 0.0), 1 / math.sqrt(q.shape[1]))
    return out[:, cols], w, tol, tw


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_attend_wide_ranges(om, ctx, type):
    """A small part of the query beside a large one decides (the large one meets zeros), and
    values of very different size: nothing may be lost that 32 bits keep."""
    rng = np.random.default_rng(11)
    D, n = 128, 300
    c = Cache(om, ctx, type, 20, 16, 1, D, seed=4)
    c.k[..., 0] = 0.0
    c.v[..., 1] *= 2.0 ** -20
    c.write()
    table = tables(rng, [n], 16, 20, 19)
    q = rng.standard_normal((1, 4, D)).astype(np.float32)
    q[:, :, 0] = np.float32(2.0) ** np.array([20, 45, 60, 100], np.float32)
    k, v = c.rows(table[0], n)
    out = attend(om, ctx, c, q, [n], table)
    q0 = q[0].copy()
    q0[:, 0] = 0.0
    want, _, _, tw = attend64(q0, k, v, 1 / math.sqrt(D))
    for d in range(D):  # every dimension by its own size
        lim = (tw + 6 * math.sqrt(n) * EPS) * np.abs(v[..., d]).max()
        assert np.abs(out[0][:, d] - want[:, d]).max() <= lim, d
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("type", list(DTYPE))
def test_attend_large_and_growing_scores(om, ctx, type):
    """Scores far above the exponential's range that grow with the token: the last ones count."""
    rng = np.random.default_rng(13)
    D, n = 64, 700
    c = Cache(om, ctx, type, 50, 16, 1, D, seed=6)
    table = tables(rng, [n], 16, 50, 44)
    for t in range(n):
        c.k[table[0, t // 16], 0, t % 16, 0] = float(stored([t / 8.0], type).float())
    c.write()
    q = rng.standard_normal((1, 3, D)).astype(np.float32)
    q[0, :, 0] = [40.0, -40.0, 0.0]
    check_attend(om, ctx, c, q, [n], table)
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("n,kv,G,pages", [(140, 2, 3, 30), (180, 2, 4, 30), (300, 2, 1, 30),
                                          (700, 2, 4, 30), (3000, 4, 2, 64), (150, 2, 4, 1),
                                          (700, 1, 5, 1)])
def test_attend_many_rows(om, ctx, n, kv, G, pages):
    """More rows than are looked at together; at 3000 x 4 heads over a table of 65,536 tokens
    the units of the work are larger, too.  Rows share pages and have junk behind their last."""
    rng = np.random.default_rng(n)
    c = Cache(om, ctx, "bf16", 9, 1024, kv, 64, seed=n)
    lens = [int(x) for x in rng.integers(0, 700, n)]
    lens[5], lens[n - 1], lens[n // 2] = (5000, 0, 9000) if pages > 1 else (1024, 0, 1)
    table = np.full((n, pages), -1, np.int32)
    table[:, 0] = rng.integers(0, 9, n)
    for b in (5, n // 2):
        table[b, :9] = rng.permutation(9)[:pages]
    q = rng.standard_normal((n, kv * G, 64)).astype(np.float32)
    score = rng.uniform(0, 1, (n, kv, 9001)).astype(np.float32) if n < 1000 else None
    got = attend(om, ctx, c, q, lens, table, score=score, max_len=max(lens) if n < 1000 else 0)
    out = got[0] if score is not None else got
    for b in range(n) if n < 1000 else list(range(0, n, 97)) + [5, 255, 256, 257, 511, 512, n // 2, n - 1]:
        k, v = c.rows(table[b], lens[b]) if lens[b] else (np.zeros((kv, 0, 64)),) * 2
        want, w, tol, tw = attend64(q[b], k, v, 1 / 8)
        assert np.abs(out[b] - want).max() <= tol, (b, lens[b])
        if score is not None:
            add = w.reshape(kv, G, -1).sum(1)
            ws = score[b, :, :lens[b]] + add
            assert (np.abs(got[1][b, :, :lens[b]] - ws) <= (tw + EPS * G) * add + 4 * EPS * np.abs(ws)).all()
            assert (got[1][b, :, lens[b]:] == -9.0).all()
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("type,n_pages", [("f32", 600), ("bf16", 1200), ("e4m3", 2200)])
def test_pages_past_4_gb(om, ctx, type, n_pages):
    """Append, attention and eviction in the last pages of a cache of over 4 GB."""
    rng = np.random.default_rng(3)
    kv, D, page = 8, 256, 1024
    nbytes = n_pages * kv * page * D * DTYPE[type].itemsize
    assert nbytes > 1 << 32
    K, V = ctx.alloc(nbytes), ctx.alloc(nbytes)
    pages = om.kv_pages(K, V, type, n_pages, page, kv, D)
    n, far = 1500, n_pages - 3
    table = i32([[n_pages - 1, far]])
    k, v = (rng.standard_normal((n, kv, D)).astype(np.float32) for _ in range(2))
    slots = i32([table[0, t // page] * page + t % page for t in range(n)])
    q = rng.standard_normal((1, 16, D)).astype(np.float32)
    bufs = [ctx.upload(x) for x in (k, v, slots, q, np.zeros_like(q), table, i32([n]),
                                    np.zeros((1, kv, 2048), np.float32), i32([[n_pages - 2]]), i32([0]),
                                    np.zeros((1, kv, 400), np.int32))]
    kb, vb, sb, qb, ob, tb, lb, scb, dt, dl, kept = bufs
    om.kv_append(ctx, pages, kb, vb, n, sb)
    om.kv_attend(ctx, pages, ob, qb, 1, 16, tb, 2, lb,
                 om.attend_opts(score_out=scb, score_stride=2048))
    kk, vv = (value(stored(x, type)).transpose(1, 0, 2) for x in (k, v))
    want, w, tol, tw = attend64(q[0], kk, vv, 1 / 16)
    assert np.abs(ctx.download(ob, np.float32, q.shape)[0] - want).max() <= tol
    score = ctx.download(scb, np.float32, (1, kv, 2048))
    om.kv_evict(ctx, pages, 1, tb, 2, lb, scb, 2048, dt, 1, dl, None, 0, kept, om.evict_opts(400, 4, 50))
    ids = ctx.download(kept, np.int32, (1, kv, 400))
    om.kv_attend(ctx, pages, ob, qb, 1, 16, dt, 1, dl)
    for h in range(kv):
        assert ids[0, h].tolist() == choose(score[0, h], n, 400, 4, 50)
    k2, v2 = (np.stack([x[h][ids[0, h]] for h in range(kv)]) for x in (kk, vv))
    want, _, tol, _ = attend64(q[0], k2, v2, 1 / 16)
    assert np.abs(ctx.download(ob, np.float32, q.shape)[0] - want).max() <= tol
    for b in bufs + [K, V]:
        b.free()


@pytest.mark.gpu
@pytest.mark.parametrize("stride", [64, 67])
@pytest.mark.parametrize("fresh", [0, 1, 3, 50, 2 ** 31 - 1])
def test_attend_tokens_without_a_score(om, ctx, fresh, stride):
    """The last tokens' score_in holds anything, also a NaN."""
    rng = np.random.default_rng(fresh % 97)
    lens = [1, 2, 40, 61, 0]
    c = Cache(om, ctx, "bf16", 20, 16, 2, 64, seed=4)
    table = tables(rng, lens, 16, 20, 4)
    q = rng.standard_normal((5, 4, 64)).astype(np.float32)
    score = rng.uniform(0, 1, (5, 2, stride)).astype(np.float32)
    for b, n in enumerate(lens):
        score[b, :, max(n - fresh, 0):n] = np.nan
    bufs = [ctx.upload(x) for x in (q, np.zeros_like(q), table, i32(lens), score)]
    om.kv_attend(ctx, c.pages, bufs[1], bufs[0], 5, 4, bufs[2], 4, bufs[3],
                 om.attend_opts(score_in=bufs[4], score_out=bufs[4], score_stride=stride, decay=0.5,
                                score_new=fresh))
    got = ctx.download(bufs[4], np.float32, score.shape)
    for b, n in enumerate(lens):
        k, v = c.rows(table[b], n) if n else (np.zeros((2, 0, 64)),) * 2
        _, w, _, tw = attend64(q[b], k, v, 1 / 8)
        add = w.reshape(2, 2, n).sum(1)
        ws = add + 0.5 * np.nan_to_num(score[b, :, :n].astype(np.float64))
        assert (np.abs(got[b, :, :n] - ws) <= (tw + EPS * 2) * add + 4 * EPS * np.abs(ws)).all()
        assert same(torch.tensor(got[b, :, n:]), torch.tensor(score[b, :, n:]))
    for b in bufs:
        b.free()
    c.free()


@pytest.mark.gpu
def test_decode_loop_without_the_host(om, ctx):
    """Lengths, slots and positions of all steps are there beforehand; nothing is read back
    until the end, and the scores live on the device only."""
    rng = np.random.default_rng(41)
    B, H, kv, D, page, width, steps = 2, 4, 2, 64, 16, 3, 40
    keep, full = 20, 30
    c = Cache(om, ctx, "f32", B * width, page, kv, D, seed=1)
    table = i32(rng.permutation(B * width).reshape(B, width))
    tb, junk = ctx.upload(table), np.full((B, kv, width * page), np.nan, np.float32)
    sb, kept = ctx.upload(junk), ctx.upload(np.zeros((B, kv, keep), np.int32))
    rope = om.rope_axes([D // 2], 1e4)
    lens, outs, bufs = [0, 0], [], []
    cache = [[[] for _ in range(kv)] for _ in range(B)]  # key, value, score, its tolerance
    for step in range(steps):
        q = rng.standard_normal((B, H, D)).astype(np.float32)
        k, v = (rng.standard_normal((B, kv, D)).astype(np.float32) for _ in range(2))
        slots = i32([table[b, lens[b] // page] * page + lens[b] % page for b in range(B)])
        lens = [n + 1 for n in lens]
        x = [ctx.upload(y) for y in (q, k, v, slots, i32([step] * B), i32(lens), np.zeros_like(q))]
        bufs += x
        om.kv_append(ctx, c.pages, x[1], x[2], B, x[3], x[0], x[0], H, x[4], rope, flags=om.KV_ASYNC)
        om.kv_attend(ctx, c.pages, x[6], x[0], B, H, tb, width, x[5],
                     om.attend_opts(flags=om.KV_ASYNC, score_in=sb, score_out=sb, score_new=1,
                                    score_stride=width * page))
        q64, k64 = (rope64(y, np.array([[step] * B]), [D // 2], 1e4, 0, 0)[0] for y in (q, k))
        want, tol = np.zeros((B, H, D)), 0.0
        for b in range(B):
            for h in range(kv):
                cache[b][h].append([k64[b, h], v[b, h].astype(np.float64), 0.0, 0.0])
                kk, vv = (np.stack([t[i] for t in cache[b][h]])[None] for i in (0, 1))
                g = slice(h * H // kv, (h + 1) * H // kv)
                want[b, g], w, t1, tw = attend64(q64[b, g], kk, vv, 1 / 8)
                # the rotations of q and k are off by 6 e (|u| + |v|) each
                extra = 24 * EPS * np.abs(kk).max() * np.abs(q64[b, g]).max() * D / 8
                tol = max(tol, t1 + 2 * extra * np.abs(vv).max())
                for t, add in zip(cache[b][h], w.sum(0)):
                    t[2] += add
                    t[3] += (tw + 2 * extra + 2 * EPS) * add + 2 * EPS * t[2]
        outs.append((x[6], want, tol))
        if lens[0] == full:
            om.kv_evict(ctx, c.pages, B, tb, width, x[5], sb, width * page, tb, width, x[5], sb,
                        width * page, kept, om.evict_opts(keep, 2, 6, flags=om.KV_ASYNC))
            for b in range(B):
                for h in range(kv):
                    s = np.array([t[2] for t in cache[b][h]])
                    mid = np.sort(s[2:full - 6])[::-1]
                    off = max(t[3] for t in cache[b][h])
                    assert mid[keep - 9] - mid[keep - 8] > 2 * off  # rounding does not choose
                    cache[b][h] = [cache[b][h][i] for i in choose(s.astype(np.float32), full, keep, 2, 6)]
            lens = [keep] * B
    assert om.lib().gpu_kv_check(ctx.ptr) == 0
    for o, want, tol in outs:
        assert np.abs(ctx.download(o, np.float32, want.shape) - want).max() <= tol
    got = ctx.download(sb, np.float32, junk.shape)
    for b in range(B):
        for h in range(kv):
            assert (np.abs(got[b, h, :lens[b]] - [t[2] for t in cache[b][h]]) <= [t[3] for t in cache[b][h]]).all()
    for b in bufs + [tb, sb, kept]:
        b.free()
    c.free()


@pytest.mark.gpu
def test_two_contexts_at_once(om):
    """Asynchronous calls of two contexts, each with its stream and workspace, on pages that
    both read."""
    rng = np.random.default_rng(31)
    one, two = om.Context(), om.Context()
    c = Cache(om, one, "bf16", 300, 16, 2, 128, seed=10)
    table = tables(rng, [4000], 16, 300, 250)
    q = rng.standard_normal((2, 1, 8, 128)).astype(np.float32)
    s = rng.uniform(0, 1, (1, 2, 4000)).astype(np.float32)
    alone = [attend(om, one, c, q[i], [4000], table, score=s) for i in (0, 1)]
    jobs = []
    for x, i in ((one, 0), (two, 1)):
        b = [x.upload(y) for y in (q[i], np.zeros_like(q[i]), table, i32([4000]), s, np.zeros_like(s))]
        jobs.append((x, b, om.attend_opts(flags=om.KV_ASYNC, score_in=b[4], score_out=b[5],
                                          score_stride=4000)))
    for _ in range(5):
        for x, b, o in jobs:
            om.kv_attend(x, c.pages, b[1], b[0], 1, 8, b[2], 250, b[3], o)
    for i, (x, b, _) in enumerate(jobs):
        assert om.lib().gpu_kv_check(x.ptr) == 0
        assert np.array_equal(x.download(b[1], np.float32, q[i].shape), alone[i][0])
        assert np.array_equal(x.download(b[5], np.float32, s.shape), alone[i][1])
    two.close()
    c.free()
    one.close()


@pytest.mark.gpu
def test_attend_scale_zero_is_the_default_and_uniform_weights(om, ctx):
    """Equal keys: every token has the weight 1 / n, and the scores of a kv head add up to its
    query heads."""
    c = Cache(om, ctx, "bf16", 40, 16, 1, 64, seed=8)
    c.k[:] = 1.0
    c.write()
    rng = np.random.default_rng(0)
    table = tables(rng, [513], 16, 40, 33)
    q = np.ones((1, 6, 64), np.float32)
    out, sc = attend(om, ctx, c, q, [513], table, score=np.zeros((1, 1, 528), np.float32))
    _, v = c.rows(table[0], 513)
    assert np.abs(out[0] - v[0].mean(0)).max() <= 64 * EPS
    assert np.abs(sc[0, 0, :513] - 6 / 513).max() <= 16 * EPS
    c.free()


@pytest.mark.gpu
def test_attend_shared_pages_and_scores_in_place(om, ctx):
    """Two sequences with a common prefix in the same pages; scores in one buffer."""
    rng = np.random.default_rng(15)
    c = Cache(om, ctx, "f16", 12, 16, 2, 64, seed=9)
    table = i32([[3, 5, 7, 1], [3, 5, 2, 9]])
    lens = [64, 50]
    q = rng.standard_normal((2, 4, 64)).astype(np.float32)
    check_attend(om, ctx, c, q, lens, table)
    score = rng.uniform(0, 1, (2, 2, 64)).astype(np.float32)
    want = attend(om, ctx, c, q, lens, table, score=score)[1]
    sb, bufs = ctx.upload(score), [ctx.upload(x) for x in (q, np.zeros_like(q), table, i32(lens))]
    o = om.attend_opts(score_in=sb, score_out=sb, score_stride=64)
    om.kv_attend(ctx, c.pages, bufs[1], bufs[0], 2, 4, bufs[2], 4, bufs[3], o)
    got = ctx.download(sb, np.float32, score.shape)
    for b, n in enumerate(lens):
        assert np.array_equal(got[b, :, :n], want[b, :, :n])
        assert np.array_equal(got[b, :, n:], score[b, :, n:])
    for b in bufs + [sb]:
        b.free()
    c.free()


@pytest.mark.gpu
def test_calls_in_a_row_do_not_wait_for_each_other(om, ctx):
    """Asynchronous calls of growing and shrinking size on one workspace: each gives what it
    gives alone, and again the same bits."""
    rng = np.random.default_rng(17)
    c = Cache(om, ctx, "bf16", 300, 16, 2, 128, seed=10)
    alone, jobs = [], []
    for n in (40, 4000, 7, 1000):
        table = tables(rng, [n], 16, 300, 250)
        q = rng.standard_normal((1, 8, 128)).astype(np.float32)
        s = rng.uniform(0, 1, (1, 2, 4000)).astype(np.float32)
        alone.append(attend(om, ctx, c, q, [n], table, score=s))
        b = [ctx.upload(x) for x in (q, np.zeros_like(q), table, i32([n]), s, np.full_like(s, -9.0))]
        jobs.append((b, om.attend_opts(flags=om.KV_ASYNC, score_in=b[4], score_out=b[5],
                                       score_stride=4000)))
    for b, o in jobs:
        om.kv_attend(ctx, c.pages, b[1], b[0], 1, 8, b[2], 250, b[3], o)
    assert om.lib().gpu_kv_check(ctx.ptr) == 0
    for (b, _), (out, sc) in zip(jobs, alone):
        assert np.array_equal(ctx.download(b[1], np.float32, out.shape), out)
        assert np.array_equal(ctx.download(b[5], np.float32, sc.shape), sc)
        for x in b:
            x.free()
    c.free()


def evict(om, ctx, c, lens, table, score, keep, sink, recent, dst=None, in_place=False):
    """One call; dst: the destination table (None with in_place)."""
    B, kv, stride = score.shape
    b = dict(table=ctx.upload(i32(table)), lens=ctx.upload(i32(lens)), score=ctx.upload(score),
             kept=ctx.upload(np.full((B, kv, keep), -5, np.int32)))
    own = dict(b)
    if in_place:
        b.update(dst=b["table"], dl=b["lens"], ds=b["score"])
        dp, dstride = table.shape[1], stride
    else:
        dp, dstride = dst.shape[1], keep + 2
        new = dict(dst=ctx.upload(i32(dst)), dl=ctx.alloc(4 * B),
                   ds=ctx.upload(np.full((B, kv, dstride), -9.0, np.float32)))
        b.update(new)
        own.update(new)
    try:
        om.kv_evict(ctx, c.pages, B, b["table"], table.shape[1], b["lens"], b["score"], stride,
                    b["dst"], dp, b["dl"], b["ds"], dstride, b["kept"],
                    om.evict_opts(keep, sink, recent))
        return (ctx.download(b["kept"], np.int32, (B, kv, keep)), ctx.download(b["dl"], np.int32, (B,)),
                ctx.download(b["ds"], np.float32, (B, kv, dstride)))
    finally:
        for x in own.values():
            x.free()


def check_evict(om, ctx, c, lens, table, score, keep, sink, recent, dst=None):
    """Against the definition; c's tensors follow the device's."""
    in_place = dst is None
    kept, dl, ds = evict(om, ctx, c, lens, table, score, keep, sink, recent, dst, in_place)
    to = table if in_place else dst
    k, v = c.k.clone(), c.v.clone()
    fill = -9.0 if not in_place else None
    for b, n in enumerate(lens):
        m = min(n, keep)
        assert dl[b] == m
        for h in range(score.shape[1]):
            want = choose(score[b, h], n, keep, sink, recent)
            assert kept[b, h].tolist() == want + [-1] * (keep - m), (b, h)
            rest = np.full(ds.shape[2] - m, fill, np.float32) if fill else score[b, h, m:]
            both = np.concatenate([score[b, h, want], rest])
            assert np.array_equal(ds[b, h].view(np.uint32), both.astype(np.float32).view(np.uint32))
            for j, i in enumerate(want):
                for x, y in ((k, c.k), (v, c.v)):
                    x[to[b, j // c.page], h, j % c.page] = y[table[b, i // c.page], h, i % c.page]
    got_k, got_v = c.read()
    assert same(got_k, k) and same(got_v, v)  # nothing else has changed
    c.k, c.v = k, v
    return kept, dl, ds


EVICTS = [  # kv, D, page, lengths, keep, sink, recent
    (2, 64, 16, [100, 0, 20, 1, 21], 20, 4, 6), (1, 256, 16, [700], 350, 4, 64),
    (3, 33, 8, [90, 41], 40, 0, 0), (1, 1, 8, [50], 1, 0, 0), (2, 7, 16, [64, 65], 64, 64, 0),
    (1, 128, 32, [300, 299], 40, 0, 40), (4, 80, 64, [2500, 130, 1025], 1000, 10, 100),
    (1, 8, 8, [5000], 4999, 1, 1), (2, 8, 64, [17000, 16384], 4000, 0, 9), (1, 4, 128, [70001], 20000, 2, 2), (2, 96, 16, [33], 500, 3, 3), (1, 4, 1024, [9000], 3001, 5, 7)]


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("type", list(DTYPE))
@pytest.mark.parametrize("kv,D,page,lens,keep,sink,recent", EVICTS)
def test_evict(om, ctx, type, kv, D, page, lens, keep, sink, recent, in_place):
    rng = np.random.default_rng(D + keep)
    width, new = -(-max(lens) // page), -(-keep // page)
    used = sum(-(-n // page) for n in lens)
    n_pages = used + len(lens) * new + 1
    c = Cache(om, ctx, type, n_pages, page, kv, D, seed=keep)
    ids = rng.permutation(n_pages)
    table = np.full((len(lens), width), -3, np.int32)
    n = 0
    for b, length in enumerate(lens):
        table[b, :-(-length // page)] = ids[n:n - (-length // page)]
        n -= -length // page
    dst = None if in_place else ids[used:used + len(lens) * new].reshape(len(lens), new)
    score = np.exp(2 * rng.standard_normal((len(lens), kv, width * page + 5))).astype(np.float32)
    score[rng.random(score.shape) < 0.3] = 0.0       # ties
    score[..., ::7] = np.float32(0.125)              # more of them
    score[rng.random(score.shape) < 0.02] = -0.0
    score[rng.random(score.shape) < 0.01] = np.nan   # the lowest
    score[rng.random(score.shape) < 0.01] = -1.5
    score[rng.random(score.shape) < 0.005] = np.inf
    check_evict(om, ctx, c, lens, table, score, keep, sink, recent, dst)
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("fill", [0.0, 1.0, -np.inf, np.nan])
def test_evict_equal_scores_keep_the_first(om, ctx, fill):
    c = Cache(om, ctx, "bf16", 200, 16, 1, 64, seed=1)
    table = tables(np.random.default_rng(1), [1500], 16, 200, 94)
    score = np.full((1, 1, 1504), fill, np.float32)
    kept, _, _ = check_evict(om, ctx, c, [1500], table, score, 600, 3, 50)
    assert kept[0, 0, :550].tolist() == list(range(550))
    c.free()


@pytest.mark.gpu
def test_numbers_out_of_range(om, ctx):
    """Pages, slots and lengths outside their bounds: reported, left out, and nothing else
    touched."""
    rng = np.random.default_rng(21)
    c = Cache(om, ctx, "f16", 12, 16, 1, 64, seed=5)
    q = rng.standard_normal((2, 4, 64)).astype(np.float32)
    good = tables(rng, [60, 60], 16, 12, 4)
    for bad in (-1, 12, 2 ** 31 - 1, -2 ** 31):
        table = good.copy()
        table[1, 2] = bad
        with pytest.raises(RuntimeError, match="page number of row 1"):
            attend(om, ctx, c, q, [60, 60], table)
        assert om.lib().gpu_kv_check(ctx.ptr) == 0
        # asynchronous: the others' results are there, the report comes after
        b = [ctx.upload(x) for x in (q, np.zeros_like(q), table, i32([60, 60]))]
        om.kv_attend(ctx, c.pages, b[1], b[0], 2, 4, b[2], 4, b[3], om.attend_opts(flags=om.KV_ASYNC))
        assert om.lib().gpu_kv_check(ctx.ptr) == -1 and "row 1" in ctx.last_error()
        out = ctx.download(b[1], np.float32, q.shape)
        for row, on in ((0, np.arange(60)), (1, np.r_[0:32, 48:60])):
            k, v = c.rows(good[row], 60)
            want, _, tol, _ = attend64(q[row], k[:, on], v[:, on], 1 / 8)
            assert np.abs(out[row] - want).max() <= tol
        for x in b:
            x.free()
    for lens in ([60, 65], [60, -1], [60, 2 ** 31 - 1], [-2 ** 31, 60]):
        with pytest.raises(RuntimeError, match="the length of sequence"):
            attend(om, ctx, c, q, lens, good)
    with pytest.raises(RuntimeError, match="the length of sequence"):
        attend(om, ctx, c, q, [41, 40], good, max_len=40)
    score = np.zeros((2, 1, 64), np.float32)
    table = good.copy()
    table[0, 1] = 99
    with pytest.raises(RuntimeError, match="page number of row 0"):
        evict(om, ctx, c, [60, 60], table, score, 30, 0, 30, in_place=True)
    c.write()
    with pytest.raises(RuntimeError, match="the length of sequence 1"):
        evict(om, ctx, c, [60, 70], good, score, 64, 0, 0, in_place=True)
    c.write()
    kb = [ctx.upload(x) for x in (np.ones((3, 1, 64), np.float32), i32([5, 192, -2]))]
    with pytest.raises(RuntimeError, match="slot of token"):
        om.kv_append(ctx, c.pages, kb[0], kb[0], 3, kb[1])
    c.k[0, :, 5] = c.v[0, :, 5] = 1.0
    got = c.read()
    assert same(got[0], c.k) and same(got[1], c.v)
    for x in kb:
        x.free()
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f32", "bf16", "e4m3"])
def test_decode_steps(om, ctx, type):
    """An engine's loop: every step rotates and appends a token of each sequence, attends over
    its pages, adds the weights up, and cuts a cache that is full to the tokens that took most
    of the weight, in its own pages."""
    rng = np.random.default_rng(23)
    B, H, kv, D, page, width = 3, 8, 2, 64, 8, 6
    full, keep, sink, recent = 40, 24, 2, 8
    c = Cache(om, ctx, type, B * width + 1, page, kv, D, seed=7)
    table = i32(rng.permutation(B * width + 1)[:B * width].reshape(B, width))
    rope, stride = om.rope_axes([12, 10, 10], 1e4, halves=True, interleaved=True), width * page
    lens, score = [0, 3, 20], np.zeros((B, kv, stride), np.float32)
    tb, sb = ctx.upload(table), ctx.upload(score)
    pos0 = 1000
    for step in range(60):
        q = rng.standard_normal((B, H, D)).astype(np.float32)
        k, v = (rng.standard_normal((B, kv, D)).astype(np.float32) for _ in range(2))
        slots = i32([table[b, lens[b] // page] * page + lens[b] % page for b in range(B)])
        if step % 5 == 4:
            slots[1] = -1  # this sequence waits
        pos = i32(pos0 + step + rng.integers(0, 3, (3, B)))
        lens = [n + (s >= 0) for n, s in zip(lens, slots)]
        for b in range(B):
            if slots[b] >= 0:
                score[b, :, lens[b] - 1] = 0.0
        om.lib().gpu_copy_to_device(ctx.ptr, sb.ptr, om._p(score), score.nbytes)
        bufs = [ctx.upload(x) for x in (q, k, v, slots, pos, i32(lens), np.zeros_like(q),
                                        np.zeros((B, kv, keep), np.int32))]
        qb, kb, vb, sl, pb, lb, ob, keptb = bufs
        om.kv_append(ctx, c.pages, kb, vb, B, sl, qb, qb, H, pb, rope, flags=om.KV_ASYNC)
        om.kv_attend(ctx, c.pages, ob, qb, B, H, tb, width, lb,
                     om.attend_opts(flags=om.KV_ASYNC, score_in=sb, score_out=sb, score_stride=stride,
                                    decay=0.9))
        evicts = max(lens) >= full
        if evicts:
            om.kv_evict(ctx, c.pages, B, tb, width, lb, sb, stride, tb, width, lb, sb, stride, keptb,
                        om.evict_opts(keep, sink, recent, flags=om.KV_ASYNC))
        assert om.lib().gpu_kv_check(ctx.ptr) == 0
        # the append: the cache's own bits are taken for the rest, once they are near
        got_k, got_v = c.read()
        q64, _ = rope64(q, pos, [12, 10, 10], 1e4, 1, 1)
        k64, tol = rope64(k, pos, [12, 10, 10], 1e4, 1, 1)
        half, small = STEP[type]
        old_k, old_v = c.k.clone(), c.v.clone()
        for b, s in enumerate(slots):
            if s >= 0:
                c.k[s // page, :, s % page] = stored(k64[b], type)
                c.v[s // page, :, s % page] = stored(v[b], type)
        if not evicts:
            near = np.abs(value(got_k) - value(c.k))
            lim = 2 * half * np.abs(value(c.k)) + 2 * small + 12 * EPS * 8
            assert (near <= lim).all() and same(got_v, c.v)
            c.k = got_k
        out = ctx.download(ob, np.float32, q.shape)
        sc = ctx.download(sb, np.float32, score.shape)
        new = []
        for b, n in enumerate(lens):
            kk, vv = c.rows(table[b], n)
            want, w, t, tw = attend64(q64[b], kk, vv, 1 / 8)
            # a rotated query is off by 6 e (|u| + |v|), and a key just stored (on an evicting
            # step taken from the definition) by a step of its type
            extra = 24 * EPS * np.abs(kk).max() * np.abs(q64[b]).max() * D / 8
            if evicts:
                extra += 2 * half * np.abs(kk).max() * np.abs(q64[b]).max() * 8 * (half > 1e-6)
            assert np.abs(out[b] - want).max() <= t + 2 * extra * np.abs(vv).max(), (step, b)
            add = 0.9 * score[b, :, :n] + w.reshape(kv, H // kv, n).sum(1)
            if not evicts:
                assert np.abs(sc[b, :, :n] - add).max() <= 4 * (tw + extra + 4 * EPS) * 4, (step, b)
                score[b, :, :n] = sc[b, :, :n]
            new.append(add)
        if evicts:
            kept = ctx.download(keptb, np.int32, (B, kv, keep))
            dl = ctx.download(lb, np.int32, (B,))
            k2, v2 = c.k.clone(), c.v.clone()
            for b, n in enumerate(lens):
                m = min(n, keep)
                assert dl[b] == m
                for h in range(kv):
                    ids = kept[b, h, :m]
                    assert (np.diff(ids) > 0).all() and ids[0] == 0 and ids[-1] == n - 1
                    if n > keep:
                        # nobody who left had more than one who stayed, by the sums' own error
                        mid = np.arange(sink, n - recent)
                        stay = np.isin(mid, ids)
                        assert new[b][h, mid[stay]].min() >= new[b][h, mid[~stay]].max() - 0.05
                    for j, i in enumerate(ids):
                        for x, y in ((k2, got_k), (v2, got_v)):
                            old = (old_k if x is k2 else old_v) if i < n - 1 or slots[b] < 0 else \
                                (c.k if x is k2 else c.v)
                            mine = y[table[b, j // page], h, j % page]
                            src = old[table[b, i // page], h, i % page]
                            if i < n - 1 or x is v2:
                                assert same(mine, src), (step, b, h, j, i)
            c.k, c.v = got_k, got_v
            lens, score = [int(n) for n in dl], sc
        for x in bufs:
            x.free()
    tb.free()
    sb.free()
    c.free()


@pytest.mark.gpu
def test_a_layers_logits_stay_readable(om, ctx):
    """The paged cache's workspace is its own: gpu_moe_last_logits after a forward is not
    touched by calls between."""
    st = om.Store(ctx, 1, 256, 256, 16, 8, True, prefill_layout=2)
    st.fill_synthetic(0, 5)
    x = om.synth_normal(5, om.synth_stream(0, om.SYN_ACT, 0), 4 * 256, 1.0).reshape(4, 256)
    xb, ob = ctx.upload(x), ctx.alloc(x.nbytes)
    st.forward(0, xb, 4, ob)
    before = st.last_logits(4)
    rng = np.random.default_rng(1)
    c = Cache(om, ctx, "bf16", 70, 16, 1, 64, seed=5)
    q = rng.standard_normal((1, 8, 64)).astype(np.float32)
    attend(om, ctx, c, q, [1000], tables(rng, [1000], 16, 70, 64), score=np.zeros((1, 1, 1024), np.float32))
    assert np.array_equal(before, st.last_logits(4))
    st.close()
    for b in (xb, ob):
        b.free()
    c.free()

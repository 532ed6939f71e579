"""Norms of heads with the rotation (gpu_norm_rope_axes, gpu_norm_kv_append), linear
attention with decays (gpu_linear_attend) and sampling (gpu_sample).

CPU: what the host refuses (csrc/host/*.c over launches that only count).

GPU: each call against its definition in 64 bits.  With e = 2^-24 (half a step of fp32):
  norm    a sum of D squares by lanes: a chain of at most D / 64 + 8 rounded sums in a lane
          and 6 joining them, so its relative error is below (D / 64 + 14) e; the mean, eps,
          the root (which halves what came before) and the reciprocal, the two products with
          the factor and the weight round by e each, the root and the reciprocal possibly by
          2 e: below n = (D / 64 + 16) / 2 + 6 of e in all.  A rotation adds 6 e (|u| + |v|)
          (three roundings and an angle off by 2^-25 half turns).  The cache's type adds half
          a step.
  linear  an output is a sum over the earlier tokens and the key's dimensions.  Relative to
          the same sum of absolute values: every decay, of which the logarithm's sum is exact
          to 2^-40, is off by at most 4 e, products by 4 e in all, and the chains of at most
          2 L + dk sums by independent roundings, whose 6 standard deviations are below
          6 sqrt(2 L + dk) e.  Chains of decays (token by token, or chunk by chunk) round
          twice for each of L tokens: in that sum.  So is what products of bf16 parts leave
          out, less than 4 e of each and of either sign (its deviation is below e).
  sample  tokens are equal.  A weight is rounded to 2^-45 of the largest or finer at the sizes
          here (up to 2^17 tokens), a sum of n of them is off by at most n 2^-46, a border (a
          share of one) by as much: where the 64-bit sums come within n 2^-44 of a border of
          the choice, either side is right.  prob is rounded once (e) beside that.
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
STEP = {"f32": (2.0 ** -24, 2.0 ** -150), "f16": (2.0 ** -11, 2.0 ** -25),
        "bf16": (2.0 ** -8, 2.0 ** -134), "e4m3": (2.0 ** -4, 2.0 ** -10)}


@pytest.fixture(scope="module")
def om():
    import ornith_moe
    ornith_moe.lib()
    return ornith_moe


# ------------------------------------------------------------ the host, on the CPU
class Host:
    """An entry point's file over counting launches."""

    def __init__(self, om, so, prefix):
        self.om, self.L, self.prefix = om, C.CDLL(so), prefix
        real = om.lib()
        names = ["gpu_norm_rope_axes", "gpu_norm_kv_append", "gpu_kv_check"] if prefix == "kv_test" \
            else ["gpu_linear_attend", "gpu_sample"]
        for n in names:
            getattr(self.L, n).argtypes = getattr(real, n).argtypes
        for n in ("context", "buffer"):
            self._fn(n).restype = C.c_void_p
        self._fn("buffer").argtypes = [C.c_size_t]
        self._fn("error").restype = C.c_char_p
        self._fn("error").argtypes = [C.c_void_p]
        self._fn("mark").argtypes = [C.c_void_p, C.c_int, C.c_int]
        self.ctx = self._fn("context")(0)

    def _fn(self, n):
        return getattr(self.L, f"{self.prefix}_{n}")

    def int(self, n):
        return C.c_int.in_dll(self.L, n)

    def buf(self, n):
        return self._fn("buffer")(n)

    def error(self):
        return self._fn("error")(self.ctx).decode()

    def mark(self, what, at):
        self._fn("mark")(self.ctx, what, at)

    def call(self, fn, args):
        count = self.int("kv_launches" if self.prefix == "kv_test" else "decode_launches")
        n = count.value
        rc = getattr(self.L, fn)(self.ctx, *[C.byref(v) if isinstance(v, C.Structure) else v
                                             for v in args.values()])
        return rc, count.value - n


def _host(om, tmp, source, prefix):
    so = str(tmp.mktemp("host") / "host.so")
    r = subprocess.run(["gcc", "-std=gnu99", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-shared",
                        "-fPIC", "-o", so, os.path.join(HERE, source), "-lm"], capture_output=True,
                       text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    return Host(om, so, prefix)


@pytest.fixture(scope="module")
def kv_host(om, tmp_path_factory):
    return _host(om, tmp_path_factory, "kv_host.c", "kv_test")


@pytest.fixture(scope="module")
def host(om, tmp_path_factory):
    return _host(om, tmp_path_factory, "decode_host.c", "decode")


def rope_call(h, append):
    """5 tokens, 4 heads over 2 kv heads of 32."""
    om, T, H, kv, D = h.om, 5, 4, 2, 32
    norm = om.HeadNorm(0, 1e-6, h.buf(D * 4), h.buf(D * 4), 0)
    rope = om.rope_axes([4, 6, 2], 1e4)
    a = dict(q_out=h.buf(T * H * D * 4), k_out=h.buf(T * kv * D * 4), Q=h.buf(T * H * D * 4),
             K=h.buf(T * kv * D * 4), T=T, heads=H, kv=kv, D=D, norm=norm, pos=h.buf(3 * T * 4),
             rope=rope, flags=0)
    if not append:
        return "gpu_norm_rope_axes", a
    page = 9 * kv * 16 * D * 2
    pages = om.KVPages(h.buf(page), h.buf(page), om.KV_TYPES["f16"], 9, 16, kv, D, 0, 0)
    return "gpu_norm_kv_append", dict(
        pages=pages, K=a["K"], V=h.buf(T * kv * D * 4), T=T, slots=h.buf(T * 4), q_out=a["q_out"],
        Q=a["Q"], heads=H, norm=norm, pos=a["pos"], rope=rope, flags=0)


@pytest.mark.parametrize("append", [False, True])
def test_host_norms(kv_host, append):
    h = kv_host

    def call(**change):
        fn, a = rope_call(h, append)
        for k, v in change.items():
            if k in ("kind", "eps", "q_weight", "k_weight", "per_head"):
                setattr(a["norm"], k, v)
            else:
                assert k in a
                a[k] = v
        return h.call(fn, a)

    assert call() == (0, 1)
    assert call(pos=None, rope=None) == (0, 1)
    assert call(q_weight=None) == call(k_weight=None) == (0, 1)
    assert call(eps=0.0) == (0, 1)
    assert call(T=0) == (0, 0)
    assert call(per_head=1, q_weight=h.buf(4 * 32 * 4), k_weight=h.buf(2 * 32 * 4)) == (0, 1)
    for bad in (dict(norm=None), dict(kind=2), dict(kind=-1), dict(eps=-1e-6), dict(eps=math.inf),
                dict(eps=math.nan), dict(per_head=1), dict(q_weight=h.buf(31 * 4)),
                dict(k_weight=h.buf(31 * 4)), dict(pos=None), dict(rope=None), dict(T=6), dict(T=-1),
                dict(K=None), dict(Q=None), dict(heads=5), dict(heads=0),
                dict(per_head=1, q_weight=h.buf(4 * 32 * 4), k_weight=h.buf(2 * 32 * 4 - 1))):
        rc, n = call(**bad)
        assert rc < 0 and n == 0 and h.error(), bad
    # outputs that are other arguments
    big = h.buf(1 << 20)
    for bad in (dict(q_out=big, q_weight=big), dict(q_out=big, k_weight=big), dict(q_out=big, K=big),
                dict(q_out=big, pos=big)):
        assert call(**bad) == (-1, 0), bad
    assert call(q_out=big, Q=big) == (0, 1)


def test_host_norms_of_one_side(kv_host):
    h = kv_host
    fn, a = rope_call(h, False)
    a.update(K=None, k_out=None, kv=0)
    assert h.call(fn, a) == (0, 1)
    fn, a = rope_call(h, True)
    a.update(Q=None, q_out=None, heads=0)
    assert h.call(fn, a) == (0, 1)


def linear_call(h):
    """3 sequences, 7 tokens, 4 heads of 16 x 24 (2 of Q and K), 5 slots."""
    om, T, H, dk, dv = h.om, 7, 4, 16, 24
    st = om.LinearStates(h.buf(5 * H * dk * dv * 4), 5, H, dk, dv)
    opts = om.LinearOpts(0, 1, 0, 4, 0)
    return dict(st=st, out=h.buf(T * H * dv * 4), Q=h.buf(T * 2 * dk * 4), K=h.buf(T * 2 * dk * 4),
                V=h.buf(T * H * dv * 4), qh=2, kh=2, vh=4, T=T, decay=h.buf(T * H * 4), B=3,
                starts=h.buf(16), slots_in=h.buf(12), slots_out=h.buf(12), opts=opts)


def test_host_linear(host):
    h = host

    def call(**change):
        a = linear_call(h)
        for k, v in change.items():
            if k in ("S", "n_slots", "n_heads", "key_dim", "value_dim"):
                setattr(a["st"], k, v)
            elif k in ("scale", "per_token", "max_len", "flags"):
                setattr(a["opts"], k, v)
            else:
                assert k in a
                a[k] = v
        return h.call("gpu_linear_attend", a)

    assert call() == (0, 1) and h.L.decode_max_len() == 4
    assert call(max_len=0) == (0, 1) and h.L.decode_max_len() == 7
    assert call(max_len=100) == (0, 1) and h.L.decode_max_len() == 7
    assert call(opts=None, decay=h.buf(16)) == (0, 1)
    assert call(B=0) == (0, 0)
    assert call(starts=None, B=7, slots_in=h.buf(28), slots_out=h.buf(28)) == (0, 1)
    assert h.L.decode_max_len() == 1
    assert call(slots_in=None) == call(slots_out=None) == (0, 1)
    assert call(slots_in=None, slots_out=None, S=None) == (0, 1)
    same = h.buf(12)
    assert call(slots_in=same, slots_out=same) == (0, 1)
    same = h.buf(1 << 16)
    assert call(Q=same, K=same, V=same) == (0, 1)
    for bad in (dict(st=None), dict(out=None), dict(Q=None), dict(K=None), dict(V=None),
                dict(decay=None), dict(T=8), dict(T=-1), dict(B=4), dict(B=-1), dict(starts=None),
                dict(qh=4), dict(kh=4), dict(kh=3), dict(qh=0), dict(vh=8), dict(S=None),
                dict(n_slots=6), dict(n_slots=-1), dict(n_heads=8), dict(n_heads=0),
                dict(n_heads=65536), dict(key_dim=17), dict(key_dim=257), dict(key_dim=0),
                dict(value_dim=25), dict(value_dim=257), dict(value_dim=0), dict(scale=math.inf),
                dict(scale=math.nan), dict(max_len=-1), dict(starts=h.buf(12)),
                dict(slots_in=h.buf(8)), dict(slots_out=h.buf(8)), dict(B=65536),
                dict(decay=h.buf(16)), dict(T=1 << 30), dict(n_slots=1 << 30)):
        rc, n = call(**bad)
        assert rc < 0 and n == 0 and h.error().startswith("gpu_linear_attend"), bad
    big = h.buf(1 << 16)
    for o in ("Q", "K", "V", "decay", "starts", "slots_in", "slots_out"):
        assert call(**{"out": big, o: big}) == (-1, 0), o
        assert call(**{"S": big, o: big}) == (-1, 0), o
    assert call(out=big, S=big) == (-1, 0)
    h.int("decode_no_room").value = 1
    assert call() == (-2, 0)
    h.int("decode_no_room").value = 0


def test_host_sample(host):
    h = host

    def call(**change):
        a = dict(tokens=h.buf(20), prob=h.buf(20), logits=h.buf(5 * 100 * 4), rows=5, vocab=100,
                 stride=0, requests=h.buf(80), u=h.buf(20), flags=0)
        assert set(change) <= set(a)
        a.update(change)
        return h.call("gpu_sample", a)

    h.L.decode_unit.restype = C.c_double
    assert call() == (0, 1) and h.L.decode_unit() == 2.0 ** 51
    assert call(prob=None) == (0, 1)
    assert call(rows=0) == (0, 0)
    assert call(rows=4, stride=120) == (0, 1)
    for bad in (dict(tokens=None), dict(logits=None), dict(requests=None), dict(u=None), dict(rows=-1),
                dict(rows=6), dict(vocab=0), dict(vocab=101), dict(stride=99), dict(stride=101),
                dict(stride=-100), dict(requests=h.buf(79)), dict(u=h.buf(19)), dict(prob=h.buf(19)),
                dict(rows=65536), dict(vocab=(1 << 20) + 1)):
        rc, n = call(**bad)
        assert rc < 0 and n == 0 and h.error().startswith("gpu_sample"), bad
    big = h.buf(1 << 20)
    for o in ("logits", "requests", "u"):
        assert call(**{"tokens": big, o: big}) == (-1, 0)
        assert call(**{"prob": big, o: big}) == (-1, 0)
    assert call(tokens=big, prob=big) == (-1, 0)
    # n units of the largest sum fit 62 bits
    for vocab in (1, 1023, 1024, 1025, 248320, 1 << 20):
        assert call(rows=1, vocab=vocab, logits=h.buf(vocab * 4)) == (0, 1)
        assert vocab * h.L.decode_unit() <= 2.0 ** 62
        assert h.L.decode_unit() == 2.0 ** 51 or vocab * h.L.decode_unit() >= 2.0 ** 61


def test_host_reports_and_keeps_the_device(host, om):
    h = host
    a = linear_call(h)
    for word, text in ((3, "a slot of sequence 2"), (4, "the tokens of sequence 2"), (5, "row 2")):
        h.mark(word, 2)
        assert h.call("gpu_linear_attend", a) == (-1, 1) and text in h.error()
        assert h.call("gpu_linear_attend", a) == (0, 1)
    h.mark(3, 1)
    a["opts"].flags = om.KV_ASYNC
    assert h.call("gpu_linear_attend", a) == (0, 1)
    a["opts"].flags = 0
    a["B"] = 0  # nothing of its own to do: what was marked is reported all the same
    assert h.call("gpu_linear_attend", a) == (-1, 0)
    h.int("decode_device").value = 3
    assert h.call("gpu_linear_attend", linear_call(h)) == (0, 1)
    assert h.int("decode_device").value == 3
    h.int("decode_device").value = 0


# ------------------------------------------------------------ the GPU
@pytest.fixture(scope="module")
def ctx(om):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    c = om.Context()
    yield c
    c.close()


def _up(ctx, *tensors):
    return [ctx.upload(t.contiguous().view(torch.uint8).numpy() if t.dtype in (torch.bfloat16, torch.float8_e4m3fn)
                       else t.contiguous().numpy()) for t in tensors]


def _down(ctx, buf, shape, dtype=torch.float32):
    n = math.prod(shape) * dtype.itemsize
    return torch.from_numpy(ctx.download(buf, np.uint8, (n,))).view(dtype).reshape(shape)


def _close(got, want, tol):
    got = got.double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {((got - want).abs() / tol).max():.3g} of the bound"


# ---------------------------------------- norms
def _norm64(x, w, kind, eps):
    x = x.double()
    ss = (x * x).sum(-1, keepdim=True)
    y = x / torch.sqrt((ss / x.shape[-1] if kind == "rms" else ss) + eps)
    return y if w is None else y * w.double()


def _rope64(y, pairs, base, halves, pos, tol):
    """y rotated, and `tol` (of y, relative) turned into absolute bounds."""
    z, b, R = y.clone(), y.abs() * tol * EPS, sum(pairs)
    p = 0
    for a, n in enumerate(pairs):
        for p in range(p, p + n):
            i, j = (p, p + R) if halves else (2 * p, 2 * p + 1)
            ang = pos[a].double() * base ** (-p / R)
            c, s = ang.cos()[:, None], ang.sin()[:, None]
            z[..., i], z[..., j] = y[..., i] * c - y[..., j] * s, y[..., i] * s + y[..., j] * c
            both = (y[..., i].abs() + y[..., j].abs()) * (tol + 6) * EPS
            b[..., i], b[..., j] = both, both
        p += 1 if n else 0
    return z, b


def _weights(g, heads, D, how):
    if how == "no":
        return None
    return 1.0 + 0.5 * torch.randn(heads if how == "each" else 1, D, generator=g)


NORM_CASES = [
    # T, heads, kv, D, pairs, halves, kind, weights
    (1, 16, 2, 256, [32], False, "rms", "one"),
    (7, 8, 2, 128, [16, 24, 24], True, "rms", "each"),
    (33, 5, 1, 64, [32], True, "l2", "no"),
    (700, 3, 3, 96, [], True, "rms", "one"),
    (5, 4, 4, 80, [9, 0, 11], False, "l2", "each"),
    (9, 2, 1, 33, [16], True, "rms", "one"),
    (4, 3, 2, 1, [], False, "rms", "no"),
    (3, 2, 2, 7, [2], False, "l2", "one"),
    (6, 2, 1, 130, [33, 32], True, "rms", "each"),
    (2, 3, 1, 4, [2], False, "rms", "one"),
    (513, 1, 1, 12, [4], True, "rms", "no"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", NORM_CASES + [
    (3, 2, 1, 4096, [100, 156], True, "rms", "one"), (2, 1, 2, 1000, [64], False, "l2", "each"),
    (2, 1, 1, 2001, [256], True, "rms", "no")])
@pytest.mark.parametrize("in_place", [False, True])
def test_norm_rope(om, ctx, case, in_place):
    T, H, kv, D, pairs, halves, kind, weights = case
    g = torch.Generator().manual_seed(T + D)
    q = torch.randn(T, H, D, generator=g) * torch.exp(2 * torch.randn(T, H, 1, generator=g))
    k = torch.randn(T, kv, D, generator=g) * torch.exp(2 * torch.randn(T, kv, 1, generator=g))
    q[0, 0] = 0.0  # a row of zeros stays one
    qw, kw = _weights(g, H, D, weights), _weights(g, kv, D, weights)
    pos = torch.randint(0, 200000, (max(1, len(pairs)), T), generator=g, dtype=torch.int32)
    qb, kb, pb = _up(ctx, q, k, pos)
    wb = [None if w is None else _up(ctx, w)[0] for w in (qw, kw)]
    qo, ko = (qb, kb) if in_place else (ctx.alloc(q.numel() * 4), ctx.alloc(k.numel() * 4))
    rope = om.rope_axes(pairs, 1e6, halves=halves) if pairs else None
    om.norm_rope_axes(ctx, qo, ko, qb, kb, T, H, kv, D, om.head_norm(kind, 1e-6, *wb, weights == "each"),
                      pb if pairs else None, rope)
    n = (D / 64 + 16) / 2 + 6
    for x, w, o in ((q, qw, qo), (k, kw, ko)):
        want, tol = _rope64(_norm64(x, w, kind, 1e-6), pairs, 1e6, halves, pos, n)
        _close(_down(ctx, o, x.shape), want, tol + 1e-45)


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f32", "f16", "bf16", "e4m3"])
@pytest.mark.parametrize("case", NORM_CASES)
def test_norm_append(om, ctx, case, type):
    T, H, kv, D, pairs, halves, kind, weights = case
    g = torch.Generator().manual_seed(T * 3 + D)
    page = 8
    pages = -(-T // page) + 2
    q, k, v = (torch.randn(T, h, D, generator=g) for h in (H, kv, kv))
    qw, kw = _weights(g, H, D, weights), _weights(g, kv, D, weights)
    pos = torch.randint(0, 200000, (max(1, len(pairs)), T), generator=g, dtype=torch.int32)
    slots = torch.randperm(pages * page, generator=g)[:T].to(torch.int32)
    if T > 2:
        slots[1] = -1
    pool = torch.randn(2, pages, kv, page, D, generator=g).to(DTYPE[type])
    qb, kb, vb, pb, sb = _up(ctx, q, k, v, pos, slots)
    kp, vp = _up(ctx, pool[0], pool[1])
    wb = [None if w is None else _up(ctx, w)[0] for w in (qw, kw)]
    qo = ctx.alloc(q.numel() * 4)
    kvp = om.kv_pages(kp, vp, type, pages, page, kv, D, 0.5, 0.25)
    om.norm_kv_append(ctx, kvp, kb, vb, T, sb, qo, qb, H,
                      om.head_norm(kind, 1e-5, *wb, weights == "each"), pb if pairs else None,
                      om.rope_axes(pairs, 1e4, halves=halves) if pairs else None)
    n = (D / 64 + 16) / 2 + 6
    want, tol = _rope64(_norm64(q, qw, kind, 1e-5), pairs, 1e4, halves, pos, n)
    _close(_down(ctx, qo, q.shape), want, tol + 1e-45)
    yk, tk = _rope64(_norm64(k, kw, kind, 1e-5), pairs, 1e4, halves, pos, n)
    rel, least = STEP[type]
    for buf, before, y, tol, scale in ((kp, pool[0], yk, tk, 0.5),
                                       (vp, pool[1], v.double(), torch.zeros_like(yk), 0.25)):
        scale = scale if type == "e4m3" else 1.0
        got = _down(ctx, buf, before.shape, DTYPE[type])
        rows = got.double().permute(0, 2, 1, 3).reshape(-1, kv, D)
        on = slots >= 0
        at = slots[on].long()
        y, tol = y[on] / scale, tol[on] / scale
        lim = 448.0 if type == "e4m3" else math.inf
        _close(rows[at], y.clamp(-lim, lim), tol + (y.abs() + tol) * rel + least)
        left = torch.ones(pages * page, dtype=torch.bool)
        left[at] = False  # the other slots are as they were
        raw = [x.view(torch.uint8).reshape(pages, kv, page, -1).permute(0, 2, 1, 3).reshape(pages * page, -1)
               for x in (got, before)]
        assert torch.equal(raw[0][left], raw[1][left])


@pytest.mark.gpu
def test_norm_of_bad_slots_and_values(om, ctx):
    """A slot past the pages is left out and reported; a NaN or an infinity stays in its row."""
    T, H, kv, D, page = 6, 2, 1, 64, 8
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(T, h, D, generator=g) for h in (H, kv, kv))
    q[1, 0, 3], q[2, 1, 5] = math.nan, math.inf
    slots = torch.tensor([0, 99, 2, -7, 4, 5], dtype=torch.int32)
    pool = torch.zeros(2, kv, page, D)
    qb, kb, vb, sb, kp, vp = _up(ctx, q, k, v, slots, pool, pool)
    qo = ctx.alloc(q.numel() * 4)
    pages = om.kv_pages(kp, vp, "f32", 2, page, kv, D)
    with pytest.raises(RuntimeError, match="slot of token"):
        om.norm_kv_append(ctx, pages, kb, vb, T, sb, qo, qb, H, om.head_norm("rms"))
    got = _down(ctx, qo, q.shape)
    bad = torch.zeros(T, H, dtype=torch.bool)
    bad[1, 0] = bad[2, 1] = True
    assert torch.isfinite(got[~bad]).all() and torch.isnan(got[1, 0]).all()
    assert torch.isnan(got[2, 1, 5]) and (got[2, 1, :5] == 0).all()  # x / infinity
    rows = _down(ctx, vp, (2, kv, page, D)).permute(0, 2, 1, 3).reshape(16, kv, D)
    for s, t in ((0, 0), (2, 2), (4, 4), (5, 5)):
        assert torch.equal(rows[s], v[t])
    assert (rows[[1, 3] + list(range(6, 16))] == 0).all()


# ---------------------------------------- linear attention
def _linear64(q, k, v, g, starts, S0, scale, complement):
    """Token by token in 64 bits, with the same sums of absolute values.  S0: [B][H][dk][dv]."""
    H = S0.shape[1]
    q, k, v = (x.double().repeat_interleave(H // x.shape[1], dim=1) for x in (q, k, v))
    a = torch.exp(g.double()).expand(q.shape[0], H)
    b = 1.0 - a if complement else torch.ones_like(a)
    out, bound = torch.zeros_like(v[:, :, :S0.shape[3]]), torch.zeros_like(v)
    ends, end_bounds = S0.double().clone(), S0.double().abs()
    for s, (t0, t1) in enumerate(zip(starts[:-1], starts[1:])):
        S, A = ends[s], end_bounds[s]
        for t in range(t0, t1):
            f, kv = a[t][:, None, None], k[t][:, :, None] * v[t][:, None] * b[t][:, None, None]
            S, A = torch.where(f == 0, kv, S * f + kv), torch.where(f == 0, kv.abs(), A * f + kv.abs())
            out[t] = (S * q[t][:, :, None]).sum(1) * scale
            bound[t] = (A * q[t][:, :, None].abs()).sum(1) * scale
        ends[s], end_bounds[s] = S, A
    return out, bound, ends, end_bounds


def _linear_inputs(lens, H, qh, kh, vh, dk, dv, gates, seed):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens)
    q, k, v = (torch.randn(T, h, d, generator=g) for h, d in ((qh, dk), (kh, dk), (vh, dv)))
    k *= dk ** -0.5
    if gates == "token":
        decay = -torch.exp(-6 + 8 * torch.rand(H, generator=g)) * torch.rand(T, H, generator=g)
    elif gates == "strong":  # next to nothing, all at once, and in between
        decay = -torch.rand(T, H, generator=g) * 10 ** (4 * torch.rand(T, H, generator=g) - 3)
        decay[torch.rand(T, H, generator=g) < 0.1] = -math.inf
        decay[torch.rand(T, H, generator=g) < 0.2] = 0.0
    else:
        decay = -torch.exp2(-8 * torch.rand(H, generator=g))
    return g, q, k, v, decay


def _linear_run(om, ctx, lens, H, qh, kh, vh, dk, dv, q, k, v, decay, S, ins, outs, steps=False,
                complement=False, max_len=0, scale=0.0, tail=0, flags=0, in_place=False):
    T = q.shape[0]
    starts = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    bufs = _up(ctx, q, k, v, decay)
    sb, ib, ob, tb = _up(ctx, S, torch.tensor(ins, dtype=torch.int32),
                         torch.tensor(outs, dtype=torch.int32), starts)
    if in_place:
        ob = ib
    mark = torch.full((T + tail, H, dv), 7.5)
    out = _up(ctx, mark)[0]
    om.linear_attend(ctx, om.linear_states(sb, S.shape[0], H, dk, dv), out, *bufs[:3], qh, kh, vh, T,
                     bufs[3], len(lens), None if steps else tb, ib, ob,
                     om.linear_opts(scale, decay.dim() == 2, complement, max_len, flags))
    o = _down(ctx, out, (T + tail, H, dv))
    assert torch.equal(o[T:], mark[T:])
    return o[:T], _down(ctx, sb, S.shape)


def _check_linear(om, ctx, lens, H, qh, kh, vh, dk, dv, gates="token", complement=False, seed=0,
                  max_len=0, steps=False, scale=0.0):
    g, q, k, v, decay = _linear_inputs(lens, H, qh, kh, vh, dk, dv, gates, seed)
    B = len(lens)
    S = torch.randn(2 * B + 2, H, dk, dv, generator=g)
    perm = torch.randperm(2 * B + 2, generator=g).tolist()
    ins = [p if i % 3 else -1 for i, p in enumerate(perm[:B])]
    outs = [p if i % 4 != 2 else -1 for i, p in enumerate(perm[B:2 * B])]
    S[perm[2 * B]] = math.nan  # a slot that no sequence uses
    for i, p in enumerate(perm[:B]):
        if ins[i] < 0:
            S[p] = math.nan  # one that is not read
    for p in outs:
        if p >= 0:
            S[p] = math.inf  # what a slot held does not matter to what is written
    o, S1 = _linear_run(om, ctx, lens, H, qh, kh, vh, dk, dv, q, k, v, decay, S, ins, outs, steps,
                        complement, max_len, scale, tail=2)
    S0 = torch.stack([S[i] if i >= 0 else torch.zeros_like(S[0]) for i in ins])
    starts = [sum(lens[:i]) for i in range(B + 1)]
    want, bound, ends, eb = _linear64(q, k, v, decay, starts, S0, scale or dk ** -0.5, complement)
    c = (8 + 6 * math.sqrt(2 * max(lens) + dk)) * EPS
    _close(o, want, bound * c + 1e-37)
    for b, p in enumerate(outs):
        if p >= 0:
            _close(S1[p], ends[b], eb[b] * c + 1e-37)
    rest = [p for p in range(2 * B + 2) if p not in outs]
    assert torch.equal(S1[rest].view(torch.int32), S[rest].view(torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("H,qh,kh,vh,dk,dv", [
    (4, 4, 4, 4, 128, 128), (6, 2, 3, 6, 64, 64), (4, 4, 1, 1, 33, 47), (3, 1, 1, 3, 1, 1),
    (2, 2, 2, 2, 256, 256), (5, 5, 5, 1, 96, 80), (2, 1, 2, 2, 20, 200)])
@pytest.mark.parametrize("gates", ["token", "head", "strong"])
def test_linear_steps(om, ctx, H, qh, kh, vh, dk, dv, gates):
    for B in (1, 5):
        _check_linear(om, ctx, [1] * B, H, qh, kh, vh, dk, dv, gates, complement=B == 5, steps=True,
                      seed=B + dk, scale=0.3 if B == 5 else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[1], [2, 0, 1], [31, 32, 33], [64], [65, 17], [300, 5, 0, 129], [0, 3]])
@pytest.mark.parametrize("H,qh,kh,vh,dk,dv", [(2, 2, 2, 2, 128, 128), (4, 2, 1, 4, 64, 40),
                                              (2, 2, 2, 2, 33, 47)])
def test_linear_lengths(om, ctx, lens, H, qh, kh, vh, dk, dv):
    _check_linear(om, ctx, lens, H, qh, kh, vh, dk, dv, seed=sum(lens))


@pytest.mark.gpu
@pytest.mark.parametrize("H,qh,kh,vh,dk,dv", [
    (1, 1, 1, 1, 1, 1), (2, 1, 1, 2, 4, 8), (3, 3, 1, 1, 32, 100), (2, 2, 2, 1, 96, 80),
    (1, 1, 1, 1, 256, 256), (2, 1, 2, 2, 200, 130), (2, 2, 2, 2, 63, 65), (1, 1, 1, 1, 129, 3)])
@pytest.mark.parametrize("gates,complement", [("token", True), ("head", False), ("strong", False),
                                              ("strong", True)])
def test_linear_shapes(om, ctx, H, qh, kh, vh, dk, dv, gates, complement):
    _check_linear(om, ctx, [70, 1, 131], H, qh, kh, vh, dk, dv, gates, complement, seed=dk + dv,
                  max_len=200)


@pytest.mark.gpu
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (48, 130)])
def test_linear_long(om, ctx, dk, dv):
    """Long enough to be cut between work groups."""
    _check_linear(om, ctx, [2500, 900], 2, 1, 2, 2, dk, dv, "token", seed=5)
    _check_linear(om, ctx, [1100], 2, 1, 1, 2, dk, dv, "strong", True, seed=6)


@pytest.mark.gpu
def test_linear_in_place_and_in_parts(om, ctx):
    """A prompt in parts, then token by token, each going on in its own slot."""
    H, dk, dv, lens = 2, 64, 96, [150, 37]
    g, q, k, v, decay = _linear_inputs(lens, H, 1, 1, 2, dk, dv, "token", 3)
    S = torch.randn(3, H, dk, dv, generator=g)
    want, bound, ends, eb = _linear64(q, k, v, decay, [0, 150, 187], S[:2], dk ** -0.5, False)
    c = (8 + 6 * math.sqrt(300 + dk)) * EPS
    cut = [(0, 100), (100, 149), (149, 150)]
    second = [(0, 20), (20, 36), (36, 37)]
    state, rows = S, {}
    for (a0, a1), (b0, b1) in zip(cut, second):
        at = list(range(a0, a1)) + list(range(150 + b0, 150 + b1))
        step = a1 - a0 == 1
        o, state = _linear_run(om, ctx, [a1 - a0, b1 - b0], H, 1, 1, 2, dk, dv, q[at], k[at], v[at],
                               decay[at], state, [0, 1], [0, 1], steps=step, in_place=True)
        rows.update(zip(at, o))
    _close(torch.stack([rows[t] for t in range(187)]), want, bound * c)
    _close(state[:2], ends, eb * c)
    assert torch.equal(state[2], S[2])


@pytest.mark.gpu
def test_linear_forks_a_state(om, ctx):
    H, dk, dv = 2, 32, 32
    g, q, k, v, decay = _linear_inputs([3, 70], H, 2, 2, 2, dk, dv, "token", 4)
    S = torch.randn(4, H, dk, dv, generator=g)
    o, S1 = _linear_run(om, ctx, [3, 70], H, 2, 2, 2, dk, dv, q, k, v, decay, S, [1, 1], [0, 3])
    want, bound, ends, eb = _linear64(q, k, v, decay, [0, 3, 73], S[[1, 1]], dk ** -0.5, False)
    c = (8 + 6 * math.sqrt(140 + dk)) * EPS
    _close(o, want, bound * c)
    _close(S1[[0, 3]], ends, eb * c)
    assert torch.equal(S1[[1, 2]], S[[1, 2]])


@pytest.mark.gpu
@pytest.mark.parametrize("dk,dv", [(128, 128), (40, 24)])
def test_linear_keeps_later_tokens_out(om, ctx, dk, dv):
    """What is not finite takes no part before its token, and only in its own columns of V."""
    H, L = 2, 90
    g, q, k, v, decay = _linear_inputs([L], H, 1, 1, 2, dk, dv, "token", 8)
    S = torch.randn(2, H, dk, dv, generator=g)
    plain, _ = _linear_run(om, ctx, [L], H, 1, 1, 2, dk, dv, q, k, v, decay, S, [0], [1])
    for at, value in ((0, math.inf), (37, math.nan), (50, -math.inf), (89, math.inf)):
        v1 = v.clone()
        v1[at, 0, 3] = value
        o, S1 = _linear_run(om, ctx, [L], H, 1, 1, 2, dk, dv, q, k, v1, decay, S, [0], [1])
        same = torch.ones(L, H, dv, dtype=torch.bool)
        same[at:, 0, 3] = False
        assert torch.isfinite(o[same]).all() and not torch.isfinite(o[at:, 0, 3]).any()
        _close(o[same], plain[same].double(), plain[same].double().abs() * 1e-4 + 1e-4)
        assert torch.isfinite(S1[1, 1]).all() and torch.isfinite(S1[1, 0, :, 4:]).all()
        assert not torch.isfinite(S1[1, 0, :, 3]).any()
        for which in (0, 1):
            x = [q.clone(), k.clone()]
            x[which][at, 0, 1] = value
            o, _ = _linear_run(om, ctx, [L], H, 1, 1, 2, dk, dv, x[0], x[1], v, decay, S, [0], [1])
            assert torch.isfinite(o[:at]).all() and not torch.isfinite(o[at]).any()
            if which == 0:
                assert torch.isfinite(o[at + 1:]).all()
        d = decay.clone()
        d[at, 0] = math.nan
        o, _ = _linear_run(om, ctx, [L], H, 1, 1, 2, dk, dv, q, k, v, d, S, [0], [1])
        assert torch.isfinite(o[:at]).all() and torch.isnan(o[at:, 0]).all()
        assert torch.isfinite(o[:, 1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("L", [200, 700, 1500])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 40), (96, 80), (33, 47)])
def test_linear_parts_that_are_not_finite(om, ctx, L, dk, dv):
    """In a sequence that is cut, in place: what is finite is right beside what is not."""
    H, at, lens = 2, 130, [L, 90]
    g, q, k, v, decay = _linear_inputs(lens, H, 1, 2, 2, dk, dv, "token", L + dk)
    S = torch.randn(2, H, dk, dv, generator=g)
    want, bound, ends, eb = _linear64(q, k, v, decay, [0, L, L + 90], S, dk ** -0.5, False)
    c = (8 + 6 * math.sqrt(2 * L + dk)) * EPS
    v[at, 0, 3], v[at + 1, 0, 5] = math.inf, math.nan
    o, S1 = _linear_run(om, ctx, lens, H, 1, 2, 2, dk, dv, q, k, v, decay, S, [0, 1], [0, 1], in_place=True)
    bad = torch.zeros(L + 90, H, dv, dtype=torch.bool)
    bad[at:L, 0, 3] = bad[at + 1:L, 0, 5] = True
    assert not torch.isfinite(o[bad]).any() and not torch.isfinite(S1[0, 0][:, [3, 5]]).any()
    _close(o[~bad], want[~bad], bound[~bad] * c)
    S1[0, 0][:, [3, 5]] = 0.0
    ends[0, 0][:, [3, 5]] = 0.0
    _close(S1, ends, eb * c + 1e-37)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** 100])
def test_linear_of_small_and_large_values(om, ctx, scale):
    """V and the state by a power of two: the same digits."""
    H, L, d = 2, 300, 128
    g, q, k, v, decay = _linear_inputs([L], H, 2, 2, 2, d, d, "head", 12)
    S = torch.randn(1, H, d, d, generator=g)
    want, bound, ends, eb = _linear64(q, k, v * scale, decay, [0, L], S * scale, d ** -0.5, False)
    c = (8 + 6 * math.sqrt(2 * L + d)) * EPS
    o, S1 = _linear_run(om, ctx, [L], H, 2, 2, 2, d, d, q, k, v * scale, decay, S * scale, [0], [0], in_place=True)
    _close(o, want, bound * c)
    _close(S1, ends, eb * c)


@pytest.mark.gpu
def test_linear_agrees_with_the_gated_step(om, ctx):
    """gpu_deltanet_step_gated: its K is the value, its V the key, its gate the decay."""
    n, gate = 64, 0.75
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(n, generator=g) for _ in range(3))
    S = torch.randn(n, n, generator=g)
    sb, qb, kb, vb = _up(ctx, S, q, k, v)
    out = ctx.alloc(n * 4)
    assert om.lib().gpu_deltanet_step_gated(ctx.ptr, sb.ptr, qb.ptr, kb.ptr, vb.ptr, out.ptr, n, gate) == 0
    decay = torch.tensor([math.log(gate)])
    o, S1 = _linear_run(om, ctx, [1], 1, 1, 1, 1, n, n, q.view(1, 1, n), v.view(1, 1, n), k.view(1, 1, n),
                        decay, S.view(1, 1, n, n), [0], [0], steps=True, complement=True, scale=1.0)
    c = (8 + 6 * math.sqrt(2 + n)) * EPS
    A = S.abs() * gate + 0.25 * v.abs()[:, None] * k.abs()
    _close(S1[0, 0], _down(ctx, sb, (n, n)).double(), 2 * c * A.double())
    _close(o[0, 0], _down(ctx, out, (n,)).double(), 2 * c * (A * q.abs()[:, None]).sum(0).double())


@pytest.mark.gpu
def test_linear_reports_bad_numbers(om, ctx):
    H, dk, dv = 2, 16, 16
    g, q, k, v, decay = _linear_inputs([4, 4, 4], H, 2, 2, 2, dk, dv, "token", 9)
    S = torch.randn(4, H, dk, dv, generator=g)
    sb, ib, ob = _up(ctx, S, torch.tensor([0, 4, 1], dtype=torch.int32),
                     torch.tensor([0, 2, -2], dtype=torch.int32))
    bufs = _up(ctx, q, k, v, decay)
    st = om.linear_states(sb, 4, H, dk, dv)
    mark = torch.full((12, H, dv), 7.5)

    def call(starts, slots, max_len=0, n=3, flags=0):
        out, tb = _up(ctx, mark, torch.tensor(starts, dtype=torch.int32))
        om.linear_attend(ctx, st, out, *bufs[:3], 2, 2, 2, 12, bufs[3], n, tb, *slots,
                         om.linear_opts(0, True, False, max_len, flags))
        return out

    with pytest.raises(RuntimeError, match="a slot of sequence"):
        call([0, 4, 8, 12], (ib, ob))
    after = _down(ctx, sb, S.shape)
    assert torch.equal(after[1:], S[1:]) and not torch.equal(after[0], S[0])
    for starts, max_len in (([0, 4, 3, 12], 0), ([-1, 4, 8, 12], 0), ([0, 4, 8, 13], 0),
                            ([0, 4, 8, 12], 3)):
        with pytest.raises(RuntimeError, match="the tokens of sequence"):
            call(starts, (None, None), max_len)
    out = call([0, 2, 13, 14], (None, None), n=3, flags=om.KV_ASYNC)
    assert om.lib().gpu_kv_check(ctx.ptr) == -1 and om.lib().gpu_kv_check(ctx.ptr) == 0
    assert torch.equal(_down(ctx, out, (12, H, dv))[2:], mark[2:])  # the first sequence alone
    assert (_down(ctx, out, (12, H, dv))[:2] != 7.5).all()


# ---------------------------------------- sampling
def _choices(x, temperature, top_k, top_p, min_p, u):
    """The tokens that 64-bit sums allow, and their shares: more than one next to a border only."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    on = int((x > -np.inf).sum())
    if not on:
        return {-1: [0.0]}
    order = np.lexsort((np.arange(x.size), -x))[:on]
    if temperature == 0:
        return {int(order[0]): [1.0]}
    top = x[order[0]]
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / float(np.float32(temperature))))
    off = x.size * 2.0 ** -44
    if 0 < top_k < on:
        w = w[:top_k]
    before = np.cumsum(w) - w
    found = {}
    for sign in (-1.0, 1.0):  # the borders as far apart as rounding may put them
        last = before < float(np.float32(top_p)) * w.sum() + sign * off
        last &= w >= float(np.float32(min_p)) * (1.0 - sign * 1e-15)
        last[0] = True
        kept = w[last]
        c = np.cumsum(kept)
        for s in (-1.0, 1.0):
            i = int(np.searchsorted(c, float(np.float32(u)) * c[-1] + s * off, side="right"))
            i = min(i, len(kept) - 1)
            found.setdefault(int(order[i]), []).append(kept[i] / c[-1])
    return found


def _sample(om, ctx, x, requests, u, stride=0, prob=True):
    rows = x.shape[0]
    r = np.array([tuple(q) for q in requests], om.SAMPLE_REQUEST)
    xb = ctx.upload(np.ascontiguousarray(x, np.float32))
    rb, ub = ctx.upload(r), ctx.upload(np.asarray(u, np.float32))
    tb, pb = ctx.upload(np.full(rows + 1, 77, np.int32)), ctx.upload(np.full(rows + 1, 7.5, np.float32))
    n = x.shape[1] if not stride else min(stride, x.shape[1])
    err = None
    try:
        om.sample(ctx, tb, pb if prob else None, xb, rows, n, rb, ub, stride)
    except RuntimeError as e:
        err = str(e)
    t, p = ctx.download(tb, np.int32, (rows + 1,)), ctx.download(pb, np.float32, (rows + 1,))
    for b in (xb, rb, ub, tb, pb):
        b.free()
    assert t[-1] == 77 and p[-1] == 7.5
    return t[:-1], p[:-1], err


def _check_sample(om, ctx, x, requests, u):
    t, p, err = _sample(om, ctx, x, requests, u)
    assert err is None
    several = 0
    for i, (row, q) in enumerate(zip(x, requests)):
        ok = _choices(row, *q, u[i])
        several += len(ok) > 1
        assert int(t[i]) in ok, (i, q, u[i], int(t[i]), ok)
        want = min(ok[int(t[i])], key=lambda w: abs(p[i] - w))
        assert abs(p[i] - want) <= want * (EPS + 2 * x.shape[1] * 2.0 ** -45), (i, q, p[i], want)
    assert several <= len(requests) // 8  # the borders are seldom near


REQUESTS = [(0.7, 20, 0.8, 0.0), (1.0, 0, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.2, 0, 1.0, 0.05),
            (0.8, 40, 0.95, 0.05), (1.0, 0, 1.0, 0.0), (0.6, 1000, 0.9, 0.0), (1.0, 1, 1.0, 0.0),
            (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (100.0, 0, 0.5, 0.0), (0.01, 50, 0.99, 0.1),
            (1e-30, 0, 1.0, 0.0), (3.0, 7, 0.3, 0.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 1000, 4099, 32000, 100003])
@pytest.mark.parametrize("what", ["spread", "flat", "grid", "masked"])
def test_sample(om, ctx, n, what):
    g = np.random.default_rng(n + len(what))
    rows = 2 * len(REQUESTS)
    x = g.standard_normal((rows, n)) * {"spread": 4.0, "flat": 0.05}.get(what, 2.0)
    if what == "grid":
        x = np.round(x * 4) / 4  # many equal logits
    x = x.astype(np.float32)
    if what == "masked":
        x[g.random((rows, n)) < 0.7] = -np.inf
        x[g.random((rows, n)) < 0.1] = np.nan
        x[g.random((rows, n)) < 0.1] = np.finfo(np.float32).min
    u = g.random(rows).astype(np.float32)
    u[u == 1.0] = 0.5
    _check_sample(om, ctx, x, REQUESTS * 2, u)


@pytest.mark.gpu
def test_sample_of_equal_logits(om, ctx):
    """All equal: the k-th of the kept, in order."""
    n = 5000
    x = np.zeros((6, n), np.float32)
    x[0, ::2] = -0.0  # equal to 0
    x[1] = np.finfo(np.float32).min
    x[2] = -3.5
    x[3] = 1e30
    u = np.array([0.5, 0.25, 0.0, 1 - 2.0 ** -24, 0.75, 0.1], np.float32)
    req = [(1.0, 0, 1.0, 0.0), (2.0, 1000, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 0, 1.0, 1.0),
           (0.5, 100, 0.5, 0.5), (0.0, 0, 1.0, 0.0)]
    t, p, err = _sample(om, ctx, x, req, u)
    assert err is None
    assert t.tolist() == [2500, 250, 0, 4999, 37, 0]
    assert np.allclose(p, [1 / 5000, 1 / 1000, 1 / 2500, 1 / 5000, 1 / 50, 1.0], rtol=2e-7, atol=0)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [9000, 40000])
def test_sample_of_many_equal_logits(om, ctx, n):
    """More of them next to a border than are put in order, and others above and below."""
    g = np.random.default_rng(n)
    x = np.zeros((2 * len(REQUESTS), n), np.float32)
    x[::3, g.integers(0, n, 50)] = 1.5
    x[1::2, g.integers(0, n, 50)] = -2.0
    x[::4, g.integers(0, n, 3000)] = -np.inf
    u = (g.random(len(x)) * 0.999).astype(np.float32)
    requests = REQUESTS + [(1.0, 5000, 0.9, 0.0), (1.0, 8500, 1.0, 0.0), (2.0, 8999, 0.5, 0.1)] + REQUESTS[3:]
    _check_sample(om, ctx, x, requests, u)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [20000, 60000])
def test_sample_with_a_large_top_k(om, ctx, n):
    g = np.random.default_rng(n)
    requests = [(1.0, k, p, m) for k in (1, 2, 64, 4096, 4097, 12000, n - 1, n, 2 ** 31 - 1)
                for p, m in ((1.0, 0.0), (0.9, 0.0), (0.999, 0.001))]
    x = (g.standard_normal((len(requests), n)) * 2).astype(np.float32)
    _check_sample(om, ctx, x, requests, g.random(len(x)).astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [7001, 30000, 32769, 90001])
@pytest.mark.parametrize("what", ["sorted", "one bin", "few values", "two bins"])
def test_sample_of_crowded_rows(om, ctx, n, what):
    """The largest beside each other; more tokens between two borders than are put in order."""
    g = np.random.default_rng(n + len(what))
    requests = [(T, k, p, m) for T, p, m in ((1.0, 0.9, 0.0), (50.0, 0.7, 0.0), (40.0, 1.0, 0.0), (30.0, 0.999, 0.2))
                for k in (0, 1000, 2048, 6000)]
    x = g.standard_normal((len(requests), n)) * 2
    if what == "sorted":
        x = -np.sort(-x, axis=1)
    elif what == "few values":
        x = np.round(x)
    else:  # what lies far below makes the bins wide
        x *= 0.01
        x[:, g.integers(0, n, 7)] = -500.0
        if what == "two bins":
            x[:, n // 2:] -= 40.0
    x = x.astype(np.float32)
    _check_sample(om, ctx, x, requests, (g.random(len(x)) * 0.999).astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [9000, 40000])
def test_sample_where_weights_end(om, ctx, n):
    """More tokens of the top_k than have a weight; logits farther apart than the largest number."""
    g = np.random.default_rng(n)
    x = np.full((6, n), -80.0, np.float32)
    x[:, 0] = 0.0
    x[:4, 10:1000] = -30.0 - 0.001 * g.random((4, 990))
    x[:4, 1000:8000] = -36.6 - 0.1 * g.random((4, 7000))  # 2^-53 of the largest
    x[4] = np.where(g.random(n) < 0.5, -3e38, 3e38)
    x[5] = np.linspace(-3.4e38, 3.4e38, n)
    requests = [(1.0, 3000, 1.0, 0.0), (1.0, 300, 0.9999999, 0.0), (1.0, 0, 1.0, 0.0), (1.0, 1000, 0.9, 0.0),
                (1e38, 0, 1.0, 0.0), (2e38, 0, 0.9, 0.01)]
    _check_sample(om, ctx, x, requests, np.array([0.3, 0.99, 0.999999, 0.5, 0.999, 0.9], np.float32))


@pytest.mark.gpu
def test_sample_of_special_rows(om, ctx):
    n = 300
    g = np.random.default_rng(3)
    x = g.standard_normal((8, n)).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 17], x[2, 250] = np.inf, np.inf
    x[3] = -np.inf
    x[3, 299] = -1e38
    x[4, 5] = 3e38  # far above all others
    x[5] *= 1e-42   # subnormal
    x[6, 1:] = np.nan
    req = [(1.0, 0, 0.9, 0.0)] * 8
    u = np.full(8, 0.6, np.float32)
    t, p, err = _sample(om, ctx, x, req, u)
    assert err is None
    assert t[:5].tolist() == [-1, -1, 250, 299, 5] and t[6] == 0
    assert p[:5].tolist() == [0, 0, 0.5, 1, 1] and p[6] == 1
    _check_sample(om, ctx, x[5:6], req[:1], u[:1])
    _check_sample(om, ctx, x[7:], req[:1], u[:1])
    x[0, 3] = 1.0
    t, _, _ = _sample(om, ctx, x, [(0.0, 5, 0.5, 0.9)] * 8, u)
    assert t.tolist() == [3, -1, 17, 299, 5, int(x[5].argmax()), 0, int(x[7].argmax())]


@pytest.mark.gpu
def test_sample_strides_and_no_prob(om, ctx):
    g = np.random.default_rng(4)
    x = g.standard_normal((5, 1003)).astype(np.float32)
    x[:, 900:] = 50.0  # not the rows'
    u = g.random(5).astype(np.float32)
    rb = ctx.upload(np.array([REQUESTS[i] for i in range(5)], om.SAMPLE_REQUEST))
    xb, ub, tb = ctx.upload(x), ctx.upload(u), ctx.alloc(20)
    om.sample(ctx, tb, None, xb, 5, 900, rb, ub, stride=1003)
    got = ctx.download(tb, np.int32, (5,))
    for i in range(5):
        assert int(got[i]) in _choices(x[i, :900], *REQUESTS[i], u[i])


@pytest.mark.gpu
def test_sample_refuses_requests(om, ctx):
    g = np.random.default_rng(5)
    good = (1.0, 0, 1.0, 0.0)
    bad = [(-1.0, 0, 1.0, 0.0), (math.nan, 0, 1.0, 0.0), (math.inf, 0, 1.0, 0.0),
           (1.0, 0, -0.1, 0.0), (1.0, 0, 1.1, 0.0), (1.0, 0, math.nan, 0.0), (1.0, 0, 1.0, -0.1),
           (1.0, 0, 1.0, 1.5), (1.0, 0, 1.0, math.nan)]
    req = [good] + bad + [good] * 4
    u = [0.5] * (1 + len(bad)) + [-0.1, 1.0, math.nan, 0.0]
    x = g.standard_normal((len(req), 777)).astype(np.float32)
    t, p, err = _sample(om, ctx, x, req, u)
    assert "row" in err
    assert (t[1:-1] == -1).all() and (p[1:-1] == 0).all()
    for i in (0, len(req) - 1):
        assert int(t[i]) in _choices(x[i], *good, u[i])
    assert om.lib().gpu_kv_check(ctx.ptr) == 0


@pytest.mark.gpu
def test_sample_repeats(om, ctx):
    """The same call gives the same tokens and shares, bit for bit."""
    g = np.random.default_rng(6)
    x = (g.standard_normal((14, 50021)) * 0.3).astype(np.float32)
    u = g.random(14).astype(np.float32)
    first = _sample(om, ctx, x, REQUESTS, u)
    for _ in range(3):
        again = _sample(om, ctx, x, REQUESTS, u)
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])


# ---------------------------------------- together, and at the limits
def _unit(x, eps=1e-6):
    return _norm64(x, None, "l2", eps)


@pytest.mark.gpu
@pytest.mark.parametrize("flags", ["sync", "async"])
def test_decode_loop(om, ctx, flags):
    """A hybrid stack's loop: prompts and then tokens through a linear layer (unit queries and
    keys, states in slots) and an attention layer (normed, rotated and appended; attended),
    the LM head's product and a sampled token for each sequence, whose row of an embedding is the
    next input.  Against 64 bits, the tokens being the device's own."""
    F = om.KV_ASYNC if flags == "async" else 0
    g = torch.Generator().manual_seed(11)
    B, H, kv, D, V, page, steps = 3, 4, 2, 32, 400, 8, 5
    lens = [37, 5, 70]
    W = H * D
    emb, head = torch.randn(V, W, generator=g), torch.randn(W, V, generator=g) * 0.3
    qw, kw = 1 + 0.2 * torch.randn(1, D, generator=g), 1 + 0.2 * torch.randn(1, D, generator=g)
    rate = -torch.rand(H, generator=g)
    width = -(-(max(lens) + steps) // page)
    table = torch.randperm(B * width, generator=g).view(B, width).to(torch.int32)
    kp, vp, S = (ctx.alloc(B * width * kv * page * D * 4), ctx.alloc(B * width * kv * page * D * 4),
                 ctx.alloc((B + 1) * H * D * D * 4))
    pages = om.kv_pages(kp, vp, "f32", B * width, page, kv, D)
    states = om.linear_states(S, B + 1, H, D, D)
    rope = om.rope_axes([12], 1e4, halves=True)
    slots = torch.tensor([3, 0, 2], dtype=torch.int32)
    none = torch.full((B,), -1, dtype=torch.int32)
    tb, qwb, kwb, rb, slb, nb, headb = _up(ctx, table, qw, kw, rate, slots, none, head)
    norm, unit = om.head_norm("rms", 1e-6, qwb, kwb), om.head_norm("l2", 1e-6)
    requests = np.array([(0.8, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.02), (0.0, 0, 1.0, 0.0)], om.SAMPLE_REQUEST)
    reqb = ctx.upload(requests)

    # 64 bits: a sequence's own state and cache
    S64 = torch.zeros(B, H, D, D, dtype=torch.float64)
    K64, V64 = [torch.zeros(0, kv, D, dtype=torch.float64) for _ in range(B)], [torch.zeros(0, kv, D, dtype=torch.float64) for _ in range(B)]

    tokens = [torch.randint(0, V, (n,), generator=g) for n in lens]
    done = [0] * B
    for step in range(steps):
        x = torch.cat([emb[t] for t in tokens]).view(-1, H, D)  # the layers' projections
        n = [len(t) for t in tokens]
        T = sum(n)
        pos = torch.cat([torch.arange(d, d + m) for d, m in zip(done, n)]).to(torch.int32)
        at = torch.cat([table[b, (torch.arange(d, d + m) // page)] * page + torch.arange(d, d + m) % page
                        for b, (d, m) in enumerate(zip(done, n))]).to(torch.int32)
        starts = torch.tensor([sum(n[:b]) for b in range(B + 1)], dtype=torch.int32)
        k2 = x[:, :kv].contiguous()
        xb, k2b, pb, ab, stb, lb = _up(ctx, x, k2, pos, at, starts,
                                       torch.tensor([d + m for d, m in zip(done, n)], dtype=torch.int32))
        uq, uk, lin, q2 = (ctx.alloc(T * W * 4) for _ in range(4))
        om.norm_rope_axes(ctx, uq, uk, xb, xb, T, H, H, D, unit, flags=F)
        om.linear_attend(ctx, states, lin, uq, uk, xb, H, H, H, T, rb, B, stb if step == 0 else None,
                         nb if step == 0 else slb, slb, om.linear_opts(max_len=max(n), flags=F))
        om.norm_kv_append(ctx, pages, k2b, k2b, T, ab, q2, xb, H, norm, pb, rope, flags=F)
        last = starts[1:].long() - 1
        if step == 0:  # the last token's query of each prompt
            ctx.check(om.lib().gpu_kv_check(ctx.ptr), "check")
            qb = _up(ctx, _down(ctx, q2, (T, H, D))[last])[0]
        else:
            qb = q2
        att, logits, tok, prob = ctx.alloc(B * W * 4), ctx.alloc(B * V * 4), ctx.alloc(B * 4), ctx.alloc(B * 4)
        om.kv_attend(ctx, pages, att, qb, B, H, tb, width, lb, om.attend_opts(flags=F))
        ctx.check(om.lib().gpu_kv_check(ctx.ptr), "check")
        y = _down(ctx, lin, (T, H, D))[last] + _down(ctx, att, (B, H, D))
        yb = _up(ctx, y)[0]
        om.lib().gpu_matmul(ctx.ptr, logits.ptr, yb.ptr, headb.ptr, B, V, W, 0, 0)
        u = torch.rand(B, generator=g)
        ub = _up(ctx, u)[0]
        om.sample(ctx, tok, prob, logits, B, V, reqb, ub, flags=F)
        ctx.check(om.lib().gpu_kv_check(ctx.ptr), "check")
        got = _down(ctx, tok, (B,), torch.int32)

        # the same in 64 bits
        x64 = x.double()
        uq64 = _unit(x64)
        lin64 = torch.zeros(T, H, D, dtype=torch.float64)
        qn, _ = _rope64(_norm64(x, qw, "rms", 1e-6), [12], 1e4, True, pos[None], 0)
        kn, _ = _rope64(_norm64(k2, kw, "rms", 1e-6), [12], 1e4, True, pos[None], 0)
        att64 = torch.zeros(B, H, D, dtype=torch.float64)
        for b in range(B):
            for t in range(int(starts[b]), int(starts[b + 1])):
                S64[b] = S64[b] * torch.exp(rate.double())[:, None, None] + uq64[t][:, :, None] * x64[t][:, None]
                lin64[t] = (S64[b] * uq64[t][:, :, None]).sum(1) / math.sqrt(D)
            rows = slice(int(starts[b]), int(starts[b + 1]))
            K64[b], V64[b] = torch.cat([K64[b], kn[rows]]), torch.cat([V64[b], k2[rows].double()])
            for h in range(H):
                w = torch.softmax(K64[b][:, h // 2] @ qn[last[b], h] / math.sqrt(D), 0)
                att64[b, h] = w @ V64[b][:, h // 2]
        # each part's own bound (of heads of 32, up to 75 tokens; values of a few units)
        assert (y.double() - (lin64[last] + att64)).abs().max() < 2e-5
        shown = _down(ctx, logits, (B, V)).numpy()
        for b in range(B):
            assert int(got[b]) in _choices(shown[b], *[r.item() for r in requests[b]], u[b].item())
        done = [d + m for d, m in zip(done, n)]
        tokens = [got[b:b + 1].long() for b in range(B)]
    ends = _down(ctx, S, (B + 1, H, D, D))[slots.long()]
    assert (ends.double() - S64).abs().max() < 2e-5


@pytest.mark.gpu
def test_two_contexts_at_once(om, ctx):
    """Calls of two contexts in flight together, each with its own workspace."""
    other = om.Context()
    try:
        H, D, L, n = 4, 64, 1500, 50000
        g, q, k, v, decay = _linear_inputs([L], H, H, H, H, D, D, "token", 21)
        x = torch.randn(4, n, generator=g)
        u = torch.rand(4, generator=g)
        requests = np.array([REQUESTS[i] for i in (0, 1, 3, 5)], om.SAMPLE_REQUEST)
        results = []
        for together in (False, True):
            got = []
            work = []
            for c in (ctx, other):
                b = _up(c, q, k, v, decay, x, u) + [c.upload(requests)]
                work.append((c, b, c.alloc(L * H * D * 4), c.alloc(16), c.alloc(16)))
            for rep in range(3):
                for c, b, out, tok, prob in work:
                    F = om.KV_ASYNC if together else 0
                    om.linear_attend(c, om.linear_states(None, 0, H, D, D), out, *b[:3], H, H, H, L, b[3], 1,
                                     _up(c, torch.tensor([0, L], dtype=torch.int32))[0], None, None,
                                     om.linear_opts(per_token=True, flags=F))
                    om.sample(c, tok, prob, b[4], 4, n, b[6], b[5], flags=F)
            for c, b, out, tok, prob in work:
                c.check(om.lib().gpu_kv_check(c.ptr), "check")
                got.append((_down(c, out, (L, H, D)), _down(c, tok, (4,), torch.int32), _down(c, prob, (4,))))
            results += got
        for r in results[1:]:
            assert all(torch.equal(a, b) for a, b in zip(results[0], r))
    finally:
        other.close()


@pytest.mark.gpu
def test_many_sequences_and_rows(om, ctx):
    """More sequences than are ordered by length, as many as there may be, as many rows."""
    _check_linear(om, ctx, [(b * 37) % 70 for b in range(300)], 1, 1, 1, 1, 16, 16, seed=1)
    B = 65535
    q, k, v = (torch.arange(B, dtype=torch.float32).view(B, 1, 1) % m for m in (7, 5, 3))
    bufs = _up(ctx, q, k, v, torch.zeros(1))
    out = ctx.alloc(B * 4)
    om.linear_attend(ctx, om.linear_states(None, 0, 1, 1, 1), out, *bufs[:3], 1, 1, 1, B, bufs[3], B,
                     opts=om.linear_opts(scale=1.0))
    assert torch.equal(_down(ctx, out, (B, 1, 1)), q * k * v)
    x = (torch.arange(B * 5) % 7).float().view(B, 5)
    r = np.zeros(B, om.SAMPLE_REQUEST)
    r["top_p"] = 1.0
    xb, ub, rb, tok = ctx.upload(x.numpy()), ctx.alloc(B * 4), ctx.upload(r), ctx.alloc(B * 4)
    om.sample(ctx, tok, None, xb, B, 5, rb, ub)
    assert torch.equal(_down(ctx, tok, (B,), torch.int32).long(), x.argmax(1))


@pytest.mark.gpu
def test_more_tokens_than_groups(om, ctx):
    """Heads of more tokens than a launch has groups."""
    T = (1 << 20) + 77
    x = torch.randn(T, 1, 4, generator=torch.Generator().manual_seed(3))
    xb = _up(ctx, x)[0]
    out = ctx.alloc(T * 16)
    om.norm_rope_axes(ctx, out, None, xb, None, T, 1, 0, 4, om.head_norm("rms"))
    want = _norm64(x, None, "rms", 1e-6)
    _close(_down(ctx, out, x.shape), want, want.abs() * (4 / 64 + 16) * EPS)


@pytest.mark.gpu
def test_states_and_logits_past_4_gb(om, ctx):
    H, D = 64, 256
    n_slots = (5 << 30) // (H * D * D * 4)
    S = ctx.alloc(n_slots * H * D * D * 4)
    for L in (1, 40):
        g, q, k, v, decay = _linear_inputs([L], H, 1, 1, 1, D, D, "head", L)
        ib, ob = _up(ctx, torch.tensor([n_slots - 1], dtype=torch.int32), torch.tensor([n_slots - 2], dtype=torch.int32))
        bufs = _up(ctx, q, k, v, decay)
        out = ctx.alloc(L * H * D * 4)
        om.linear_attend(ctx, om.linear_states(S, n_slots, H, D, D), out, *bufs[:3], 1, 1, 1, L, bufs[3], 1,
                         _up(ctx, torch.tensor([0, L], dtype=torch.int32))[0], ib, ob)
        want, bound, ends, _ = _linear64(q, k, v, decay, [0, L], torch.zeros(1, H, D, D), D ** -0.5, False)
        c = (8 + 6 * math.sqrt(2 * L + D)) * EPS
        _close(_down(ctx, out, (L, H, D)), want, bound * c + 1e-37)
        # the state, seen by another token that starts from it
        one = torch.zeros(1, 1, D)
        qb, kb = _up(ctx, q[:1], one)
        out = ctx.alloc(H * D * 4)
        om.linear_attend(ctx, om.linear_states(S, n_slots, H, D, D), out, qb, kb, kb, 1, 1, 1, 1,
                         _up(ctx, torch.zeros(H))[0], 1, None, ob, None)
        got = _down(ctx, out, (1, H, D))
        want = (ends[0] * q[0].double()[:, :, None]).sum(1) * D ** -0.5
        _close(got[0], want, (ends[0].abs() * q[0].double().abs()[:, :, None]).sum(1) * D ** -0.5 * 2 * c + 1e-37)
    S.free()
    rows, stride = 1200, 1 << 20
    xb = ctx.alloc(rows * stride * 4)  # zeros
    r = np.zeros(rows, om.SAMPLE_REQUEST)
    r["temperature"], r["top_p"] = 1.0, 1.0
    u = np.linspace(0, 0.999, rows).astype(np.float32)
    rb, ub, tok = ctx.upload(r), ctx.upload(u), ctx.alloc(rows * 4)
    om.sample(ctx, tok, None, xb, rows, 1000, rb, ub, stride=stride)
    xb.free()
    got = ctx.download(tok, np.int32, (rows,))
    assert np.abs(got - u.astype(np.float64) * 1000).max() <= 1.0 and (got == np.floor(u.astype(np.float64) * 1000)).mean() > 0.99

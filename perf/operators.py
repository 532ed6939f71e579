"""Operators of the attention side of a decode step, as cases that can be timed.

  rope     rotary positions of several axes on the query and key heads of some tokens
  append   the same rotation, with K and V stored into the pages of a key-value cache
  attend   one new token of each sequence over its pages; with `score`, the weights that
           every cached token got are added up for the eviction
  evict    every kv head keeps its first, its last and its most attended tokens, in new pages

The cache's pages are [page][kv head][slot of the page][head_dim], in 32, 16 or 8 bits; a
sequence's pages are a row of `table`.  Activations are fp32.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
         "e4m3": torch.float8_e4m3fn}
E4M3_MAX = 448.0


# ---------------------------------------------------------------- cases
def _rope(T, heads, kv, D, pairs, halves=True, interleaved=False, base=1e7):
    """pairs: the rotated pairs of each axis ("24" or "16+24+24")."""
    return {"kind": "rope", "T": T, "heads": heads, "kv": kv, "D": D, "pairs": pairs,
            "halves": halves, "interleaved": interleaved, "base": base}


def _append(T, heads, kv, D, pairs, type, page, halves=True, interleaved=False, base=1e7):
    """A few of the tokens are padding, which is not stored."""
    return dict(_rope(T, heads, kv, D, pairs, halves, interleaved, base), kind="append", type=type,
                page=page)


def _attend(B, heads, kv, D, type, page, len, ragged=False, empty=0, score=False):
    """len: the longest sequence; ragged: the others are shorter; empty: rows without a sequence."""
    return {"kind": "attend", "B": B, "heads": heads, "kv": kv, "D": D, "type": type, "page": page,
            "len": len, "ragged": ragged, "empty": empty, "score": score}


def _evict(B, kv, D, type, page, len, keep, sink, recent, ragged=False):
    return {"kind": "evict", "B": B, "kv": kv, "D": D, "type": type, "page": page, "len": len,
            "keep": keep, "sink": sink, "recent": recent, "ragged": ragged}


def listed():
    return [
        # a decode step's token at this engine's attention shape: 16 heads, 2 kv heads of 256,
        # the first 64 dimensions rotated in adjacent pairs
        dict(_rope(1, 16, 2, 256, "32", halves=False), name="rope_token"),
        # an image's patches in a prompt: time, height and width dealt out over the pairs
        dict(_rope(4099, 32, 8, 128, "24+20+20", interleaved=True, base=1e6), name="rope_image"),
        # a decode batch stores its tokens
        dict(_append(16, 16, 2, 256, "32", "bf16", 16, halves=False), name="append_batch"),
        # a prompt stores its tokens in 8 bits
        dict(_append(8190, 32, 8, 128, "16+24+24", "e4m3", 64), name="append_prompt"),
        # the first tokens of a conversation
        dict(_attend(1, 16, 2, 256, "bf16", 16, 37), name="attend_short"),
        # one conversation with a long context
        dict(_attend(1, 16, 2, 256, "bf16", 16, 131071), name="attend_long"),
        # a serving batch of sequences of all lengths, their weights added up for the eviction
        dict(_attend(64, 32, 8, 128, "f16", 16, 8192, ragged=True, empty=3, score=True),
             name="attend_serving"),
        # the same kind of batch on an 8-bit cache, sixteen heads to a kv head
        dict(_attend(32, 64, 4, 128, "e4m3", 64, 16384, ragged=True), name="attend_8bit"),
        # as many kv heads as heads, 32 bits
        dict(_attend(5, 12, 12, 64, "f32", 8, 2047), name="attend_f32"),
        # heads of a size that is no power of two
        dict(_attend(24, 20, 4, 80, "bf16", 32, 4001, ragged=True, score=True),
             name="attend_80"),
        # one conversation's cache cut to half
        dict(_evict(1, 2, 256, "bf16", 16, 4096, 2048, 4, 512), name="evict_one"),
        # a serving batch's caches cut to a quarter
        dict(_evict(32, 8, 128, "f16", 16, 16384, 4096, 16, 1024, ragged=True),
             name="evict_serving"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "append"] + ["attend"] * 5 + ["evict"] * 2)
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4, 5, 8, 16])
    D = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256, 256])
    type = rng.choice(["f32", "f16", "bf16", "bf16", "e4m3"])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    if kind in ("rope", "append"):
        R = D // 2 if rng.random() < 0.6 else D // 4
        n = rng.randint(1, 4)
        cut = sorted(rng.randint(0, R) for _ in range(n - 1))
        pairs = "+".join(str(b - a) for a, b in zip([0] + cut, cut + [R]))
        T = min(_log(rng, 1, 8190), max(1, (150 << 20) // ((heads + 2 * kv) * D * 4)))
        c = (T, heads, kv, D, pairs)
        more = {"halves": rng.random() < 0.6, "interleaved": rng.random() < 0.5,
                "base": rng.choice([1e4, 1e6, 1e7])}
        return _rope(*c, **more) if kind == "rope" else _append(*c, type, page, **more)
    row = 2 * kv * D * TYPES[type].itemsize
    if kind == "attend":
        B = _log(rng, 1, 256)
        L = min(_log(rng, 1, 131072), max(1, (512 << 20) // (B * row)))
        return _attend(B, heads, kv, D, type, page, L, ragged=rng.random() < 0.6,
                       empty=rng.randint(0, 3) if B > 4 and rng.random() < 0.3 else 0,
                       score=rng.random() < 0.4)
    B = _log(rng, 1, 64)
    L = min(_log(rng, 16, 65536), max(16, (512 << 20) // (B * row)))
    keep = rng.randint(1, L)
    sink = rng.randint(0, min(keep, 32))
    return _evict(B, kv, D, type, page, L, keep, sink, rng.randint(0, (keep - sink) // 2),
                  ragged=rng.random() < 0.6)


def _lens(case):
    """The sequences' lengths: the first is the longest, the last `empty` rows have none."""
    B, L = case["B"], case["len"]
    if case["ragged"]:
        lens = [L] + [1 + int((b * 0.6180339887498949) % 1.0 * (L - 1)) for b in range(1, B)]
    else:
        lens = [L] * B
    e = case.get("empty", 0)
    return lens[:B - e] + [0] * e


def _pairs(case):
    return [int(n) for n in case["pairs"].split("+")]


def work(case):
    kind, kv, D = case["kind"], case["kv"], case["D"]
    if kind in ("rope", "append"):
        T, H, R = case["T"], case["heads"], sum(_pairs(case))
        flops = T * (H + kv) * R * 6
        q, k = T * H * D * 4, T * kv * D * 4
        if kind == "rope":
            return {"bytes": 2 * (q + k), "flops": flops}
        return {"bytes": 2 * (q + k) + 2 * T * kv * D * TYPES[case["type"]].itemsize, "flops": flops}
    b, lens = TYPES[case["type"]].itemsize, _lens(case)
    if kind == "attend":
        H, n = case["heads"], sum(lens)
        return {"bytes": 2 * n * kv * D * b + 8 * len(lens) * H * D +
                (8 * n * kv if case["score"] else 0), "flops": 4 * n * H * D}
    kept = sum(min(n, case["keep"]) for n in lens)
    return {"bytes": kv * (4 * sum(lens) + kept * (4 * D * b + 8)), "flops": kv * sum(lens)}


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _stored(x, type):
    """x as the cache holds it: rounded to nearest; the 8-bit type ends at its largest value."""
    if type == "e4m3":
        x = x.clamp(-E4M3_MAX, E4M3_MAX)
    return x.to(TYPES[type])


def _positions(case, g):
    """[axis][token]: text counts on, on every axis alike; far into a long context."""
    T, n = case["T"], len(_pairs(case))
    t = torch.arange(T, device="cuda", dtype=torch.int32)
    start = int(torch.randint(0, 200000, (1,), generator=g, device="cuda"))
    if n == 1 or T < 64:
        return (start + t).repeat(n, 1).contiguous()
    side = max(1, int(math.sqrt(T)))  # an image: its time, its rows, its columns
    axes = [torch.zeros_like(t), t // side, t % side, t // 7][:n]
    return (start + torch.stack(axes)).contiguous()


def _pool(g, pages, kv, page, D, type):
    """Pages as an engine finds them: every slot holds something, used or left behind."""
    x = torch.empty(pages, kv, page, D, dtype=TYPES[type], device="cuda")
    for i in range(0, pages, 4096):
        x[i:i + 4096] = _stored(_randn(g, min(4096, pages - i), kv, page, D), type)
    return x


def _tensors(case, seed):
    """The inputs of a call."""
    g, kind, kv, D = _gen(seed), case["kind"], case["kv"], case["D"]
    if kind in ("rope", "append"):
        T = case["T"]
        t = {"q": _randn(g, T, case["heads"], D), "k": _randn(g, T, kv, D),
             "positions": _positions(case, g)}
        if kind == "append":
            page = case["page"]
            pages = -(-T // page) + 3
            t["v"] = _randn(g, T, kv, D)
            slots = torch.randperm(pages, generator=g, device="cuda")[:, None] * page + \
                torch.arange(page, device="cuda")
            slots = slots.reshape(-1)[:T].to(torch.int32)
            if T > 8:  # padding
                slots[torch.randint(0, T, (T // 50 + 1,), generator=g, device="cuda")] = -1
            t["slots"] = slots.contiguous()
            # the last page takes the plain form's padding
            t["kp"] = _pool(g, pages + 1, kv, page, D, case["type"])
            t["vp"] = _pool(g, pages + 1, kv, page, D, case["type"])
        return t
    B, page, L = case["B"], case["page"], case["len"]
    width = -(-L // page)
    lens = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")
    t = {"lens": lens}
    if kind == "attend":
        pages = B * width + 1
        ids = torch.randperm(pages, generator=g, device="cuda")[:B * width]
        t["q"] = _randn(g, B, case["heads"], D)
        if case["score"]:
            t["score"] = torch.rand(B, kv, width * page, generator=g, device="cuda")
    else:
        # every sequence's pages, the pages its kept tokens go to, and one for the plain form's padding
        new = -(-case["keep"] // page)
        pages = B * (width + new) + 1
        ids = torch.randperm(pages - 1, generator=g, device="cuda")
        t["dst"] = ids[B * width:].reshape(B, new).to(torch.int32).contiguous()
        ids = ids[:B * width]
        # a few tokens take most of the weight, and many took none: ties
        s = torch.exp(2.0 * _randn(g, B, kv, width * page))
        t["score"] = torch.where(torch.rand(s.shape, generator=g, device="cuda") < 0.1, 0.0, s)
    t["table"] = ids.reshape(B, width).to(torch.int32).contiguous()
    t["kp"] = _pool(g, pages, kv, page, D, case["type"])
    t["vp"] = _pool(g, pages, kv, page, D, case["type"])
    return t


class _State:
    """What a program holds before the call."""


def prepare(case, seed):
    s = _State()
    s.case, s.t = case, _tensors(case, seed)
    s.axis = torch.tensor(_axis_of_pair(case) if "pairs" in case else [], dtype=torch.int64,
                          device="cuda")
    if own:
        _to_buffers(s)
    return s


# ---------------------------------------------------------------- the plain form
def _axis_of_pair(case):
    n = _pairs(case)
    if not case["interleaved"]:
        return [a for a, k in enumerate(n) for _ in range(k)]
    axes = [(i, a) for a, k in enumerate(n) for i in range(k)]  # dealt out in turn
    return [a for _, a in sorted(axes)]


def _rotated(case, x, positions, axis):
    """Angles in 64 bits: a position far into the context leaves fp32 no digits behind its turns."""
    R = sum(_pairs(case))
    p = torch.arange(R, dtype=torch.float64, device="cuda")
    angle = positions[axis].t().double() * case["base"] ** (-p / max(R, 1))  # [T][R]
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    y = x.clone()
    if case["halves"]:
        a, b = x[..., :R], x[..., R:2 * R]
        y[..., :R], y[..., R:2 * R] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., 0:2 * R:2], x[..., 1:2 * R:2]
        y[..., 0:2 * R:2], y[..., 1:2 * R:2] = a * c - b * s, a * s + b * c
    return y


def _rows(pool, table):
    """A sequence's slots in order, in 32 bits: [B][kv][slots][D]."""
    x = pool.view(torch.uint8)[table] if pool.dtype == TYPES["e4m3"] else pool[table]
    B, n, kv, page, D = x.shape
    x = x.permute(0, 2, 1, 3, 4).reshape(B, kv, n * page, D)
    return (x.view(pool.dtype) if pool.dtype == TYPES["e4m3"] else x).float()


def _plain_rope(case, t, axis):
    return {n: _rotated(case, t[n], t["positions"], axis) for n in ("q", "k")}


def _plain_append(case, t, axis):
    r = _plain_rope(case, t, axis)
    pages, page, type = t["kp"].shape[0], case["page"], case["type"]
    slots = torch.where(t["slots"] < 0, (pages - 1) * page, t["slots"])  # padding: the spare page
    for pool, x in ((t["kp"], r["k"]), (t["vp"], t["v"])):
        x = _stored(x, type)
        if type == "e4m3":
            pool, x = pool.view(torch.uint8), x.view(torch.uint8)
        pool[slots // page, :, slots % page] = x
    return {"q": r["q"], "k": t["kp"][:-1], "v": t["vp"][:-1]}


def _plain_attend(case, t, _):
    B, H, kv, D = case["B"], case["heads"], case["kv"], case["D"]
    k, v = _rows(t["kp"], t["table"]), _rows(t["vp"], t["table"])
    on = torch.arange(k.shape[2], device="cuda")[None] < t["lens"][:, None]  # [B][slots]
    v = torch.where(on[:, None, :, None], v, 0.0)
    s = t["q"].view(B, kv, H // kv, D) @ k.transpose(2, 3) * (1.0 / math.sqrt(D))
    s = torch.where(on[:, None, None], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    w = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    r = {"out": (w @ v).reshape(B, H, D)}
    if case["score"]:
        r["score"] = torch.where(on[:, None], t["score"] + w.sum(2), 0.0)
    return r


def _plain_evict(case, t, _):
    kv, page, keep = case["kv"], case["page"], case["keep"]
    lens, score = t["lens"].long()[:, None, None], t["score"]
    B, _, n = score.shape
    i = torch.arange(n, device="cuda").expand(B, kv, n)
    stays = (i < case["sink"]) | (i >= lens - case["recent"])
    order = torch.where(i < lens, torch.where(stays, math.inf, score), -math.inf)
    best = torch.argsort(order, dim=-1, descending=True, stable=True)  # ties: the lowest slot
    rank = torch.empty_like(best).scatter_(-1, best, i)
    kept = (rank < keep) & (i < lens)
    src = torch.argsort((~kept).to(torch.uint8), dim=-1, stable=True)[..., :keep]  # in order
    count = lens.clamp_max(keep)
    j = torch.arange(src.shape[-1], device="cuda").expand(B, kv, -1)
    on = j < count
    b = torch.arange(B, device="cuda")[:, None, None]
    h = torch.arange(kv, device="cuda")[None, :, None]
    spare = t["kp"].shape[0] - 1
    from_page = t["table"].long()[b, torch.where(on, src // page, 0)]
    to_page = torch.where(on, t["dst"].long()[b, j // page], spare)
    for pool in (t["kp"], t["vp"]):
        pool = pool.view(torch.uint8) if case["type"] == "e4m3" else pool
        pool[to_page, h, j % page] = pool[from_page, h, src % page]
    return {"kept": torch.where(on, src, -1).int(), "lens": count.reshape(-1).int(),
            "score": torch.where(on, score.gather(-1, src), 0.0),
            "k": t["kp"][:-1], "v": t["vp"][:-1]}


def run(s):
    case, t = s.case, s.t
    if own:
        return _call(s)
    return {"rope": _plain_rope, "append": _plain_append, "attend": _plain_attend,
            "evict": _plain_evict}[case["kind"]](case, t, s.axis)


# ---------------------------------------------------------------- the framework's calls
_context = None


def _library():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    if os.path.join(root, "ornith-flight_amd") not in sys.path:
        sys.path.insert(0, os.path.join(root, "ornith-flight_amd"))
    import ornith_moe
    return ornith_moe


def _ctx():
    """The process's context: one stream, as an engine has."""
    global _context
    if _context is None:
        torch.cuda.init()
        _context = _library().Context()
    return _context


class _Device:
    """A device buffer of the framework, freed with its last user; `tensor` shows it and keeps it."""

    def __init__(self, nbytes):
        self.buf = _ctx().alloc(nbytes)
        self.ptr = self.buf.ptr

    def tensor(self, shape, dtype):
        n = math.prod(shape) * dtype.itemsize
        self.__cuda_array_interface__ = {
            "shape": (n,), "typestr": "|u1", "version": 2, "strides": None,
            "data": (_library().lib().gpu_device_ptr(_ctx().ptr, self.ptr), False)}
        return torch.as_tensor(self, device="cuda").view(dtype).view(shape)

    def __del__(self):
        c = _ctx()
        c.sync()
        c._bufs = [b for b in c._bufs if b is not self.buf]
        self.buf.free()


def _buffer(x):
    b = _Device(x.numel() * x.element_size())
    b.tensor(tuple(x.shape), x.dtype).copy_(x)
    return b


def _result(*shape, dtype=torch.float32):
    b = _Device(math.prod(shape) * dtype.itemsize)
    return b, b.tensor(shape, dtype)


def _to_buffers(s):
    """The inputs in the framework's buffers, room for the results, and the calls' descriptions."""
    om, case, t, kind = _library(), s.case, s.t, s.case["kind"]
    s.b = {n: _buffer(x) for n, x in t.items()}
    s.result = {}

    def out(name, *shape, dtype=torch.float32):
        s.b[name + "_out"], s.result[name] = _result(*shape, dtype=dtype)

    if kind in ("rope", "append"):
        s.rope = om.rope_axes(_pairs(case), case["base"], halves=case["halves"],
                              interleaved=case["interleaved"])
        out("q", *t["q"].shape)
    if kind == "rope":
        out("k", *t["k"].shape)
    else:
        kp = t["kp"]
        s.pages = om.kv_pages(s.b["kp"], s.b["vp"], case["type"], kp.shape[0], case["page"],
                              case["kv"], case["D"])
    if kind in ("append", "evict"):
        for n in ("k", "v"):
            s.result[n] = s.b[n + "p"].tensor(tuple(kp.shape), kp.dtype)[:-1]
    if kind == "attend":
        out("out", *t["q"].shape)
        if case["score"]:
            out("score", *t["score"].shape)
        s.opts = om.attend_opts(max_len=case["len"], flags=om.KV_ASYNC,
                                **({"score_in": s.b["score"], "score_out": s.b["score_out"],
                                    "score_stride": t["score"].shape[2], "decay": 1.0}
                                   if case["score"] else {}))
    if kind == "evict":
        B, kv, keep = case["B"], case["kv"], case["keep"]
        out("kept", B, kv, keep, dtype=torch.int32)
        out("lens", B, dtype=torch.int32)
        out("score", B, kv, keep)
        s.opts = om.evict_opts(keep=keep, sink=case["sink"], recent=case["recent"],
                               max_len=case["len"], flags=om.KV_ASYNC)
    s.shape = {n: tuple(x.shape) for n, x in t.items()}
    s.t = None


def _call(s):
    om, c, case, b = _library(), _ctx(), s.case, s.b
    kind = case["kind"]
    if kind == "rope":
        om.rope_axes_apply(c, b["q_out"], b["k_out"], b["q"], b["k"], case["T"], case["heads"],
                           case["kv"], case["D"], b["positions"], s.rope, flags=om.KV_ASYNC)
    elif kind == "append":
        om.kv_append(c, s.pages, b["k"], b["v"], case["T"], b["slots"], b["q_out"], b["q"],
                     case["heads"], b["positions"], s.rope, flags=om.KV_ASYNC)
    elif kind == "attend":
        om.kv_attend(c, s.pages, b["out_out"], b["q"], case["B"], case["heads"], b["table"],
                     s.shape["table"][1], b["lens"], s.opts)
    else:
        om.kv_evict(c, s.pages, case["B"], b["table"], s.shape["table"][1], b["lens"], b["score"],
                    s.shape["score"][2], b["dst"], s.shape["dst"][1], b["lens_out"],
                    b["score_out"], case["keep"], b["kept_out"], s.opts)
    return s.result


# ---------------------------------------------------------------- 64-bit results
def _turn(case, x, positions):
    """x rotated as complex numbers."""
    n, T = _pairs(case), case["T"]
    R = sum(n)
    y = x.double().clone()
    left, axis = list(n), []
    while len(axis) < R:  # the pairs' axes: runs, or one pair of each axis in turn
        for a in range(len(n)):
            take = min(left[a], 1) if case["interleaved"] else left[a]
            axis += [a] * take
            left[a] -= take
    for p in range(R):
        i, j = (p, p + R) if case["halves"] else (2 * p, 2 * p + 1)
        angle = positions[axis[p]].double() * math.exp(-p / R * math.log(case["base"]))
        z = torch.complex(x[..., i].double(), x[..., j].double()) * \
            torch.polar(torch.ones_like(angle), angle).view(T, 1)
        y[..., i], y[..., j] = z.real, z.imag
    return y


def exact(case, seed):
    kind, t = case["kind"], _tensors(case, seed)
    if kind == "rope":
        return {"q": _turn(case, t["q"], t["positions"]), "k": _turn(case, t["k"], t["positions"])}
    if kind == "append":
        r = {"q": _turn(case, t["q"], t["positions"])}
        on = t["slots"] >= 0
        at = t["slots"][on].long()
        for name, pool, x in (("k", t["kp"], _turn(case, t["k"], t["positions"])),
                              ("v", t["vp"], t["v"].double())):
            y = pool[:-1].double()
            y[at // case["page"], :, at % case["page"]] = x[on]
            r[name] = y
        return r
    if kind == "evict":
        return None  # the outputs are copies and whole numbers
    B, H, kv, D, page = case["B"], case["heads"], case["kv"], case["D"], case["page"]
    r = {"out": torch.zeros(B, H, D, dtype=torch.float64, device="cuda")}
    if case["score"]:
        r["score"] = torch.zeros(t["score"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lens(case)):
        if not n:
            continue
        ids = t["table"][b, :-(-n // page)].long()
        for h in range(kv):
            k, v = (pool.view(torch.uint8)[ids, h].view(pool.dtype).reshape(-1, D)[:n].double()
                    for pool in (t["kp"], t["vp"]))
            for q in range(h * H // kv, (h + 1) * H // kv):
                w = torch.softmax((k * t["q"][b, q].double()).sum(1) / math.sqrt(D), 0)
                r["out"][b, q] = (w[:, None] * v).sum(0)
                if case["score"]:
                    r["score"][b, h, :n] += w
            if case["score"]:
                r["score"][b, h, :n] += t["score"][b, h, :n].double()
    return r

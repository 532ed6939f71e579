"""Operators of a hybrid stack's decode loop, as cases that can be timed.

  heads   norms of the query and key heads (root mean square or length) and the rotation of
          rotary positions, in one pass; with a cache, K and V go to their pages in it, too
  linear  linear attention with a decay for each head: prompts, or one token per sequence;
          every sequence goes on from a state in a slot and leaves its own in another
  sample  a token for each row of logits from a random number, by temperature, top-k, top-p
          and min-p

Activations, states and logits are fp32.  The cache's pages are [page][kv head][slot of the
page][head_dim], in 32, 16 or 8 bits.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
         "e4m3": torch.float8_e4m3fn}
E4M3_MAX = 448.0
CHUNK = 64  # tokens that the plain linear attention takes at a time

# what the requests of one batch ask for: temperature, top-k, top-p, min-p
REQUESTS = [(0.7, 20, 0.8, 0.0), (1.0, 0, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.2, 0, 1.0, 0.05),
            (0.8, 40, 0.95, 0.05), (1.0, 0, 1.0, 0.0), (0.6, 1000, 0.9, 0.0)]


# ---------------------------------------------------------------- cases
def _heads(T, heads, kv, D, pairs, norm="rms", weights="one", type="", page=16, halves=True,
           base=1e7):
    """pairs: the rotated pairs of each axis ("16+24+24"; "": no rotation).  weights: "one" for
    all heads, "each" head's own, or "no".  type: of the cache; "": none is written."""
    return {"kind": "heads", "T": T, "heads": heads, "kv": kv, "D": D, "pairs": pairs, "norm": norm,
            "weights": weights, "type": type, "page": page, "halves": halves, "base": base}


def _linear(B, len, qk, heads, dk, dv, gates=True, complement=False, ragged=False, begins=False):
    """len: the longest sequence (1 for all: a decode step); qk: heads of Q and K, each read by
    heads / qk heads.  gates: a decay for each token; else one that stays.  begins: half of the
    sequences have no state yet."""
    return {"kind": "linear", "B": B, "len": len, "qk": qk, "heads": heads, "dk": dk, "dv": dv,
            "gates": gates, "complement": complement, "ragged": ragged, "begins": begins}


def _sample(rows, vocab, request=-1, spread=2.5, grid=False, masked=0.0):
    """request: all rows' in REQUESTS, -1: they take turns.  grid: logits of a bf16 product, with
    many equal ones; masked: the share of tokens that a grammar rules out."""
    return {"kind": "sample", "rows": rows, "vocab": vocab, "request": request, "spread": spread,
            "grid": grid, "masked": masked}


def listed():
    return [
        # a decode step's token at this engine's attention shape: 16 heads, 2 kv heads of 256, the
        # first 64 dimensions rotated in adjacent pairs
        dict(_heads(1, 16, 2, 256, "32", type="bf16", halves=False), name="heads_token"),
        # a prompt with an image: normed, rotated on three axes and stored
        dict(_heads(8190, 32, 8, 128, "16+24+24", type="f16", page=64, base=1e6),
             name="heads_prompt"),
        # queries and keys of unit length for the linear attention, no rotation
        dict(_heads(4099, 16, 16, 128, "", norm="l2", weights="no"), name="heads_unit"),
        # one conversation's next token
        dict(_linear(1, 1, 16, 32, 128, 128), name="linear_token"),
        # a serving batch's next tokens
        dict(_linear(64, 1, 16, 32, 128, 128), name="linear_batch"),
        # one long prompt, as many heads of Q and K as of V
        dict(_linear(1, 8191, 16, 16, 128, 128, begins=True), name="linear_prompt"),
        # prompts of all lengths, or parts of them, with decays that stay
        dict(_linear(24, 1501, 16, 32, 128, 128, gates=False, ragged=True, begins=True),
             name="linear_ragged"),
        # a few short prompts of smaller heads that are no power of two
        dict(_linear(5, 333, 6, 12, 96, 80, complement=True), name="linear_96"),
        # one conversation's token
        dict(_sample(1, 248320, 0), name="sample_token"),
        # a serving batch whose requests ask for different things
        dict(_sample(64, 248320), name="sample_batch"),
        # all tokens of flat rows count; a vocabulary of no round size
        dict(_sample(16, 100003, 1, spread=0.5, grid=True), name="sample_flat"),
        # many rows of a smaller vocabulary, most of it ruled out
        dict(_sample(256, 32000, 3, masked=0.9), name="sample_small"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["heads"] * 3 + ["linear"] * 5 + ["sample"] * 4)
    if kind == "heads":
        kv = rng.choice([1, 2, 4, 8, 16])
        heads = min(64, kv * rng.choice([1, 2, 4, 5, 8]))
        D = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256, 256])
        R = rng.choice([0, D // 4, D // 2, D // 2])
        cut = sorted(rng.randint(0, R) for _ in range(rng.randint(0, 2)))
        pairs = "+".join(str(b - a) for a, b in zip([0] + cut, cut + [R])) if R else ""
        T = min(_log(rng, 1, 8190), max(1, (150 << 20) // ((heads + 2 * kv) * D * 4)))
        return _heads(T, heads, kv, D, pairs, norm=rng.choice(["rms", "rms", "l2"]),
                      weights=rng.choice(["one", "one", "each", "no"]),
                      type=rng.choice(["", "", "f32", "f16", "bf16", "e4m3"]),
                      page=rng.choice([8, 16, 64]), halves=rng.random() < 0.6,
                      base=rng.choice([1e4, 1e6, 1e7]))
    if kind == "linear":
        dk = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256])
        dv = rng.choice([dk, dk, dk, 64, 128, 200])
        qk = rng.choice([1, 2, 4, 6, 8, 16])
        heads = qk * rng.choice([1, 1, 2, 4])
        step = rng.random() < 0.35
        B = min(_log(rng, 1, 256), max(1, (128 << 20) // (heads * dk * dv * 4)))
        L = 1 if step else min(_log(rng, 2, 16384), max(2, (1 << 31) // (B * heads * dk * dv)),
                               max(2, (64 << 20) // (B * heads * (dk + dv))))
        return _linear(B, L, qk, heads, dk, dv, gates=rng.random() < 0.6,
                       complement=rng.random() < 0.3, ragged=not step and rng.random() < 0.6,
                       begins=rng.random() < 0.5)
    rows = _log(rng, 1, 256)
    vocab = min(_log(rng, 300, 248320), max(300, (64 * 248320) // rows))
    return _sample(rows, vocab, rng.randint(-1, len(REQUESTS) - 1),
                   spread=rng.choice([0.3, 1.0, 2.5, 4.0]), grid=rng.random() < 0.3,
                   masked=rng.choice([0.0, 0.0, 0.5, 0.9]))


def _lens(case):
    """The sequences' lengths: the first is the longest, and one of several is empty."""
    B, L = case["B"], case["len"]
    if not case["ragged"]:
        return [L] * B
    lens = [L] + [1 + int((b * 0.6180339887498949) % 1.0 * (L - 1)) for b in range(1, B)]
    if B > 2:
        lens[B // 2] = 0
    return lens


def _pairs(case):
    return [int(n) for n in case["pairs"].split("+")] if case["pairs"] else []


def work(case):
    kind = case["kind"]
    if kind == "heads":
        T, H, kv, D = case["T"], case["heads"], case["kv"], case["D"]
        flops = T * (H + kv) * (5 * D + 6 * sum(_pairs(case)))
        rows = 8 * T * H * D  # queries in and out
        if case["type"]:
            return {"bytes": rows + 2 * T * kv * D * (4 + TYPES[case["type"]].itemsize),
                    "flops": flops}
        return {"bytes": rows + 8 * T * kv * D, "flops": flops}
    if kind == "linear":
        lens, H, dk, dv = _lens(case), case["heads"], case["dk"], case["dv"]
        T, known = sum(lens), sum(_continues(case))
        n = T * (2 * case["qk"] * dk + 2 * H * dv + (H if case["gates"] else 0))
        return {"bytes": 4 * (n + (known + len(lens)) * H * dk * dv), "flops": 4 * T * H * dk * dv}
    n = case["rows"] * case["vocab"]
    return {"bytes": 4 * n + 28 * case["rows"], "flops": 8 * n}


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


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
    axes = [torch.zeros_like(t), t // side, t % side][:n]
    return (start + torch.stack(axes)).contiguous()


def _heads_tensors(case, g):
    T, H, kv, D = case["T"], case["heads"], case["kv"], case["D"]
    # projections' outputs: some tokens are larger than others
    t = {"q": _randn(g, T, H, D) * torch.exp(_randn(g, T, 1, 1)),
         "k": _randn(g, T, kv, D) * torch.exp(_randn(g, T, 1, 1))}
    if case["pairs"]:
        t["positions"] = _positions(case, g)
    if case["weights"] != "no":
        each = case["weights"] == "each"
        t["qw"] = 1.0 + 0.3 * _randn(g, H if each else 1, D)
        t["kw"] = 1.0 + 0.3 * _randn(g, kv if each else 1, D)
    if case["type"]:
        page = case["page"]
        pages = -(-T // page) + 3
        t["v"] = _randn(g, T, kv, D)
        slots = torch.randperm(pages, generator=g, device="cuda")[:, None] * page + \
            torch.arange(page, device="cuda")
        slots = slots.reshape(-1)[:T].to(torch.int32)
        if T > 8:  # padding, which is not stored
            slots[torch.randint(0, T, (T // 50 + 1,), generator=g, device="cuda")] = -1
        t["slots"] = slots.contiguous()
        for n in ("kp", "vp"):  # the last page takes the plain form's padding
            t[n] = _stored(_randn(g, pages + 1, kv, page, D), case["type"])
    return t


def _continues(case):
    """Which sequences go on from a state."""
    return [not (case["begins"] and b % 2 == 0) for b in range(case["B"])]


def _linear_tensors(case, g):
    B, H, qk, dk, dv = case["B"], case["heads"], case["qk"], case["dk"], case["dv"]
    lens = _lens(case)
    T = sum(lens)
    unit = torch.nn.functional.normalize
    t = {"q": unit(_randn(g, T, qk, dk), dim=-1) * math.sqrt(dk),
         "k": unit(_randn(g, T, qk, dk), dim=-1), "v": _randn(g, T, H, dv)}
    if case["gates"]:
        # a rate for each head times a step for each token: from nearly none to all at once
        rate = torch.exp(-5.0 + 7.0 * _rand(g, H))
        t["decay"] = -rate * torch.nn.functional.softplus(_randn(g, T, H))
    else:
        t["decay"] = -torch.exp2(-8.0 * (torch.arange(H, device="cuda") + _rand(g, 1)) / H)
    t["starts"] = torch.tensor([sum(lens[:b]) for b in range(B + 1)], dtype=torch.int32,
                               device="cuda")
    ids = torch.randperm(2 * B + 1, generator=g, device="cuda").to(torch.int32)
    goes_on = torch.tensor(_continues(case), device="cuda")
    t["slots_in"] = torch.where(goes_on, ids[:B], -1).contiguous()
    t["slots_out"] = ids[B:2 * B].contiguous()
    t["states"] = _randn(g, 2 * B + 1, H, dk, dv) * 0.5
    return t


def _sample_tensors(case, g):
    rows, V = case["rows"], case["vocab"]
    x = _randn(g, rows, V) * case["spread"]
    # a few tokens stand out, as the likely next ones do
    likely = torch.randint(0, V, (rows, 40), generator=g, device="cuda")
    x.scatter_add_(1, likely, 2.0 * case["spread"] * -torch.log1p(-_rand(g, rows, 40)))
    if case["grid"]:
        x = x.bfloat16().float()
    if case["masked"]:
        x = torch.where(_rand(g, rows, V) < case["masked"], -math.inf, x)
    r = case["request"]
    asked = [REQUESTS[(b if r < 0 else r) % len(REQUESTS)] for b in range(rows)]
    words = np.empty((rows, 4), np.int32)  # temperature, top-k, top-p, min-p as they lie in memory
    for i, d in enumerate((np.float32, np.int32, np.float32, np.float32)):
        words[:, i] = np.array([a[i] for a in asked], d).view(np.int32)
    return {"logits": x, "requests": torch.from_numpy(words).cuda(), "u": _rand(g, rows)}


def _tensors(case, seed):
    """The inputs of a call."""
    return {"heads": _heads_tensors, "linear": _linear_tensors,
            "sample": _sample_tensors}[case["kind"]](case, _gen(seed))


class _State:
    """What a program holds before the call."""


def prepare(case, seed):
    s = _State()
    s.case, s.t, s.plan = case, _tensors(case, seed), {}
    if case["kind"] == "heads":
        axis = [a for a, k in enumerate(_pairs(case)) for _ in range(k)]
        s.plan["axis"] = torch.tensor(axis, dtype=torch.int64, device="cuda")
    elif case["kind"] == "linear":
        s.plan.update(_chunks(case))
    if own:
        _to_buffers(s)
    return s


# ---------------------------------------------------------------- the plain form
def _normed(case, x, w):
    ss = (x * x).sum(-1, keepdim=True)
    if case["norm"] == "rms":
        ss = ss / case["D"]
    x = x / torch.sqrt(ss + 1e-6)
    return x if w is None else x * w


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


def _plain_heads(case, t, plan):
    r = {n: _normed(case, t[n], t.get(n + "w")) for n in ("q", "k")}
    if case["pairs"]:
        r = {n: _rotated(case, x, t["positions"], plan["axis"]) for n, x in r.items()}
    if not case["type"]:
        return r
    pages, page, type = t["kp"].shape[0], case["page"], case["type"]
    slots = torch.where(t["slots"] < 0, (pages - 1) * page, t["slots"])  # padding: the spare page
    for pool, x in ((t["kp"], r["k"]), (t["vp"], t["v"])):
        x = _stored(x, type)
        if type == "e4m3":
            pool, x = pool.view(torch.uint8), x.view(torch.uint8)
        pool[slots // page, :, slots % page] = x
    return {"q": r["q"], "k": t["kp"][:-1], "v": t["vp"][:-1]}


def _chunks(case):
    """Where the tokens lie in rows of whole chunks, a row for each sequence."""
    lens = _lens(case)
    n = max(1, -(-max(lens) // CHUNK)) if max(lens) > 1 else 1
    c = CHUNK if max(lens) > 1 else 1
    at = torch.zeros(len(lens), n * c, dtype=torch.int64)
    on = torch.zeros(len(lens), n * c, dtype=torch.bool)
    start = 0
    for b, m in enumerate(lens):
        at[b, :m] = torch.arange(start, start + m)
        on[b, :m] = True
        start += m
    return {"at": at.cuda(), "on": on.cuda(), "n": n, "c": c}


def _plain_linear(case, t, plan):
    """All chunks' products at once, and the states from chunk to chunk; the decays' sums in 64 bits."""
    B, H, dk, dv, n, c = (case["B"], case["heads"], case["dk"], case["dv"], plan["n"], plan["c"])
    at, on = plan["at"], plan["on"]

    def rows(x, heads):  # [T][heads][...] as [B][H][chunk][token][...]
        x = torch.where(on.view(B, n * c, *[1] * (x.dim() - 1)), x[at], 0.0)
        x = x.repeat_interleave(H // heads, dim=2) if heads < H else x
        return x.view(B, n, c, *x.shape[2:]).movedim(3, 1)

    q, k, v = rows(t["q"], case["qk"]), rows(t["k"], case["qk"]), rows(t["v"], H)
    g = t["decay"].double()
    g = g.expand(t["q"].shape[0], H) if g.dim() == 1 else g
    g = rows(g, H)  # [B][H][n][c]
    if case["complement"]:
        k = k * torch.where(on.view(B, 1, n, c), -torch.expm1(g), 0.0).float()[..., None]
    G = g.cumsum(-1)
    causal = torch.ones(c, c, dtype=torch.bool, device="cuda").tril()
    D = torch.where(causal, G[..., :, None] - G[..., None, :], -math.inf).exp().float()
    scale = 1.0 / math.sqrt(dk)
    out = ((q @ k.transpose(-1, -2)) * D) @ v
    left = (G[..., -1:] - G).exp().float()[..., None]
    add = (k * left).transpose(-1, -2) @ v  # what each chunk adds to the state
    keep = G[..., -1].exp().float()[..., None, None]
    slots = t["slots_in"].long()
    S = torch.where(slots.view(B, 1, 1, 1) < 0, 0.0, t["states"][slots.clamp_min(0)])
    before = []
    for i in range(n):
        before.append(S)
        S = S * keep[:, :, i] + add[:, :, i]
    out = (out + (q * G.exp().float()[..., None]) @ torch.stack(before, 2)) * scale
    t["states"][t["slots_out"].long()] = S
    out = out.movedim(1, 3).reshape(B, n * c, H, dv)
    return {"out": out[on], "states": t["states"]}


def _plain_sample(case, t, _):
    """Weights and their sums in 64 bits: a token next to a border is on one side of it."""
    x = t["logits"]
    T, min_p = t["requests"][:, 0].view(torch.float32), t["requests"][:, 3].view(torch.float32)
    top_k, top_p = t["requests"][:, 1], t["requests"][:, 2].view(torch.float32)
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)  # ties: the lowest token
    i = torch.arange(x.shape[1], device="cuda")
    greedy = T == 0
    w = torch.exp((x - x[:, :1]).double() / torch.where(greedy, 1.0, T).double()[:, None])
    w = torch.where(greedy[:, None] & (i > 0), 0.0, w)
    w = torch.where((top_k[:, None] > 0) & (i >= top_k[:, None]), 0.0, w)
    c = w.cumsum(-1)
    before = c - w  # of the more likely tokens
    w = torch.where((before < top_p.double()[:, None] * c[:, -1:]) | (i == 0), w, 0.0)
    w = torch.where(w >= min_p.double()[:, None], w, 0.0)
    c = w.cumsum(-1)
    pick = (c <= t["u"].double()[:, None] * c[:, -1:]).sum(-1, keepdim=True)
    return {"token": order.gather(1, pick)[:, 0].int(),
            "prob": (w.gather(1, pick) / c[:, -1:])[:, 0].float()}


def run(s):
    if own:
        return _call(s)
    return {"heads": _plain_heads, "linear": _plain_linear,
            "sample": _plain_sample}[s.case["kind"]](s.case, s.t, s.plan)


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


def _to_buffers(s):
    """The inputs in the framework's buffers, room for the results, and the calls' descriptions."""
    om, case, t = _library(), s.case, s.t
    s.b = {n: _buffer(x) for n, x in t.items()}
    s.result, s.opts = {}, None

    def out(name, *shape, dtype=torch.float32):
        s.b[name + "_out"] = _Device(math.prod(shape) * dtype.itemsize)
        s.result[name] = s.b[name + "_out"].tensor(shape, dtype)

    if case["kind"] == "heads":
        s.rope = om.rope_axes(_pairs(case), case["base"], halves=case["halves"]) \
            if case["pairs"] else None
        s.norm = om.head_norm(case["norm"], 1e-6, s.b.get("qw"), s.b.get("kw"),
                              per_head=case["weights"] == "each")
        out("q", *t["q"].shape)
        if case["type"]:
            kp = t["kp"]
            s.pages = om.kv_pages(s.b["kp"], s.b["vp"], case["type"], kp.shape[0], case["page"],
                                  case["kv"], case["D"])
            for n in ("k", "v"):
                s.result[n] = s.b[n + "p"].tensor(tuple(kp.shape), kp.dtype)[:-1]
        else:
            out("k", *t["k"].shape)
    elif case["kind"] == "linear":
        out("out", t["v"].shape[0], case["heads"], case["dv"])
        s.result["states"] = s.b["states"].tensor(tuple(t["states"].shape), torch.float32)
        s.states = om.linear_states(s.b["states"], t["states"].shape[0], case["heads"], case["dk"],
                                    case["dv"])
        s.opts = om.linear_opts(per_token=case["gates"], complement=case["complement"],
                                max_len=case["len"], flags=om.KV_ASYNC)
        s.n_tokens = t["v"].shape[0]
    else:
        out("token", case["rows"], dtype=torch.int32)
        out("prob", case["rows"])
    s.t = s.plan = None


def _call(s):
    om, c, case, b = _library(), _ctx(), s.case, s.b
    if case["kind"] == "heads":
        if case["type"]:
            om.norm_kv_append(c, s.pages, b["k"], b["v"], case["T"], b["slots"], b["q_out"], b["q"],
                              case["heads"], s.norm, b.get("positions"), s.rope, flags=om.KV_ASYNC)
        else:
            om.norm_rope_axes(c, b["q_out"], b["k_out"], b["q"], b["k"], case["T"], case["heads"],
                              case["kv"], case["D"], s.norm, b.get("positions"), s.rope,
                              flags=om.KV_ASYNC)
    elif case["kind"] == "linear":
        step = case["len"] == 1 and not case["ragged"]
        om.linear_attend(c, s.states, b["out_out"], b["q"], b["k"], b["v"], case["qk"], case["qk"],
                         case["heads"], s.n_tokens, b["decay"], case["B"],
                         None if step else b["starts"], b["slots_in"], b["slots_out"], s.opts)
    else:
        om.sample(c, b["token_out"], b["prob_out"], b["logits"], case["rows"], case["vocab"],
                  b["requests"], b["u"], flags=om.KV_ASYNC)
    return s.result


# ---------------------------------------------------------------- 64-bit results
def _exact_heads(case, t):
    def one(x, w):
        x = x.double()
        y = x / torch.sqrt(torch.linalg.vecdot(x, x) / (case["D"] if case["norm"] == "rms" else 1)
                           + 1e-6)[..., None]
        y = y if w is None else y * w.double()
        z, R = y.clone(), sum(_pairs(case))
        axes = [a for a, n in enumerate(_pairs(case)) for _ in range(n)]
        for p, a in enumerate(axes):  # turned as complex numbers
            i, j = (p, p + R) if case["halves"] else (2 * p, 2 * p + 1)
            angle = t["positions"][a].double() * math.exp(-p / R * math.log(case["base"]))
            turned = torch.complex(y[..., i], y[..., j]) * \
                torch.polar(torch.ones_like(angle), angle)[:, None]
            z[..., i], z[..., j] = turned.real, turned.imag
        return z

    r = {"q": one(t["q"], t.get("qw")), "k": one(t["k"], t.get("kw"))}
    if not case["type"]:
        return r
    on = t["slots"] >= 0
    at = t["slots"][on].long()
    for name, pool, x in (("k", t["kp"], r["k"]), ("v", t["vp"], t["v"].double())):
        y = pool[:-1].double()
        y[at // case["page"], :, at % case["page"]] = x[on]
        r[name] = y
    return r


def _exact_linear(case, t):
    """Token by token."""
    B, H, lens = case["B"], case["heads"], _lens(case)
    starts = t["starts"].tolist()
    states = t["states"].double()
    out = torch.zeros(sum(lens), H, case["dv"], dtype=torch.float64, device="cuda")
    a = torch.exp(t["decay"].double()).expand(sum(lens), H)
    order = sorted(range(B), key=lambda b: -lens[b])  # the longest first
    slots = t["slots_in"].tolist()
    S = torch.stack([states[slots[b]] if slots[b] >= 0 else torch.zeros_like(states[0])
                     for b in order])
    for i in range(max(lens)):
        n = sum(m > i for m in lens)
        at = torch.tensor([starts[b] + i for b in order[:n]], device="cuda")
        q, k = (t[x][at].double().repeat_interleave(H // case["qk"], dim=1) for x in ("q", "k"))
        f = a[at][..., None, None]
        kv = k[..., None] * t["v"][at].double()[:, :, None]
        S[:n] = S[:n] * f + (kv * (1.0 - f) if case["complement"] else kv)
        out[at] = (S[:n] * q[..., None]).sum(2) / math.sqrt(case["dk"])
    states[t["slots_out"].long()[torch.tensor(order, device="cuda")]] = S
    return {"out": out, "states": states}


def _exact_sample(case, t):
    tokens, probs = [], []
    for x, words, u in zip(t["logits"].cpu().numpy(), t["requests"].cpu().numpy(),
                           t["u"].cpu().numpy().astype(np.float64)):
        T, _, top_p, min_p = (float(f) for f in words.view(np.float32))
        order = np.lexsort((np.arange(len(x)), -x))
        if T == 0:
            order = order[:1]
        if words[1] > 0:
            order = order[:words[1]]
        w = np.exp((x[order].astype(np.float64) - float(x[order[0]])) / (T or 1.0))
        at = np.searchsorted(np.cumsum(w), top_p * np.cumsum(w)[-1]) + 1
        w = w[:max(1, min(at, len(w)))]
        w = w[w >= min_p]
        c = np.cumsum(w)
        i = min(np.searchsorted(c, u * c[-1], side="right"), len(w) - 1)
        tokens.append(order[i])
        probs.append(w[i] / c[-1])
    return {"token": torch.tensor(np.array(tokens, np.int32), device="cuda"),
            "prob": torch.tensor(probs, dtype=torch.float64, device="cuda")}


def exact(case, seed):
    t = _tensors(case, seed)
    return {"heads": _exact_heads, "linear": _exact_linear,
            "sample": _exact_sample}[case["kind"]](case, t)

"""Work cases of the attention-cache operators: rotary positions with several
axes (ofb.rope), the same with the rotated key and its value written to a
paged cache (ofb.rope_append), attention of one new token over that cache
(ofb.attn_decode) and eviction from it by accumulated attention weight
(ofb.kv_evict).

`listed()` names the cases, `draw()` gives more of the same ranges, `prepare()`
makes one case's tensors on the GPU, `run()` makes one pass: the plain torch
form, or with `own` set the calls of the package's binding. `work()` counts
what a pass cannot do without and `exact()` restates the result in 64 bits.

The cache of one layer: k and v [n_pages, kv heads, page, head_dim] in bf16 or
fp16, per entry an accumulated weight (f32) and an order number (int32) laid
out alike, and a page table [sequences, pages of a sequence], -1 where a
sequence has no page.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # image and video patches: time, height and width each with frequencies of their own, neighbouring elements paired
        dict(name="rope-image", op="rope", tokens=257, heads=16, dim=64, rot=64, axes="2d", io="bf16"),
        dict(name="rope-video", op="rope", tokens=16383, heads=16, dim=128, rot=128, axes="3d", io="bf16"),
        # one new token of one sequence: the latency of a decode step
        dict(name="append-one", op="append", tokens=1, seqs=1, start=517, heads=16, kv=2, dim=128, rot=128, axes="text",
             page=16, io="f32", cache="bf16"),
        # one new token of each of 96 sequences, a quarter of the head rotated, axes dealt in turn
        dict(name="append-batch", op="append", tokens=96, seqs=96, start=1000, heads=16, kv=2, dim=256, rot=64, axes="dealt",
             page=64, io="f32", cache="f16"),
        # three prompts' chunks at once, time / height / width sections
        dict(name="append-prompt", op="append", tokens=8190, seqs=3, start=77, heads=32, kv=8, dim=128, rot=128, axes="blocks",
             page=32, io="bf16", cache="bf16"),
        # a short chat, f32 activations as the layer's other operators have them
        dict(name="attend-one", op="attend", seqs=1, lo=517, hi=517, heads=16, kv=2, dim=128, page=16, io="f32", cache="bf16", acc=False),
        # one long document
        dict(name="attend-long", op="attend", seqs=1, lo=131071, hi=131071, heads=16, kv=2, dim=128, page=64, io="bf16", cache="bf16", acc=False),
        # a ragged batch that also keeps its attention weights for eviction
        dict(name="attend-weights", op="attend", seqs=48, lo=1, hi=8191, heads=32, kv=8, dim=128, page=32, io="f32", cache="bf16", acc=True),
        # the largest: 24 long sequences, wide heads
        dict(name="attend-wide", op="attend", seqs=24, lo=8000, hi=40000, heads=16, kv=2, dim=256, page=64, io="f16", cache="f16", acc=False),
        # the cache of one sequence is one page over its budget
        dict(name="evict-page", op="evict", seqs=1, lo=1040, hi=1040, kv=2, dim=128, page=16, cache="bf16", keep=1024, recent=64),
        # a batch, each sequence up to 512 entries over
        dict(name="evict-batch", op="evict", seqs=64, lo=3900, hi=4608, kv=8, dim=128, page=32, cache="bf16", keep=4096, recent=256),
        # long prompts brought down to a sixteenth
        dict(name="evict-prompt", op="evict", seqs=3, lo=70001, hi=131072, kv=8, dim=128, page=64, cache="f16", keep=8192, recent=1024),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend", "evict"])
    dim = rng.choice([64, 128, 256])
    kv = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 12, 16])
    page = rng.choice([16, 32, 64, 128, 24])
    cache = rng.choice(["bf16", "f16"])
    io = rng.choice(["f32", cache])
    rot = rng.choice([dim, dim // 2, dim // 4])
    axes = rng.choice(["text", "blocks", "dealt", "2d", "3d"])
    if op == "rope":
        heads = rng.choice([1, 5, 12, 16, 32])
        return dict(op=op, tokens=_log(rng, 1, 16384 * 16 * 128 // (heads * dim)), heads=heads, dim=dim, rot=rot, axes=axes, io=io)
    if op == "append":
        seqs = _log(rng, 1, 128)
        heads = kv * group
        per = _log(rng, 1, max(1, 16384 * 16 * 64 // (heads * dim * seqs)))
        return dict(op=op, tokens=seqs * per, seqs=seqs, start=rng.randrange(0, 2048), heads=heads, kv=kv, dim=dim, rot=rot, axes=axes,
                    page=page, io=io, cache=cache)
    # entries of all sequences and heads together, times the head's width: bounded by the largest listed case
    most = 24 * 24000 * 2 * 256 // (kv * dim)
    if op == "attend":
        seqs = _log(rng, 1, 128)
        hi = _log(rng, 1, min(131072, most // seqs))
        return dict(op=op, seqs=seqs, lo=rng.randrange(0, hi + 1), hi=hi, heads=kv * group, kv=kv, dim=dim, page=page, io=io, cache=cache,
                    acc=rng.random() < 0.4)
    seqs = _log(rng, 1, 64)
    hi = _log(rng, 64, min(131072, most // (2 * seqs)))
    keep = rng.randrange(hi // 16 + 1, hi + 1)
    return dict(op=op, seqs=seqs, lo=rng.randrange(hi // 2, hi + 1), hi=hi, kv=kv, dim=dim, page=page, cache=cache, keep=keep,
                recent=rng.randrange(0, keep // 2 + 1))


def _lens(case):
    """Lengths spread over lo..hi, the longest first; they go by the case alone."""
    n, lo, hi = case["seqs"], case["lo"], case["hi"]
    r = np.random.RandomState(n * 7919 + lo * 31 + hi)
    l = np.sort(r.randint(lo, hi + 1, size=n))[::-1].copy()
    l[0] = hi
    return l


def _axes(case):
    """(sections, order of the pairs, own frequencies per axis, pairing, base) of a case's rotary form."""
    pairs = case["rot"] // 2
    third = pairs // 3
    return {
        "text": ([pairs], "blocked", False, "halves", 10000.0),
        "blocks": ([pairs - 2 * (third + 1), third + 1, third + 1], "blocked", False, "halves", 1e6),
        "dealt": ([pairs - 2 * third, third, third], "dealt", False, "halves", 1e7),
        "2d": ([pairs // 2, pairs - pairs // 2], "blocked", True, "adjacent", 100.0),
        "3d": ([pairs - 2 * third, third, third], "blocked", True, "adjacent", 10000.0),
    }[case["axes"]]


def _pair_tables(case):
    """Per pair its axis and its frequency (64 bits)."""
    section, order, per_axis, _, base = _axes(case)
    pairs, n = case["rot"] // 2, len(section)
    i = np.arange(pairs)
    if order == "dealt":
        axis = i % n
        axis = np.where(i // n < np.asarray(section)[axis], axis, 0)
    else:
        axis = np.repeat(np.arange(n), section)
    if per_axis:
        first = np.concatenate([[0], np.cumsum(section)[:-1]])
        freq = base ** (-(i - first[axis]) / np.asarray(section)[axis])
    else:
        freq = base ** (-i / pairs)
    return axis, freq


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _pages(g, case, lens):
    """A page table that deals the pages in no order, and the number of pages (some stay free)."""
    page, n = case["page"], len(lens)
    need = [-(-int(l) // page) for l in lens]
    total = sum(need) + 3
    free = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    row = torch.repeat_interleave(torch.arange(n), torch.tensor(need))
    col = torch.cat([torch.arange(k) for k in need]) if sum(need) else torch.empty(0, dtype=torch.int64)
    table = torch.full((n, max(max(need), 1)), -1, dtype=torch.int32, device="cuda")
    table[row.cuda(), col.cuda()] = free[:sum(need)]
    return table, total


def _cache(g, case, lens):
    table, n = _pages(g, case, lens)
    shape = (n, case["kv"], case["page"], case["dim"])
    dt = TYPES[case["cache"]]
    return dict(k=_normal(g, shape, dt), v=_normal(g, shape, dt), table=table)


def _positions(g, case, first):
    """Rotary positions [axes, tokens]: the token's number on every axis for text, else patch places behind it."""
    n, T = len(_axes(case)[0]), case["tokens"]
    if n == 1:
        return first[None].to(torch.int32)
    side = max(2, int(math.isqrt(T)))
    p = torch.randint(0, side, (n, T), generator=g, device="cuda")
    return (p + (first if case["op"] == "append" else 0)).to(torch.int32)


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    s = dict(case=case)
    if op in ("rope", "append"):
        T, d, dt = case["tokens"], case["dim"], TYPES[case["io"]]
        if op == "rope":
            s["x"] = _normal(g, (T, case["heads"], d), dt)
            s["pos"] = _positions(g, case, torch.arange(T, device="cuda"))
            return s
        per = T // case["seqs"]
        s.update(_cache(g, case, [case["start"] + per] * case["seqs"]))
        t = torch.arange(T, device="cuda")
        index = case["start"] + t % per
        s["seq"], s["index"] = (t // per).to(torch.int32), index.to(torch.int32)
        s["number"] = (index + 5000).to(torch.int32)  # the sequences have lost 5000 entries before
        # q, k and v are parts of one projection's rows
        qkv = _normal(g, (T, (case["heads"] + 2 * case["kv"]) * d), dt)
        a, b = case["heads"] * d, (case["heads"] + case["kv"]) * d
        s["q"], s["k_new"], s["v_new"] = qkv[:, :a].view(T, -1, d), qkv[:, a:b].view(T, -1, d), qkv[:, b:].view(T, -1, d)
        s["pos"] = _positions(g, case, index + 5000)
        s["weight"] = torch.rand(s["k"].shape[:3], generator=g, device="cuda")
        s["order"] = torch.randint(0, 5000, s["k"].shape[:3], generator=g, device="cuda", dtype=torch.int32)
        return s
    lens = _lens(case)
    s.update(_cache(g, case, lens))
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if op == "attend":
        # queries of norm 2 sqrt(dim): some keys take most of the weight
        s["q"] = _normal(g, (case["seqs"], case["heads"], case["dim"]), torch.float32).mul_(2).to(TYPES[case["io"]])
        if case["acc"]:
            s["weight"] = torch.rand(s["k"].shape[:3], generator=g, device="cuda")
        return s
    # heavy-tailed weights, some of them never attended to at all; order numbers that earlier evictions have mixed
    shape = s["k"].shape[:3]
    w = torch.randn(shape, generator=g, device="cuda").mul_(1.5).exp_()
    w[torch.rand(shape, generator=g, device="cuda") < 0.05] = 0
    n = case["hi"]
    i = torch.arange(n, device="cuda")
    mixed = (i + torch.rand((case["seqs"], case["kv"], n), generator=g, device="cuda") * 0.3 * n).argsort(-1).argsort(-1)
    order = torch.zeros(shape, dtype=torch.int32, device="cuda")
    live = (i < s["lens"][:, None])[:, None].expand_as(mixed)
    order.view(-1)[_flat(s["table"], n, case["kv"], case["page"])[live]] = mixed[live].to(torch.int32)
    # weight and order in one allocation, and what they hold before the eviction
    s["before"] = torch.stack([w.view(torch.int32), order])
    s["both"] = s["before"].clone()
    s["weight"], s["order"] = s["both"][0].view(torch.float32), s["both"][1]
    return s


def _flat(table, n, kv, page):
    """Flat place [sequences, kv heads, n] of each entry in a [pages, kv heads, page] buffer (of page 0 where there is none)."""
    i = torch.arange(n, device=table.device)
    p = table[:, i // page].long().clamp(min=0)
    h = torch.arange(kv, device=table.device)
    return (p[:, None] * kv + h[:, None]) * page + i % page


def _rotate(x, pos, case):
    axis, freq = _pair_tables(case)
    a = pos[torch.as_tensor(axis, device=x.device)].T.double() * torch.as_tensor(freq, device=x.device)
    c, s = a.cos().float()[:, None], a.sin().float()[:, None]
    rot = case["rot"]
    y, r = x.float(), None
    if _axes(case)[3] == "halves":
        u, v = y[..., :rot // 2], y[..., rot // 2:rot]
        r = torch.cat([u * c - v * s, v * c + u * s], -1)
    else:
        u, v = y[..., 0:rot:2], y[..., 1:rot:2]
        r = torch.stack([u * c - v * s, v * c + u * s], -1).flatten(-2)
    return torch.cat([r, y[..., rot:]], -1)


def _plain_append(s, case):
    page = case["page"]
    p = s["table"][s["seq"].long(), s["index"].long() // page].long()
    o = s["index"].long() % page
    s["k"][p, :, o] = _rotate(s["k_new"], s["pos"], case).to(s["k"].dtype)
    s["v"][p, :, o] = s["v_new"].float().to(s["v"].dtype)
    s["weight"][p, :, o] = 0.0
    s["order"][p, :, o] = s["number"][:, None]
    return dict(q=_rotate(s["q"], s["pos"], case).to(s["q"].dtype), k=s["k"], v=s["v"], weight=s["weight"], order=s["order"])


def _plain_attend(s, case):
    B, H, kv, d, n = case["seqs"], case["heads"], case["kv"], case["dim"], max(case["hi"], 1)
    flat = _flat(s["table"], n, kv, case["page"])
    live = (torch.arange(n, device=flat.device) < s["lens"][:, None])[:, None]
    k = s["k"].view(-1, d)[flat].float()
    z = torch.matmul(s["q"].float().view(B, kv, H // kv, d), k.transpose(-1, -2)) / math.sqrt(d)
    del k
    z = torch.where(live[:, :, None], z, -torch.inf)
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(m > -torch.inf, m, 0.0))
    t = e.sum(-1, keepdim=True)
    p = e / torch.where(t > 0, t, 1.0)
    v = torch.where(live[..., None], s["v"].view(-1, d)[flat].float(), 0.0)
    out = dict(out=torch.matmul(p, v).view(B, H, d).to(s["q"].dtype))
    if case["acc"]:
        add, live = p.sum(2), live.expand(B, kv, n)
        s["weight"].view(-1)[flat[live]] += add[live]
        out["weight"] = s["weight"]
    return out


def _plain_evict(s, case):
    kv, d, keep, n = case["kv"], case["dim"], case["keep"], case["hi"]
    flat = _flat(s["table"], n, kv, case["page"])
    i = torch.arange(n, device=flat.device)
    lens = s["lens"].long()[:, None, None]
    live = (i < lens).expand_as(flat)
    w, o = s["weight"].view(-1)[flat], s["order"].view(-1)[flat].long()
    newest = torch.where(live, o, torch.iinfo(torch.int64).min).amax(-1, keepdim=True)
    key = torch.where(o > newest - case["recent"], torch.inf, torch.where(w.isnan(), -torch.inf, w))
    best = torch.where(live, key, -torch.inf).argsort(dim=-1, descending=True, stable=True)
    stays = torch.zeros_like(live).scatter(-1, best[..., :keep], True) & live
    front = i < lens.clamp(max=keep)
    hole, spare = front & ~stays, stays & ~front
    spares = (~spare).to(torch.int8).argsort(dim=-1, stable=True)
    source = torch.where(hole, spares.gather(-1, (hole.long().cumsum(-1) - 1).clamp(min=0)), i)
    to, of = flat[hole], flat.gather(-1, source)[hole]
    for buffer in (s["k"].view(-1, d), s["v"].view(-1, d), s["weight"].view(-1), s["order"].view(-1)):
        buffer[to] = buffer[of]
    kept = torch.full((case["seqs"], kv, keep), -1, dtype=torch.int32, device=flat.device)
    kept[..., :n] = torch.where(front, source, -1)[..., :keep].to(torch.int32)
    return dict(kept=kept, lens=lens.flatten().clamp(max=keep).to(torch.int32), k=s["k"], v=s["v"], weight=s["weight"], order=s["order"])


def _ofb():
    """The package's binding (its folder's name is no module name)."""
    if "ornith_flight_b200.ofb" not in sys.modules:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ornith-flight_b200", "ofb.py")
        spec = importlib.util.spec_from_file_location("ornith_flight_b200.ofb", path)
        sys.modules[spec.name] = mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
    return sys.modules["ornith_flight_b200.ofb"]


def _kept_by_user(s, case):
    """What a program makes once and keeps: the rotary form, the cache's handle, the calls' scratch."""
    ofb, u = _ofb(), {}
    if "axes" in case:
        section, order, per_axis, pairing, base = _axes(case)
        u["rope"] = ofb.RopeConfig(rot_dim=case["rot"], section=section, base=base, per_axis=per_axis,
                                   pairing=ofb.ROPE_HALVES if pairing == "halves" else ofb.ROPE_ADJACENT,
                                   order=ofb.ROPE_BLOCKED if order == "blocked" else ofb.ROPE_DEALT)
    if "k" in s:
        u["cache"] = ofb.KvCache(s["k"], s["v"], s["table"], weight=s.get("weight"), order=s.get("order"))
    if case["op"] == "attend":
        u["scratch"] = ofb.attn_scratch(u["cache"], case["heads"], case["seqs"], case["hi"], accumulate=case["acc"])
    if case["op"] == "evict":
        u["scratch"] = ofb.evict_scratch(u["cache"], case["seqs"], case["keep"])
    return u


def _own(s, case):
    if "user" not in s:
        s["user"] = _kept_by_user(s, case)
    ofb, u, op = _ofb(), s["user"], case["op"]
    if op == "rope":
        return dict(x=ofb.rope(s["x"], s["pos"], u["rope"]))
    if op == "append":
        q = ofb.rope_append(u["cache"], s["k_new"], s["v_new"], s["seq"], s["index"], number=s["number"], q=s["q"], pos=s["pos"], rope=u["rope"])
        return dict(q=q, k=s["k"], v=s["v"], weight=s["weight"], order=s["order"])
    if op == "attend":
        out = dict(out=ofb.attn_decode(u["cache"], s["q"], s["lens"], max_len=case["hi"], accumulate=case["acc"], scratch=u["scratch"]))
        if case["acc"]:
            out["weight"] = s["weight"]
        return out
    kept, lens = ofb.kv_evict(u["cache"], s["lens"], keep=case["keep"], recent=case["recent"], max_len=case["hi"], scratch=u["scratch"])
    return dict(kept=kept, lens=lens, k=s["k"], v=s["v"], weight=s["weight"], order=s["order"])


def run(state):
    case = state["case"]
    if case["op"] == "evict":
        # weights go on growing between two evictions: each pass finds those of before. The entries behind the
        # kept ones are left as they were, so a second pass makes the same moves.
        state["both"].copy_(state["before"])
    if own:
        return _own(state, case)
    if case["op"] == "rope":
        return dict(x=_rotate(state["x"], state["pos"], case).to(state["x"].dtype))
    return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[case["op"]](state, case)


def work(case):
    op, d = case["op"], case["dim"]
    if op == "rope":
        n = case["tokens"] * case["heads"] * d
        return dict(bytes=2 * n * SIZE[case["io"]] + 4 * case["tokens"] * len(_axes(case)[0]), flops=3 * n)
    kv = case["kv"]
    if op == "append":
        T, H, e = case["tokens"], case["heads"], SIZE[case["io"]]
        return dict(bytes=T * ((2 * H + 2 * kv) * d * e + 2 * kv * d * 2 + 8 * kv + 4 * (3 + len(_axes(case)[0]))), flops=3 * T * (H + kv) * case["rot"])
    lens = _lens(case).astype(np.float64)
    n = float(lens.sum())
    if op == "attend":
        H, B = case["heads"], case["seqs"]
        return dict(bytes=n * kv * (4 * d + (8 if case["acc"] else 0)) + 2 * B * H * d * SIZE[case["io"]], flops=4 * n * H * d)
    # of the kept entries that are not protected, those behind the first `keep` are moved: their expected number
    keep, recent = case["keep"], case["recent"]
    over = np.maximum(lens - keep, 0)
    moved = float(np.where(over > 0, np.minimum(recent, over) + (keep - recent) * np.maximum(over - recent, 0) / np.maximum(lens - recent, 1), 0).sum())
    return dict(bytes=kv * (8 * n + moved * (8 * d + 16) + 4 * keep * case["seqs"]), flops=n * kv)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]

    def turned(x, pos):
        axis, freq = _pair_tables(case)
        angle = pos.double()[torch.as_tensor(axis, device="cuda")] * torch.as_tensor(freq, device="cuda")[:, None]
        turn = torch.polar(torch.ones_like(angle), angle).T[:, None]
        y, rot = x.double().clone(), case["rot"]
        if _axes(case)[3] == "halves":
            z = torch.complex(y[..., :rot // 2], y[..., rot // 2:rot]) * turn
            y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
        else:
            z = torch.view_as_complex(y[..., :rot].unflatten(-1, (-1, 2)).contiguous()) * turn
            y[..., :rot] = torch.view_as_real(z).flatten(-2)
        return y

    if op == "rope":
        return dict(x=turned(s["x"], s["pos"]))
    page, kv, d = case["page"], case["kv"], case["dim"]
    if op == "append":
        index = s["index"].cpu().numpy()
        pages = s["table"].cpu().numpy()[s["seq"].cpu().numpy(), index // page]
        at = torch.as_tensor(pages.astype(np.int64) * page + index % page, device="cuda")
        out = {}
        for name, new in (("k", turned(s["k_new"], s["pos"])), ("v", s["v_new"].double())):
            rows = s[name].double().transpose(1, 2).reshape(-1, kv, d)
            rows[at] = new
            out[name] = rows.view(-1, page, kv, d).transpose(1, 2)
        w = s["weight"].double().transpose(1, 2).reshape(-1, kv)
        w[at] = 0
        return dict(q=turned(s["q"], s["pos"]), weight=w.view(-1, page, kv).transpose(1, 2), order=None, **out)
    lens = s["lens"].tolist()
    if op == "attend":
        G = case["heads"] // kv
        out = torch.zeros(case["seqs"], case["heads"], d, dtype=torch.float64, device="cuda")
        weight = s["weight"].double() if case["acc"] else None
        for b, n in enumerate(lens):
            if not n:
                continue
            pages = s["table"][b, :-(-n // page)].long()
            for h in range(kv):
                k, v = (s[x][pages, h].reshape(-1, d)[:n].double() for x in "kv")
                p = torch.softmax(s["q"][b, h * G:(h + 1) * G].double() @ k.T * d ** -0.5, -1)
                out[b, h * G:(h + 1) * G] = p @ v
                if case["acc"]:
                    w = weight[pages, h].reshape(-1)
                    w[:n] += p.sum(0)
                    weight[pages, h] = w.view(-1, page)
        return dict(out=out, weight=weight) if case["acc"] else dict(out=out)
    weight, order, table = s["weight"].cpu().numpy().astype(np.float64), s["order"].cpu().numpy(), s["table"].cpu().numpy()
    keep = case["keep"]
    to, of = [], []
    kept = np.full((case["seqs"], kv, keep), -1, dtype=np.int32)
    for b, n in enumerate(lens):
        e = np.arange(n)
        for h in range(kv):
            at = (table[b, e // page].astype(np.int64) * kv + h) * page + e % page
            kept[b, h, :min(n, keep)] = e[:keep]
            if n <= keep:
                continue
            w, o = weight.reshape(-1)[at], order.reshape(-1)[at]
            young = o > o.max() - case["recent"]
            best = np.lexsort((e, -w, ~young))[:keep]  # the youngest first (fewer than `keep`), then by weight, then by place
            chosen = np.zeros(n, bool)
            chosen[best] = True
            holes, spares = e[:keep][~chosen[:keep]], e[keep:][chosen[keep:]]
            kept[b, h, holes] = spares
            to.append(at[holes])
            of.append(at[spares])
    out = dict(kept=torch.as_tensor(kept), lens=None, order=None)
    to, of = (torch.as_tensor(np.concatenate(x) if x else np.zeros(0, np.int64), device="cuda") for x in (to, of))
    for name in ("k", "v", "weight"):
        rows = s[name].reshape(-1, d if name != "weight" else 1).double()
        rows[to] = rows[of]
        out[name] = rows.view(s[name].shape)
    return out

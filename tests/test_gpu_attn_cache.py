"""Rotary positions, the paged cache, attention of one new token and eviction
(ofb_rope, ofb_rope_append, ofb_attn_decode, ofb_kv_evict) against plain 64-bit
restatements. The caches hold NaN in every place without an entry and page
numbers out of range behind each sequence's last page."""
import numpy as np
import pytest
import torch

from attn_cache_ref import DT, HALF_STEP, Cache, attend, attend_tol, evict, f64, rope, rope_close

pytestmark = pytest.mark.gpu
HALVES, ADJACENT, BLOCKED, DEALT = 0, 1, 0, 1


# ---- rotary positions ---------------------------------------------------------

ROPES = [  # heads, head_dim, rot, section, pairing, order, per_axis
    (16, 128, 128, [64], HALVES, BLOCKED, False),
    (5, 128, 128, [24, 20, 20], HALVES, BLOCKED, False),
    (3, 256, 64, [12, 10, 10], HALVES, DEALT, False),
    (2, 64, 64, [16, 16], ADJACENT, BLOCKED, True),
    (1, 64, 32, [6, 0, 4, 6], ADJACENT, BLOCKED, True),
    (7, 80, 20, [4, 3, 3], HALVES, DEALT, False),     # rot_dim no multiple of 16
    (3, 37, 6, [2, 1], ADJACENT, BLOCKED, False),     # odd head_dim
    (1, 1024, 256, [0, 128], HALVES, BLOCKED, True),
    (2, 2, 2, [1], HALVES, BLOCKED, False),
]


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T", [1, 3, 1030])
@pytest.mark.parametrize("H,d,rot,section,pairing,order,per_axis", ROPES)
def test_rope(ofb, cuda, H, d, rot, section, pairing, order, per_axis, T, io):
    g = torch.Generator().manual_seed(T * d + H)
    x = torch.randn(T, H, d, generator=g).to(DT[io])
    pos = torch.randint(-50, 5000, (len(section), T), generator=g, dtype=torch.int32)
    pos[:, -1] = 1 << 30  # far off: 2^30 times a frequency of 1
    cfg = ofb.RopeConfig(rot, section, base=10000.0, pairing=pairing, order=order, per_axis=per_axis)
    got = ofb.rope(x.to(cuda), pos.to(cuda), cfg)
    want, size = rope(f64(x), pos.numpy(), rot, section, 10000.0, pairing, order, per_axis)
    rope_close(got, want, size, io)
    assert torch.equal(got.cpu()[..., rot:], x[..., rot:])


@pytest.mark.parametrize("io,off,gap", [("f32", 0, 0), ("bf16", 1, 3), ("f16", 8, 16), ("f32", 2, 8)])
def test_rope_in_place_in_a_wider_row(ofb, cuda, io, off, gap):
    # rows inside a larger buffer at any element offset: the rest of it stays
    T, H, d = 9, 4, 64
    buf = torch.randn(T, off + H * d + gap).to(DT[io]).to(cuda)
    before = buf.clone()
    x = buf[:, off:off + H * d].view(T, H, d) if off == 0 and gap == 0 else buf[:, off:off + H * d].unflatten(1, (H, d))
    pos = torch.arange(T, dtype=torch.int32, device=cuda)[None]
    assert ofb.rope(x, pos, ofb.RopeConfig(64), out=x) is x
    want, size = rope(f64(before[:, off:off + H * d].unflatten(1, (H, d))), pos.cpu().numpy(), 64, [32])
    rope_close(x, want, size, io)
    assert torch.equal(buf[:, :off], before[:, :off]) and torch.equal(buf[:, off + H * d:], before[:, off + H * d:])


# ---- append -------------------------------------------------------------------

@pytest.mark.parametrize("io", ["f32", "own"])
@pytest.mark.parametrize("cache,kv,G,d,page,rot,T", [("bf16", 2, 8, 128, 16, 128, 1), ("f16", 1, 1, 64, 7, 32, 5), ("bf16", 8, 4, 256, 64, 64, 33),
                                                     ("f16", 3, 2, 96, 24, 90, 700), ("bf16", 2, 1, 192, 1, 0, 12)])
def test_append(ofb, cuda, cache, kv, G, d, page, rot, T, io):
    io = cache if io == "own" else io
    B, H, reach = 3, kv * G, (T + 2) // 3 + 20
    c = Cache(ofb, [0, 0, 0], kv, d, page, cache, seed=T, spread=8 * (T % 2), reach=reach, meta=True)
    g = torch.Generator().manual_seed(T)
    seq = torch.arange(T, dtype=torch.int32) % B
    index = (torch.arange(T, dtype=torch.int32) // B) + 7
    number = index + 100
    if T > 4:
        seq[2], seq[4] = -1, -5  # padding
    qkv = torch.randn(T, (H + 2 * kv) * d, generator=g).to(DT[io]).to(cuda)
    q, k, v = qkv[:, :H * d].unflatten(1, (H, d)), qkv[:, H * d:(H + kv) * d].unflatten(1, (kv, d)), qkv[:, (H + kv) * d:].unflatten(1, (kv, d))
    pos = torch.randint(0, 3000, (2, T), generator=g, dtype=torch.int32)
    section = [rot // 2 - 5, 5]
    cfg = ofb.RopeConfig(rot, section, base=1e4) if rot else None
    old = [t.clone() for t in (c.k, c.v, c.weight, c.order)]
    got = ofb.rope_append(c.handle, k, v, seq.to(cuda), index.to(cuda), number=number.to(cuda), q=q,
                          pos=pos.to(cuda) if rot else None, rope=cfg)
    turn = lambda x: rope(f64(x), pos.numpy(), rot, section) if rot else (f64(x), np.zeros(x.shape))  # noqa: E731
    rope_close(got, *turn(q), io)
    want_k, size_k = turn(k)
    new = torch.zeros(c.k.shape[:3], dtype=torch.bool, device=cuda)
    rows = [t for t in range(T) if seq[t] >= 0]
    pages = c.table.cpu()[seq[rows].long(), index[rows].long() // page].long().to(cuda)
    slots = (index[rows].long() % page).to(cuda)
    new[pages, :, slots] = True
    rope_close(c.k[pages, :, slots], want_k[rows], size_k[rows], cache)
    assert torch.equal(c.v[pages, :, slots], v[rows].to(DT[cache]))
    assert (c.weight[pages, :, slots] == 0).all() and torch.equal(c.order[pages, :, slots], number[rows].to(cuda)[:, None].expand(-1, kv))
    for t, o in zip((c.k, c.v, c.weight, c.order), old):  # all else is left as it was
        it = {2: torch.int16, 4: torch.int32}[t.element_size()]
        assert torch.equal(t.contiguous().view(it)[~new], o.contiguous().view(it)[~new])
    assert c.handle.device_errors() == 0


def test_append_alone_and_bad_places(ofb, cuda):
    # no queries, no rotation, order by index; rows outside the table are dropped and reported
    c = Cache(ofb, [0, 0], 2, 64, 16, reach=40, meta=True)
    before = c.k.clone()
    k, v = torch.randn(2, 6, 2, 64, device=cuda, dtype=torch.bfloat16)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    assert ofb.rope_append(c.handle, k, v, i32(0, 1, 2, 0, 0, 1), i32(3, 39, 0, -1, 48, 2 ** 31 - 1)) is None
    assert c.handle.device_errors() == ofb.CACHE_EINDEX and c.handle.device_errors() == 0
    for t, (b, i) in enumerate(((0, 3), (1, 39))):
        p, s = int(c.table[b, i // 16]), i % 16
        assert torch.equal(c.k[p, :, s], k[t]) and torch.equal(c.v[p, :, s], v[t]) and (c.order[p, :, s] == i).all()
        before[p, :, s] = k[t]
    assert torch.equal(before.view(torch.int16), c.k.view(torch.int16))
    c.table[0, 0] = c.n_pages
    ofb.rope_append(c.handle, k[:1], v[:1], i32(0), i32(3))
    assert c.handle.device_errors() == ofb.CACHE_EPAGE
    assert torch.equal(before.view(torch.int16), c.k.view(torch.int16))


# ---- attention ----------------------------------------------------------------

def check_attention(c, q, got, io, scale, weight_before=None, lens=None):
    for b, n in enumerate(c.lens if lens is None else lens):
        k, v = f64(c.rows("k", b, n)), f64(c.rows("v", b, n))
        want, p, size = attend(f64(q[b]), k, v, scale)
        tol = attend_tol(size, c.d)[:, None]
        # bf16 output: a probability's two bf16 parts leave 2^-17 of it
        top = np.abs(v).max() if n else 0.0
        bound = (tol + (2.0 ** -17 if io == "bf16" else 0)) * top + HALF_STEP[io] * np.abs(want) + 2.0 ** -25 * (io == "f16")
        err = np.abs(f64(got[b]) - want)
        assert (err <= bound).all(), f"sequence {b} of {n}: off by {err.max()}, bound {bound.max()}"
        if weight_before is not None and n:
            at = c.at(b, n)
            old = f64(weight_before)[at[0].numpy(), :, at[1].numpy()]
            w = f64(c.rows("weight", b, n))
            slack = tol.reshape(c.kv, -1).max(1) * p + 2.0 ** -23 * (np.abs(old) + p)
            assert (np.abs(w - old - p) <= slack).all(), f"weights of sequence {b}: off by {np.abs(w - old - p).max()}"


ATTEND = [  # cache, kv, G, d, page, lens
    ("bf16", 2, 8, 128, 16, [517]),
    ("bf16", 1, 1, 64, 16, [0, 1, 15, 16, 17, 64, 65]),
    ("f16", 2, 4, 256, 64, [1000, 0, 3, 4097]),
    ("f16", 1, 7, 96, 24, [129, 31]),
    ("bf16", 3, 3, 192, 7, [77, 1, 2000]),
    ("bf16", 1, 16, 128, 32, [333, 5000]),   # two passes per kv head
    ("f16", 2, 12, 64, 128, [0, 0, 9000]),
    ("bf16", 4, 20, 256, 16, [40, 1]),
    ("f16", 8, 8, 128, 1, [50] * 20),
    ("bf16", 1, 2, 128, 1000, [100, 20000]),
    ("f16", 1, 130, 64, 16, [70]),           # one kv head for 130 query heads
    ("bf16", 2, 1, 64, 16, [0, 0]),
]


@pytest.mark.parametrize("io", ["f32", "own"])
@pytest.mark.parametrize("acc", [False, True])
@pytest.mark.parametrize("cache,kv,G,d,page,lens", ATTEND, ids=lambda x: "x".join(map(str, x[:3])) if isinstance(x, list) else str(x))
def test_attention(ofb, cuda, cache, kv, G, d, page, lens, acc, io):
    io = cache if io == "own" else io
    c = Cache(ofb, lens, kv, d, page, cache, seed=d + G, spread=16 if acc else 0, meta=acc)
    q = (torch.randn(len(lens), kv * G, d, generator=torch.Generator().manual_seed(5)) * 2).to(DT[io]).to(cuda)
    before = c.weight.clone()
    got = ofb.attn_decode(c.handle, q, c.dlens, accumulate=acc)
    check_attention(c, q, got, io, d ** -0.5, before if acc else None)
    same = c.weight.clone() if acc else None
    if acc:  # places without an entry are left as they were
        live = torch.zeros_like(before, dtype=torch.bool)
        for b, n in enumerate(lens):
            p, s = c.at(b, n)
            live[p.to(cuda), :, s.to(cuda)] = True
        assert torch.equal(c.weight.view(torch.int32)[~live], before.view(torch.int32)[~live])
        c.weight.copy_(before)
    again = ofb.attn_decode(c.handle, q, c.dlens, accumulate=acc)
    assert torch.equal(got, again)  # reproducible
    if acc:
        assert torch.equal(same.view(torch.int32)[live], c.weight.view(torch.int32)[live])
    # a tight bound on the lengths
    check_attention(c, q, ofb.attn_decode(c.handle, q, c.dlens, max_len=max(max(lens), 1)), io, d ** -0.5)
    assert c.handle.device_errors() == 0


@pytest.mark.parametrize("io", ["f32", "own"])
@pytest.mark.parametrize("d,G,page,cache", [(64, 3, 16, "bf16"), (96, 12, 20, "f16"), (128, 20, 64, "bf16"), (192, 9, 5, "f16"), (256, 4, 32, "bf16")])
def test_attention_joins_many_parts(ofb, cuda, d, G, page, cache, io):
    # one long sequence among short ones: its parts lie in most of the runs
    lens = [7, 30011, 0, 2600]
    io = cache if io == "own" else io
    c = Cache(ofb, lens, 1, d, page, cache, seed=G, meta=True)
    q = (torch.randn(len(lens), G, d, generator=torch.Generator().manual_seed(d)) * 2).to(DT[io]).to(cuda)
    before = c.weight.clone()
    check_attention(c, q, ofb.attn_decode(c.handle, q, c.dlens, accumulate=True), io, d ** -0.5, before)
    one = Cache(ofb, lens[1:2], 2, d, page, cache, seed=G + 1)
    q = q[:1].repeat(1, 2, 1)
    check_attention(one, q, ofb.attn_decode(one.handle, q, one.dlens), io, d ** -0.5)


@pytest.mark.parametrize("kv,G,d,lens", [(1, 16, 256, [300]), (2, 20, 128, [100, 0, 31, 1]), (3, 16, 256, [9, 13] * 40),
                                         (1, 40, 64, [700]), (2, 24, 192, [60] * 90)])
def test_attention_weights_of_short_sequences_in_passes(ofb, cuda, kv, G, d, lens):
    # more query heads per kv head than a pass has: clusters of one and more CTAs, CTAs of one warp
    c = Cache(ofb, lens, kv, d, 16, "bf16", seed=G, meta=True)
    q = torch.randn(len(lens), kv * G, d, generator=torch.Generator().manual_seed(d)).to(cuda)
    before = c.weight.clone()
    check_attention(c, q, ofb.attn_decode(c.handle, q, c.dlens, accumulate=True), "f32", d ** -0.5, before)


def test_attention_many_sequences(ofb, cuda):
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 90, size=1100).tolist()
    c = Cache(ofb, lens, 1, 64, 16, "f16", seed=8)
    q = torch.randn(1100, 2, 64, device=cuda)
    check_attention(c, q, ofb.attn_decode(c.handle, q, c.dlens), "f32", 0.125)


def test_attention_strided_queries_scale_and_out(ofb, cuda):
    c = Cache(ofb, [100, 260], 2, 128, 16)
    wide = torch.randn(2, 3 * 1024 + 5, device=cuda)
    q = wide[:, 3:3 + 1024].unflatten(1, (8, 128))
    out = torch.full((2, 1500), 7.0, device=cuda)
    o = out[:, 1:1 + 1024].unflatten(1, (8, 128))
    assert ofb.attn_decode(c.handle, q, c.dlens, scale=-0.02, out=o) is o
    check_attention(c, q, o, "f32", -0.02)
    assert (out[:, :1] == 7).all() and (out[:, 1025:] == 7).all()


@pytest.mark.parametrize("size", [2.0 ** -40, 1e-3, 300.0])
@pytest.mark.parametrize("cache", ["bf16", "f16"])
def test_attention_query_sizes(ofb, cuda, cache, size):
    # f32 queries far outside what fp16 holds keep their precision
    c = Cache(ofb, [200], 1, 128, 16, cache)
    q = torch.randn(1, 8, 128, device=cuda) * size
    q[0, 0] = 0
    q[0, 1, 5] = 70000 * size
    scale = 0.05 / size
    check_attention(c, q, ofb.attn_decode(c.handle, q, c.dlens, scale=scale), "f32", scale)


def test_attention_sharp_and_low_scores(ofb, cuda):
    # one entry takes all the weight; scores at +-1e30 neither overflow nor turn into NaN
    c = Cache(ofb, [300], 1, 64, 16)
    p, s = c.at(0, 300)
    c.k.zero_()
    c.k[p[123].item(), 0, s[123].item(), 0] = 1e30
    c.k[p[7].item(), 0, s[7].item(), 0] = -1e30
    q = torch.zeros(1, 2, 64, device=cuda)
    q[0, 0, 0], q[0, 1, 0] = 8.0, -8.0
    got = ofb.attn_decode(c.handle, q, c.dlens, scale=0.125)
    v = c.rows("v", 0, 300).float()
    assert torch.equal(got[0, 0], v[123, 0]) and torch.equal(got[0, 1], v[7, 0])


def test_attention_bad_pages_and_lengths(ofb, cuda):
    c = Cache(ofb, [100, 64], 2, 64, 16, meta=True)
    q = torch.randn(2, 4, 64, device=cuda)
    full = ofb.attn_decode(c.handle, q, c.dlens)
    # a length above max_len is cut down to it
    cut = ofb.attn_decode(c.handle, q, c.dlens, max_len=80)
    assert c.handle.device_errors() == ofb.CACHE_ELEN
    check_attention(c, q, cut, "f32", 0.125, lens=[80, 64])
    # a length below 0 counts as 0
    assert (ofb.attn_decode(c.handle, q, torch.full_like(c.dlens, -3)) == 0).all()
    # entries of a page that is none are masked; a sequence of such pages only gives zeros
    table = c.table.clone()
    c.table[0, 1], c.table[1, :4] = -1, c.n_pages
    got = ofb.attn_decode(c.handle, q, c.dlens, accumulate=True)
    assert c.handle.device_errors() == ofb.CACHE_EPAGE
    assert (got[1] == 0).all()
    rest = np.r_[0:16, 32:100]
    c.table.copy_(table)
    k, v = f64(c.rows("k", 0, 100))[rest], f64(c.rows("v", 0, 100))[rest]
    want, _, size = attend(f64(q[0]), k, v, 0.125)
    assert (np.abs(f64(got[0]) - want) <= attend_tol(size, 64)[:, None] * np.abs(v).max() + 2.0 ** -24 * np.abs(want)).all()
    assert torch.equal(full, ofb.attn_decode(c.handle, q, c.dlens))


def test_attention_and_append_far_into_a_large_cache(ofb, cuda):
    # pages so far apart that elements and bytes pass 32 bits
    gap = 1_300_000_000 // 8 * 8
    store = [torch.empty(3 * gap + 2 * 16 * 64, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    k, v = (torch.as_strided(s, (4, 2, 16, 64), (gap, 16 * 64, 64, 1)) for s in store)
    k.normal_(), v.normal_()
    table = torch.tensor([[3, 0, 2]], dtype=torch.int32, device=cuda)
    weight, order = torch.zeros(4, 2, 16, device=cuda), torch.zeros(4, 2, 16, dtype=torch.int32, device=cuda)
    cache = ofb.KvCache(k, v, table, weight=weight, order=order)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    nk, nv = torch.randn(2, 2, 2, 64, device=cuda)
    ofb.rope_append(cache, nk, nv, i32(0, 0), i32(2, 40))
    assert torch.equal(k[3, :, 2], nk[0].bfloat16()) and torch.equal(v[2, :, 8], nv[1].bfloat16())
    q = torch.randn(1, 4, 64, device=cuda)
    got = ofb.attn_decode(cache, q, i32(45), accumulate=True)
    rows = lambda t: f64(torch.cat([t[3].transpose(0, 1), t[0].transpose(0, 1), t[2].transpose(0, 1)])[:45])  # noqa: E731
    want, p, size = attend(f64(q[0]), rows(k), rows(v), 0.125)
    assert (np.abs(f64(got[0]) - want) <= attend_tol(size, 64)[:, None] * np.abs(rows(v)).max() + 2.0 ** -24 * np.abs(want)).all()
    order.copy_(torch.arange(4 * 2 * 16, dtype=torch.int32, device=cuda).view(4, 2, 16))
    w = rows(weight[..., None])[..., 0]
    o = rows(order[..., None])[..., 0]
    before = rows(k)
    kept, new = ofb.kv_evict(cache, i32(45), keep=10, recent=0)
    for h in range(2):
        src = evict(w[:, h], o[:, h], 10, 0)
        assert kept[0, h].tolist() == src.tolist()
        assert np.array_equal(rows(k)[:10, h], before[src, h])
    assert new.tolist() == [10]


# ---- eviction -----------------------------------------------------------------

def check_eviction(ofb, c, keep, recent, max_len=0):
    names = ("k", "v", "weight", "order")
    bits = lambda t: t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)  # noqa: E731
    want = {x: bits(getattr(c, x)).clone() for x in names}
    lens = [min(n, max_len) if max_len else n for n in c.lens]
    src_all = np.full((len(lens), c.kv, keep), -1)
    for b, n in enumerate(lens):
        w, o = c.rows("weight", b, n).cpu().numpy(), c.rows("order", b, n).cpu().numpy()
        p, s = (x.to(c.k.device) for x in c.at(b, n))
        for h in range(c.kv):
            src = evict(w[:, h], o[:, h], keep, recent)
            src_all[b, h, :len(src)] = src
            f = torch.as_tensor(src, device=c.k.device)
            for x in names:
                want[x][p[:len(src)], h, s[:len(src)]] = bits(getattr(c, x))[p[f], h, s[f]]
    kept, new = ofb.kv_evict(c.handle, c.dlens, keep=keep, recent=recent, max_len=max_len)
    assert np.array_equal(kept.cpu().numpy(), src_all)
    assert new.tolist() == [min(n, keep) for n in lens]
    for x in names:
        assert torch.equal(bits(getattr(c, x)), want[x]), x


EVICT = [  # cache, kv, d, page, lens, keep, recent
    ("bf16", 2, 128, 16, [1040], 1024, 64),
    ("f16", 1, 64, 7, [0, 1, 2, 31, 32, 33, 100], 32, 5),
    ("bf16", 3, 256, 64, [5000, 17, 4999], 333, 333),
    ("f16", 2, 96, 24, [3000, 64], 1, 0),
    ("bf16", 1, 192, 1, [65, 70], 64, 1),
    ("f16", 4, 128, 128, [2048] * 9, 2047, 100),
    ("bf16", 1, 64, 32, [40001], 20011, 4000),
    ("f16", 2, 64, 1000, [12000, 900], 11999, 0),
]


@pytest.mark.parametrize("cache,kv,d,page,lens,keep,recent", EVICT, ids=lambda x: "x".join(map(str, x[:3])) if isinstance(x, list) else str(x))
def test_eviction(ofb, cuda, cache, kv, d, page, lens, keep, recent):
    c = Cache(ofb, lens, kv, d, page, cache, seed=keep, spread=8 if kv == 2 else 0, meta=True)
    check_eviction(ofb, c, keep, recent)
    assert c.handle.device_errors() == 0


@pytest.mark.parametrize("seqs,more", [(1, 47), (2, 48), (2, 49), (33, 48), (33, 49), (33, 128), (33, 129), (40, 600)])
def test_eviction_copies_in_either_launch(ofb, cuda, seqs, more):
    # few and many rows, with moves up to and past where a second launch makes them
    lens = [700 + more - i % 5 for i in range(seqs)]
    check_eviction(ofb, Cache(ofb, lens, 2, 64, 16, "f16", seed=more, reach=700 + more, meta=True), 700, 30, max_len=700 + more)


def test_eviction_ties_nan_and_zeros(ofb, cuda):
    # equal weights go to the lower place, across the CTAs of a cluster; NaN is lightest, -0 is 0
    c = Cache(ofb, [9000, 9000, 300], 2, 64, 16, meta=True)
    vals = torch.tensor([0.0, -0.0, 1.0, 1.0, float("nan"), float("inf"), 1e-42, -2.0], device=cuda)
    i = torch.randint(0, 8, c.weight.shape, device=cuda, generator=torch.Generator(cuda).manual_seed(1))
    c.weight.copy_(vals[i])
    c.weight[c.table[1, :563].long()] = 0.25  # a sequence of nothing but equals
    check_eviction(ofb, c, 200, 16)


def test_eviction_weights_far_apart_and_orders_at_the_ends(ofb, cuda):
    c = Cache(ofb, [4000], 1, 64, 16, meta=True)
    c.weight.copy_(torch.randn(c.weight.shape, device=cuda).mul(30).exp())
    p, s = c.at(0, 4000)
    o = c.order[p, :, s]
    o[o == 0], o[o == 3999] = -2 ** 31, 2 ** 31 - 1
    c.order[p, :, s] = o
    check_eviction(ofb, c, 1000, 500)


def test_eviction_long_sequence(ofb, cuda):
    # more keys than a CTA holds: the cluster grows
    n = 200000
    c = Cache(ofb, [n], 1, 64, 64, meta=True)
    check_eviction(ofb, c, 1500, 100)


def test_eviction_bad_page_and_cut_length(ofb, cuda):
    c = Cache(ofb, [200], 1, 64, 16, meta=True)
    check_eviction(ofb, c, 50, 10, max_len=150)
    assert c.handle.device_errors() == ofb.CACHE_ELEN
    c.table[0, 12] = -1  # entries 192..199: dropped, the youngest among them
    kept, new = ofb.kv_evict(c.handle, c.dlens, keep=150, recent=0)
    assert c.handle.device_errors() == ofb.CACHE_EPAGE and new.tolist() == [150]
    assert kept.max() < 192


# ---- together, on streams and in graphs ------------------------------------------

def test_decode_steps_with_eviction(ofb, cuda):
    """Sequences grow token by token under a budget: rotate and append, attend
    with weights, evict when over; against lists of entries kept by hand."""
    B, kv, G, d, page, keep, budget = 3, 2, 4, 64, 8, 24, 32
    H, reach = kv * G, 40
    c = Cache(ofb, [0] * B, kv, d, page, "bf16", reach=reach, meta=True)
    cfg = ofb.RopeConfig(32, [6, 5, 5], base=1e4, order=DEALT)
    g = torch.Generator().manual_seed(0)
    entries = [[[] for _ in range(kv)] for _ in range(B)]  # per head: [k row, v row, weight, order]
    lens = torch.tensor([0, 0, 0], dtype=torch.int32, device=cuda)
    for step in range(90):
        qkv = torch.randn(B, (H + 2 * kv) * d, generator=g)
        pos = torch.tensor([[step] * B, [step // 2] * B, [step // 3] * B], dtype=torch.int32)
        x = qkv.to(cuda)
        q, k, v = (t.unflatten(1, (-1, d)) for t in x.split([H * d, kv * d, kv * d], 1))
        seq = torch.arange(B, dtype=torch.int32)
        if step % 7 == 3:
            seq[1] = -1  # this sequence waits
        qr = ofb.rope_append(c.handle, k, v, seq.to(cuda), lens, number=torch.full((B,), step, dtype=torch.int32, device=cuda),
                             q=q, pos=pos.to(cuda), rope=cfg)
        lens = lens + (seq >= 0).int().to(cuda)
        for b in range(B):
            if seq[b] >= 0:
                i = int(lens[b]) - 1
                p, s = int(c.table[b, i // page]), i % page
                for h in range(kv):
                    entries[b][h].append([f64(c.k[p, h, s]), f64(c.v[p, h, s]), 0.0, step])
        want_k, size = rope(f64(k), pos.numpy(), 32, [6, 5, 5], 1e4, 0, DEALT)
        for b in range(B):
            if seq[b] >= 0:
                i = int(lens[b]) - 1
                rope_close(c.k[int(c.table[b, i // page]), :, i % page], want_k[b], size[b], "bf16")
        got = ofb.attn_decode(c.handle, qr, lens, accumulate=True)
        for b in range(B):
            for h in range(kv):
                e = entries[b][h]
                o, w, size = attend(f64(qr[b, h * G:(h + 1) * G]), np.stack([x[0] for x in e])[:, None], np.stack([x[1] for x in e])[:, None], d ** -0.5)
                assert (np.abs(f64(got[b, h * G:(h + 1) * G]) - o) <= attend_tol(size, d)[:, None] * 5 + 2.0 ** -24 * np.abs(o)).all(), step
                have = f64(c.rows("weight", b, len(e)))[:, h]
                for x, a, y in zip(e, w[:, 0], have):
                    assert abs(x[2] + a - y) <= attend_tol(size, d).max() * a + 2.0 ** -23 * y
                    x[2] = float(y)  # from here on with the cache's own f32 value
        if int(lens.max()) >= budget:
            kept, lens = ofb.kv_evict(c.handle, lens, keep=keep, recent=6)
            for b in range(B):
                for h in range(kv):
                    e = entries[b][h]
                    src = evict(np.array([x[2] for x in e]), np.array([x[3] for x in e]), keep, 6)
                    assert kept[b, h, :len(src)].tolist() == src.tolist() and (kept[b, h, len(src):] == -1).all()
                    entries[b][h] = [e[i] for i in src]
    assert c.handle.device_errors() == 0


def test_side_stream_and_own_scratch(ofb, cuda):
    c = Cache(ofb, [3000, 70], 2, 128, 16, meta=True)
    q = torch.randn(2, 8, 128, device=cuda)
    want = ofb.attn_decode(c.handle, q, c.dlens)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = [[ofb.attn_decode(c.handle, q, c.dlens, stream=s) for s in side] for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(want, x) for r in got for x in r)


def test_graph_replays_the_step(ofb, cuda):
    # rotate, append, attend with weights and evict, captured once and replayed on new contents
    c = Cache(ofb, [600, 90], 2, 128, 16, reach=700, meta=True)
    cfg = ofb.RopeConfig(128)
    k, v = torch.randn(2, 2, 2, 128, device=cuda)
    q = torch.randn(2, 8, 128, device=cuda)
    seq = torch.arange(2, dtype=torch.int32, device=cuda)
    index, pos = torch.tensor([600, 90], dtype=torch.int32, device=cuda), torch.tensor([[600, 90]], dtype=torch.int32, device=cuda)
    scratch, ev = ofb.attn_scratch(c.handle, 8, 2, 0, True), ofb.evict_scratch(c.handle, 2, 500)

    def step():
        qr = ofb.rope_append(c.handle, k, v, seq, index, q=q, pos=pos, rope=cfg)
        out = ofb.attn_decode(c.handle, qr, index + 1, accumulate=True, scratch=scratch)
        kept, lens = ofb.kv_evict(c.handle, index + 1, keep=500, recent=20, scratch=ev)
        return out, kept, lens

    state = [t.clone() for t in (c.k, c.v, c.weight, c.order)]
    restore = lambda: [t.copy_(s) for t, s in zip((c.k, c.v, c.weight, c.order), state)]  # noqa: E731
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step()
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for seed in range(3):
        torch.manual_seed(seed)
        for t in (k, v, q):
            t.normal_()
        restore()
        eager = [t.clone() for t in step()]
        after = [t.clone() for t in (c.k, c.v, c.weight, c.order)]
        restore()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, res))
        for a, t in zip(after, (c.k, c.v, c.weight, c.order)):
            it = {2: torch.int16, 4: torch.int32}[t.element_size()]
            assert torch.equal(a.view(it), t.view(it))

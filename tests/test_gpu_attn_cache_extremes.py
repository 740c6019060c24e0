"""The attention cache at the ends of its ranges: NaN and infinity among the attended
entries, and rotary positions over all of int32 against angles of 50 digits."""
from decimal import Decimal, getcontext

import numpy as np
import pytest
import torch

from attn_cache_paths import GpuCache
from attn_cache_ref import DT, HALF_STEP, f64, pair_tables

pytestmark = pytest.mark.gpu


# ---- NaN and infinity among the entries ----------------------------------------------

SHORT, LONG = [300, 90, 33], [20000, 90, 3000]  # clusters; runs and a join


@pytest.mark.parametrize("lens", [SHORT, LONG], ids=["short", "long"])
@pytest.mark.parametrize("cache,io,G,d", [("bf16", "f32", 4, 128), ("f16", "f32", 4, 64), ("bf16", "bf16", 12, 64), ("f16", "f16", 3, 256),
                                          ("bf16", "f32", 8, 256), ("f16", "f32", 12, 256)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")], ids=str)
def test_attention_keeps_nan_and_infinity_where_they_are(ofb, cuda, lens, cache, io, G, d, value):
    kv, bits = 2, lambda t: t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)  # noqa: E731
    c = GpuCache(ofb, lens, kv, d, 16, cache, seed=d + G)
    q = torch.randn(len(lens), kv * G, d, device=cuda).to(DT[io])
    weight = c.weight.clone()

    def call():
        c.weight.copy_(weight)
        return ofb.attn_decode(c.handle, q, c.dlens, accumulate=True).view(len(lens), kv, G, d), c.weight.clone()

    good, grown = call()
    assert torch.isfinite(good).all() and torch.isfinite(grown[c.live]).all()

    def only(out, where):  # all but `where` of the output is what it was
        rest = torch.ones_like(out, dtype=torch.bool)
        rest[where] = False
        assert torch.equal(bits(out)[rest], bits(good)[rest])
        return out[where]

    p, s = (int(x[17]) for x in c.at(0, 18))  # entry 17 of sequence 0
    # a value: its column of its kv head's query heads
    old = c.v[p, 1, s, 5].clone()
    c.v[p, 1, s, 5] = value
    out, w = call()
    assert not torch.isfinite(only(out, (0, 1, slice(None), 5))).any()
    assert torch.equal(bits(w), bits(grown))  # weights do not go by the values
    c.v[p, 1, s, 5] = old
    # a key: NaN makes all of its kv head's query heads NaN; an infinity may leave it without weight
    old = c.k[p, 0, s, 3].clone()
    c.k[p, 0, s, 3] = value
    out, w = call()
    touched = only(out, (0, 0))
    other = torch.ones_like(w, dtype=torch.bool)
    at = c.at(0, lens[0])
    other[at[0], 0, at[1]] = False
    assert torch.equal(bits(w)[other], bits(grown)[other])
    if value != value:
        assert touched.isnan().all() and w[at[0], 0, at[1]].isnan().all()
    c.k[p, 0, s, 3] = old
    # a query: its head
    old = q[0, G + 1, 2].clone()
    q[0, G + 1, 2] = value
    out, _ = call()
    assert only(out, (0, 1, 1)).isnan().all()
    q[0, G + 1, 2] = old
    out, w = call()
    assert torch.equal(bits(out), bits(good)) and torch.equal(bits(w), bits(grown)) and c.handle.device_errors() == 0


# ---- rotary positions far off ------------------------------------------------------------

def places(pos, pairs, rot, section, base, order, per_axis):
    """Angles of positions pos [axes, T], reduced to one turn with 50 digits, as float64 [T, pairs]."""
    getcontext().prec = 60

    def atan_inv(x):  # Machin's formula for pi
        total = term = Decimal(1) / x
        n = 1
        while abs(term) > Decimal(10) ** -58:
            term = -term / (x * x)
            n += 2
            total += term / n
        return total

    two_pi = 8 * (4 * atan_inv(5) - atan_inv(239))
    axis, _ = pair_tables(rot, section, base, order, per_axis)
    out = np.empty((pos.shape[1], pairs))
    for i in range(pairs):
        first = sum(section[:axis[i]])
        power = Decimal(-(i - first)) / section[axis[i]] if per_axis else Decimal(-i) / pairs
        turns = (Decimal(base).ln() * power).exp() / two_pi
        for t in range(pos.shape[1]):
            place = Decimal(int(pos[axis[i], t])) * turns % 1
            out[t, i] = float((place - place.to_integral_value()) * two_pi)
    return out


# The place in the turn: rounded to f32 (2^-25 half turns) from a word of 32 bits (2^-31);
# the frequency, of at most 1 / 2 pi, comes from up to 127 products in 64 bits of a power
# within a step of 64 bits (rounding by 2^-64 and 2^-63 of it each, (3 * 127 + 1) 2^-64 / 2 pi
# in all) and is cut off after 64 bits: 62 * 2^-64 turns, at positions up to 2^31 less
# than 2^-26 half turns. Together less than 2^-24.4, times pi less than 2^-22.7. Then
# sincospif's two steps and three roundings, as for near positions.
FAR_TOL = 2.0 ** -22.7 + 2 * 2.0 ** -23 + 3 * 2.0 ** -24


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("rot,section,base,order,per_axis", [
    (256, [128], 10000.0, 0, False), (256, [128], 2.0, 0, False), (128, [24, 20, 20], 1e7, 1, False), (64, [16, 16], 100.0, 0, True),
    (20, [10], 1.0, 0, False)])
def test_rope_far_positions(ofb, cuda, rot, section, base, order, per_axis, io):
    ends = [2 ** 31 - 1, -2 ** 31, 2 ** 30 + 1, -2 ** 30 - 12345, 2 ** 24 + 1, 999999937, -1]
    pos = np.array([np.roll(ends, a) for a in range(len(section))])
    x = torch.randn(len(ends), 3, 256, generator=torch.Generator().manual_seed(rot)).to(DT[io])
    cfg = ofb.RopeConfig(rot, section, base=base, order=order, per_axis=per_axis)
    got = f64(ofb.rope(x.to(cuda), torch.as_tensor(pos, dtype=torch.int32, device=cuda), cfg))
    angle = places(pos, rot // 2, rot, section, base, order, per_axis)[:, None]
    x = f64(x)
    u, v = x[..., :rot // 2], x[..., rot // 2:rot]
    want = np.concatenate([u * np.cos(angle) - v * np.sin(angle), v * np.cos(angle) + u * np.sin(angle), x[..., rot:]], -1)
    size = np.concatenate([np.abs(u) + np.abs(v)] * 2 + [np.zeros_like(x[..., rot:])], -1)
    err, tol = np.abs(got - want), FAR_TOL * size + HALF_STEP[io] * np.abs(want)
    assert (err <= tol).all(), f"off by {(err - tol).max()} more than the bound"

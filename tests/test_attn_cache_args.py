"""Refusals of the attention-cache operators: each bad argument gives its
status and a reason before anything is launched (runs without a GPU; the
pointers are never followed)."""
import ctypes

import pytest
import torch

P = 1 << 20  # a non-NULL, aligned address that no refused call reads


def rope_cfg(ofb, **kw):
    a = dict(rot_dim=128, section=[24, 20, 20], base=1e6, pairing=0, order=0, per_axis=False)
    a.update(kw)
    return ofb.RopeConfig(**a)


def cache_struct(ofb, **kw):
    a = dict(k=P, v=P, weight=P, order=P, page_table=P, errors=0, page_stride=0, type=ofb.TYPE_BF16, n_kv_heads=2,
             head_dim=128, page_size=16, n_pages=100, n_seqs=4, max_pages=20)
    a.update(kw)
    return ofb.KvCacheStruct(**a)


def call_rope(ofb, cfg=None, x=P, type=0, T=5, H=4, d=128, xs=512, pos=P, ps=5, out=2 * P, os=512):
    cfg = rope_cfg(ofb) if cfg is None else cfg
    return ofb.lib.ofb_rope(ctypes.byref(cfg) if cfg else None, x, type, T, H, d, xs, pos, ps, out, os, None)


def call_append(ofb, c=None, cfg=None, type=0, T=5, H=4, q=P, qs=512, k=P, ks=256, v=P, vs=256, pos=P, ps=5, seq=P, index=P,
                number=P, qo=2 * P, qos=512):
    c, cfg = c or cache_struct(ofb), cfg or rope_cfg(ofb)
    return ofb.lib.ofb_rope_append(ctypes.byref(c), ctypes.byref(cfg), type, T, H, q, qs, k, ks, v, vs, pos, ps, seq, index,
                                   number, qo, qos, None)


def call_attn(ofb, c=None, q=P, type=0, qs=512, H=4, scale=0.1, lens=P, B=4, max_len=0, acc=0, out=2 * P, os=512, scratch=4 * P,
              size=1 << 40):
    c = c or cache_struct(ofb)
    return ofb.lib.ofb_attn_decode(ctypes.byref(c), q, type, qs, H, scale, lens, B, max_len, acc, out, os, scratch, size, None)


def call_evict(ofb, c=None, lens=P, B=4, max_len=0, keep=64, recent=8, lens_out=2 * P, kept=P, scratch=4 * P, size=1 << 40):
    c = c or cache_struct(ofb)
    return ofb.lib.ofb_kv_evict(ctypes.byref(c), lens, B, max_len, keep, recent, lens_out, kept, scratch, size, None)


def refused(ofb, st, want):
    assert st == want, (st, ofb.lib.ofb_last_error())
    assert ofb.lib.ofb_last_error()


BAD_ROPE = [dict(rot_dim=0, section=[0]), dict(rot_dim=130), dict(rot_dim=127), dict(section=[24, 20, 19]), dict(section=[84, -10, -10]),
            dict(base=0.0), dict(base=-1.0), dict(base=float("inf")), dict(base=float("nan")), dict(pairing=2), dict(order=2),
            dict(order=1, per_axis=True), dict(order=1, section=[20, 22, 22]), dict(rot_dim=256, section=[128])]


@pytest.mark.parametrize("kw", BAD_ROPE, ids=str)
def test_rotary_form_refused(ofb, kw):
    cfg = rope_cfg(ofb, **kw)
    refused(ofb, call_rope(ofb, cfg=cfg), ofb.EINVAL)
    refused(ofb, call_append(ofb, cfg=cfg), ofb.EINVAL)


def test_rope_config_axes(ofb):
    with pytest.raises(ofb.OfbError):
        ofb.RopeConfig(16, [2, 2, 2, 1, 1])
    with pytest.raises(ofb.OfbError):
        ofb.RopeConfig(16, [])


@pytest.mark.parametrize("kw,want", [
    (dict(x=None), 1), (dict(pos=None), 1), (dict(out=None), 1), (dict(T=-1), 1), (dict(H=0), 1), (dict(d=0), 1), (dict(d=2048), 1),
    (dict(type=12), 4), (dict(xs=511), 1), (dict(os=100), 1), (dict(ps=4), 1), (dict(out=P, os=1024), 1), (dict(x=P + 2), 1),
    (dict(pos=P + 1), 1), (dict(xs=-512), 1), (dict(T=1, ps=0), 1), (dict(T=1, ps=-3), 1), (dict(T=(1 << 30) + 1, ps=1 << 40), 5)], ids=str)
def test_rope_refused(ofb, kw, want):
    refused(ofb, call_rope(ofb, **kw), want)


BAD_CACHE = [(dict(k=None), 1), (dict(v=None), 1), (dict(page_table=None), 1), (dict(type=0), 4), (dict(type=12), 4),
             (dict(head_dim=80), 4), (dict(head_dim=0), 4), (dict(n_kv_heads=0), 1), (dict(n_kv_heads=2000), 1), (dict(page_size=0), 1),
             (dict(page_size=1 << 20), 1), (dict(n_pages=0), 1), (dict(n_seqs=0), 1), (dict(max_pages=0), 1), (dict(page_stride=4088), 1),
             (dict(page_stride=4100), 1), (dict(page_stride=-8), 1), (dict(k=P + 8), 1), (dict(v=P + 2), 1), (dict(weight=P + 2), 1),
             (dict(errors=P + 1), 1)]


@pytest.mark.parametrize("kw,want", BAD_CACHE, ids=str)
def test_cache_refused(ofb, kw, want):
    c = cache_struct(ofb, **kw)
    refused(ofb, call_append(ofb, c), want)
    refused(ofb, call_attn(ofb, c), want)
    refused(ofb, call_evict(ofb, c), want)
    assert ofb.lib.ofb_attn_scratch_size(ctypes.byref(c), 4, 4, 0, 0) == 0
    assert ofb.lib.ofb_kv_evict_scratch_size(ctypes.byref(c), 4, 64) == 0


@pytest.mark.parametrize("kw,want", [
    (dict(type=1), 4), (dict(type=14), 4), (dict(T=-1), 1), (dict(H=-1), 1), (dict(H=0), 1), (dict(k=None), 1), (dict(v=None), 1),
    (dict(seq=None), 1), (dict(index=None), 1), (dict(pos=None), 1), (dict(qo=None), 1), (dict(qs=511), 1), (dict(ks=255), 1),
    (dict(vs=0), 1), (dict(qos=1), 1), (dict(ps=3), 1), (dict(qo=P, qos=1024), 1), (dict(k=P + 1), 1), (dict(seq=P + 2), 1),
    (dict(T=1, ps=-1), 1), (dict(T=(1 << 30) + 1, ps=1 << 40), 5)], ids=str)
def test_append_refused(ofb, kw, want):
    refused(ofb, call_append(ofb, **kw), want)


@pytest.mark.parametrize("kw,want", [
    (dict(type=1), 4), (dict(q=None), 1), (dict(lens=None), 1), (dict(out=None), 1), (dict(out=P), 1), (dict(H=5), 1), (dict(H=0), 1),
    (dict(B=5), 1), (dict(B=-1), 1), (dict(max_len=-1), 1), (dict(acc=2), 1), (dict(qs=511), 1), (dict(os=0), 1), (dict(q=P + 2), 1),
    (dict(scale=float("nan")), 1), (dict(scratch=None), 1), (dict(scratch=P + 8), 1), (dict(size=100), 5)], ids=str)
def test_attention_refused(ofb, kw, want):
    refused(ofb, call_attn(ofb, **kw), want)


def test_attention_limits(ofb):
    refused(ofb, call_attn(ofb, cache_struct(ofb, weight=None), acc=1), ofb.EINVAL)
    refused(ofb, call_attn(ofb, cache_struct(ofb, n_seqs=4096), B=4096), ofb.ETOOLARGE)
    refused(ofb, call_attn(ofb, cache_struct(ofb, n_seqs=2048, max_pages=1 << 24), B=2048), ofb.ETOOLARGE)
    # the scratch a call of fewer sequences or shorter ones needs is no larger
    c = cache_struct(ofb)
    size = lambda *a: ofb.lib.ofb_attn_scratch_size(ctypes.byref(c), *a)  # noqa: E731
    assert size(4, 4, 0, 1) >= size(4, 3, 0, 1) > size(4, 3, 100, 1) > size(4, 3, 100, 0) > 0


@pytest.mark.parametrize("kw,want", [
    (dict(lens=None), 1), (dict(lens_out=None), 1), (dict(lens_out=P), 1), (dict(lens_out=P + 12), 1), (dict(keep=0), 1), (dict(keep=-4), 1),
    (dict(recent=-1), 1), (dict(recent=65), 1), (dict(B=5), 1), (dict(max_len=-1), 1), (dict(scratch=None), 1), (dict(scratch=P + 4), 1),
    (dict(size=4 * 2 * 2 * 64 * 4 - 1), 5), (dict(kept=P + 1), 1)], ids=str)
def test_eviction_refused(ofb, kw, want):
    refused(ofb, call_evict(ofb, **kw), want)


def test_eviction_limits(ofb):
    refused(ofb, call_evict(ofb, cache_struct(ofb, weight=None)), ofb.EINVAL)
    refused(ofb, call_evict(ofb, cache_struct(ofb, order=None)), ofb.EINVAL)
    refused(ofb, call_evict(ofb, cache_struct(ofb, max_pages=1 << 20)), ofb.ETOOLARGE)
    refused(ofb, call_evict(ofb, cache_struct(ofb, max_pages=1 << 20), max_len=ofb.EVICT_MAX_LEN + 1), ofb.ETOOLARGE)


def test_nothing_to_do_is_ok(ofb):
    assert call_rope(ofb, T=0) == ofb.OK
    assert call_append(ofb, T=0) == ofb.OK
    assert call_attn(ofb, B=0) == ofb.OK
    assert call_evict(ofb, B=0) == ofb.OK


def test_binding_refuses_host_tensors_and_wrong_shapes(ofb):
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)  # noqa: E731
    i32 = torch.int32
    c = ofb.KvCache(z(3, 2, 16, 64), z(3, 2, 16, 64), z(1, 2, dt=i32), z(3, 2, 16, dt=torch.float32), z(3, 2, 16, dt=i32))
    q, lens = z(1, 4, 64), z(1, dt=i32)
    for bad in (lambda: ofb.KvCache(z(3, 2, 16, 64), z(3, 2, 16, 32), z(1, 2, dt=i32)),
                lambda: ofb.KvCache(z(3, 2, 16, 64, dt=torch.float32), z(3, 2, 16, 64, dt=torch.float32), z(1, 2, dt=i32)),
                lambda: ofb.KvCache(z(3, 2, 64, 16).transpose(2, 3), z(3, 2, 64, 16).transpose(2, 3), z(1, 2, dt=i32)),
                lambda: ofb.KvCache(z(1, 2, 16, 64).expand(3, -1, -1, -1), z(1, 2, 16, 64).expand(3, -1, -1, -1), z(1, 2, dt=i32)),
                lambda: ofb.KvCache(z(3, 2, 16, 64), z(3, 4, 16, 64)[:, :2], z(1, 2, dt=i32)),
                lambda: ofb.KvCache(z(3, 2, 16, 64), z(3, 2, 16, 64), z(1, 2, dt=torch.int64)),
                lambda: ofb.KvCache(z(3, 2, 16, 64), z(3, 2, 16, 64), z(1, 2, dt=i32), weight=z(3, 16, 2, dt=torch.float32)),
                lambda: ofb.attn_decode(c, q, lens),  # host tensors
                lambda: ofb.attn_decode(c, z(1, 4, 32), lens),
                lambda: ofb.attn_decode(c, q.half(), lens),
                lambda: ofb.attn_decode(c, q, z(2, dt=i32)),
                lambda: ofb.attn_decode(c, z(1, 64, 4).transpose(1, 2), lens),
                lambda: ofb.kv_evict(c, z(1, dt=torch.int64), 4),
                lambda: ofb.kv_evict(c, lens, 4),
                lambda: ofb.rope(z(2, 4, 64), z(1, 3, dt=i32), ofb.RopeConfig(64)),
                lambda: ofb.rope(z(2, 4, 64), z(1, 2, dt=i32), ofb.RopeConfig(64)),
                lambda: ofb.rope_append(c, z(1, 2, 64), z(1, 2, 64), lens, lens, rope=ofb.RopeConfig(64)),
                lambda: ofb.rope_append(c, z(1, 2, 64), z(1, 1, 64), lens, lens),
                lambda: ofb.rope_append(c, z(1, 2, 64), z(1, 2, 64), lens, lens)):
        with pytest.raises(ofb.OfbError) as e:
            bad()
        assert e.value.status == ofb.EINVAL

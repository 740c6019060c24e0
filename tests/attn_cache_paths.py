"""For the tests of the attention cache's paths: which launch a call's sizes lead
to (restated from the dispatch rules), caches built on the GPU, and 64-bit
restatements that run there, for sizes at which host loops would take too long."""
import re

import numpy as np
import torch

from attn_cache_ref import DT, HALF_STEP, attend_tol


# ---- which launch a call takes ---------------------------------------------------

def launches(call, tmp_path):
    """(mangled kernel name, CTAs, threads of a CTA, dynamic shared memory) of each
    launch of call(), which is captured into a graph and not run."""
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    graph.enable_debug_mode()
    with torch.cuda.graph(graph):
        call()
    graph.debug_dump(str(tmp_path / "graph.dot"))
    text = (tmp_path / "graph.dot").read_text()
    found = re.findall(r"\(topoId: (\d+)\) \| (\w+)\\<\\<\\<(.*?)\\>\\>\\>", text)
    out = []
    for _, name, shape in sorted(found, key=lambda f: -int(f[0])):
        *grid, block, smem = [int(x) for x in re.findall(r"\d+", shape)]
        out.append((name, tuple(grid), block, smem))
    return out


def evict_path(rows, bound, keep, recent, sms=148):
    """(CTAs of a cluster, threads of a CTA, entries of a CTA, whether order
    numbers stay in shared memory, whether rows are copied by the first launch)."""
    ctas, threads, best = 0, 256, 0
    for t in (1024, 512, 256):
        if t > 256 and t > bound // 2:
            continue
        per_sm = 1024 // t
        slots = sms * per_sm
        c = slots // rows
        while c > 1 and 8 * (16 * per_sm // c) < rows:
            c -= 1
        c = min(max(min(c, bound // 4096), 1), 8)
        while c < 8 and -(-bound // c) > 49152:
            c += 1
        n = 0 if rows > slots else rows * c * t
        if not ctas or n > best + best // 8:
            ctas, threads, best = c, t, n
    if not best:
        threads = 256
    chunk = (-(-bound // ctas) + 3) // 4 * 4
    kept = recent > 0 and (4 * (2048 + 2 * chunk) + 5120 + 1024) * (1024 // threads) <= 228 * 1024
    return ctas, threads, chunk, kept, min(bound - keep, keep) <= (48 if rows <= 64 else 128)


# ---- caches ------------------------------------------------------------------------

class GpuCache:
    """A paged cache with `lens` random entries per sequence, made on the GPU;
    `stale` in every place without an entry, page numbers out of range behind
    each sequence's last page."""

    def __init__(self, ofb, lens, kv, d, page, cache="bf16", seed=0, reach=0, stale=float("nan"), meta=True):
        dev = torch.device("cuda")
        g = torch.Generator(dev).manual_seed(seed)
        need = [-(-n // page) for n in lens]
        cols = max(1, max(need), -(-reach // page))
        self.n_pages = n = sum(need) + 2
        free = torch.randperm(n, generator=g, device=dev).to(torch.int32)
        self.table = torch.full((len(lens), cols), 2 ** 31 - 5, dtype=torch.int32, device=dev)
        self.lens, self.kv, self.d, self.page = list(lens), kv, d, page
        live = torch.zeros(n, page, dtype=torch.bool, device=dev)
        self.order = torch.full((n, kv, page), -99, dtype=torch.int32, device=dev)
        at = 0
        for b, m in enumerate(lens):
            self.table[b, :need[b]] = free[at:at + need[b]]
            at += need[b]
            p, s = self.at(b, m)
            live[p, s] = True
            self.order[p, :, s] = torch.rand(m, kv, generator=g, device=dev).argsort(0).to(torch.int32)
        self.live = live[:, None].expand(n, kv, page)
        rows = lambda: torch.where(self.live[..., None], torch.randn(n, kv, page, d, generator=g, device=dev), stale).to(DT[cache])  # noqa: E731
        self.k, self.v = rows(), rows()
        self.weight = torch.where(self.live, torch.randn(n, kv, page, generator=g, device=dev).exp(), stale)
        self.dlens = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.handle = ofb.KvCache(self.k, self.v, self.table, weight=self.weight if meta else None, order=self.order if meta else None)

    def at(self, b, n):
        """(pages, slots) of the first n entries of sequence b."""
        i = torch.arange(n, device=self.table.device)
        return self.table[b, i // self.page].long(), i % self.page

    def rows(self, name, b, n):
        """[n, kv, ...] of the first n entries of sequence b."""
        p, s = self.at(b, n)
        return getattr(self, name)[p, :, s]


# ---- 64-bit results ------------------------------------------------------------------

def evict_source(weight, order, keep, recent):
    """weight, order [n] -> source place of each of the first min(n, keep) entries."""
    n = len(weight)
    src = np.arange(min(n, keep))
    if n <= keep:
        return src
    order = order.astype(np.int64)
    old = order <= order.max() - recent if recent else np.ones(n, bool)
    heavy = np.where(np.isnan(weight), -np.inf, weight.astype(np.float64))
    best = np.lexsort((np.arange(n), np.isnan(weight) & old, np.where(old, -heavy, 0), old))[:keep]
    stays = np.zeros(n, bool)
    stays[best] = True
    src[~stays[:keep]] = np.flatnonzero(stays[keep:]) + keep
    return src


def check_eviction(ofb, c, keep, recent, max_len=0):
    """One kv_evict call against evict_source, everything it must leave included."""
    names = ("k", "v", "weight", "order")
    bits = lambda t: t.view(torch.int16 if t.element_size() == 2 else torch.int32)  # noqa: E731
    want = {x: bits(getattr(c, x)).clone() for x in names}
    lens = [min(n, max_len) if max_len else n for n in c.lens]
    kept_want = np.full((len(lens), c.kv, keep), -1)
    for b, n in enumerate(lens):
        w, o = c.rows("weight", b, n).cpu().numpy(), c.rows("order", b, n).cpu().numpy()
        p, s = c.at(b, n)
        for h in range(c.kv):
            src = evict_source(w[:, h], o[:, h], keep, recent)
            kept_want[b, h, :len(src)] = src
            moved = np.flatnonzero(src != np.arange(len(src)))
            to, of = (torch.as_tensor(x, device=p.device) for x in (moved, src[moved]))
            for x in names:
                want[x][p[to], h, s[to]] = bits(getattr(c, x))[p[of], h, s[of]]
    kept, new = ofb.kv_evict(c.handle, c.dlens, keep=keep, recent=recent, max_len=max_len)
    assert np.array_equal(kept.cpu().numpy(), kept_want)
    assert new.tolist() == [min(n, keep) for n in lens]
    for x in names:
        assert torch.equal(bits(getattr(c, x)), want[x]), x
    assert c.handle.device_errors() == 0


def check_attention(c, q, got, io, scale, weight_before=None):
    """One attn_decode call's output, and weights, against softmax in 64 bits; the
    bounds are those of the tests on small caches."""
    H, d = q.shape[1:]
    G = H // c.kv
    for b, n in enumerate(c.lens):
        if not n:
            assert (got[b] == 0).all()
            continue
        k, v = (c.rows(x, b, n).double().transpose(0, 1) for x in "kv")  # [kv, n, d]
        x = q[b].double().view(c.kv, G, d)
        p = torch.softmax(scale * (x @ k.mT), -1)
        want, p = p @ v, p.sum(1)
        size = abs(scale) * (x.abs() @ k.abs().mT).amax(-1, keepdim=True)
        tol = attend_tol(size, d)
        bound = (tol + (2.0 ** -17 if io == "bf16" else 0)) * v.abs().max() + HALF_STEP[io] * want.abs() + 2.0 ** -25 * (io == "f16")
        err = (got[b].double().view(want.shape) - want).abs()
        assert (err <= bound).all(), f"sequence {b} of {n}: off by {err.max()}, bound {bound.max()}"
        if weight_before is not None:
            pg, s = c.at(b, n)
            old, new = weight_before[pg, :, s].double().T, c.weight[pg, :, s].double().T
            slack = tol.amax(1) * p + 2.0 ** -23 * (old.abs() + p)
            assert ((new - old - p).abs() <= slack).all(), f"weights of sequence {b}"
    if weight_before is not None:
        assert torch.equal(c.weight.view(torch.int32)[~c.live], weight_before.view(torch.int32)[~c.live])
    assert c.handle.device_errors() == 0

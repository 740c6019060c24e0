"""Plain 64-bit restatements (numpy) of the attention-cache operators, for the
tests: rotary positions, attention of one token, eviction, on caches built
with stale NaN in every place that holds no entry."""
import numpy as np
import torch

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def f64(t):
    return t.detach().double().cpu().numpy()


def pair_tables(rot, section, base, order, per_axis):
    """(axis, frequency) of each pair."""
    n, pairs, axis, freq = len(section), rot // 2, [], []
    if order == 0:
        for a, k in enumerate(section):
            for j in range(k):
                freq.append(base ** (-j / k) if per_axis else base ** (-len(axis) / pairs))
                axis.append(a)
    else:
        for i in range(pairs):
            axis.append(i % n if i // n < section[i % n] else 0)
            freq.append(base ** (-i / pairs))
    return np.array(axis), np.array(freq)


def rope(x, pos, rot, section, base=10000.0, pairing=0, order=0, per_axis=False):
    """x [T, H, d] float64, pos [axes, T] -> (turned x, |u| + |v| of each element's pair)."""
    axis, freq = pair_tables(rot, section, base, order, per_axis)
    a = pos[axis].T.astype(np.float64) * freq  # [T, pairs]
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    u = np.arange(rot // 2) * (2 if pairing else 1)
    v = u + (1 if pairing else rot // 2)
    y, size = x.copy(), np.zeros_like(x)
    y[..., u] = x[..., u] * c - x[..., v] * s
    y[..., v] = x[..., v] * c + x[..., u] * s
    size[..., u] = size[..., v] = np.abs(x[..., u]) + np.abs(x[..., v])
    return y, size


# The angle is off by 2^-25 half turns (pi * 2^-25 < 2^-23), sincospif by two
# steps of its result (2^-23 each), three roundings follow (2^-24 each).
ROPE_TOL = 2.0 ** -23 + 2 * 2.0 ** -23 + 3 * 2.0 ** -24


def rope_close(got, want, size, io):
    err, tol = np.abs(f64(got) - want), ROPE_TOL * size + HALF_STEP[io] * np.abs(want) + (2.0 ** -25 if io == "f16" else 0)
    assert (err <= tol).all(), f"off by {(err - tol).max()} more than the bound"


class Cache:
    """A paged cache with `lens` random entries per sequence; NaN elsewhere,
    page numbers out of range behind each sequence's last page."""

    def __init__(self, ofb, lens, kv, d, page, cache="bf16", seed=0, dev="cuda", spread=0, reach=None, meta=False):
        g = torch.Generator().manual_seed(seed)
        B = len(lens)
        cols = max(1, max(-(-l // page) for l in (list(lens) + [reach or 0])))
        need = [-(-(reach or l) // page) for l in lens]
        self.n_pages = n = sum(need) + 2
        free = torch.randperm(n, generator=g)[:sum(need)].to(torch.int32)
        table = torch.where(torch.rand(B, cols, generator=g) < 0.5, torch.tensor(-7), torch.tensor(2 ** 31 - 5)).to(torch.int32)
        at = 0
        for b, k in enumerate(need):
            table[b, :k] = free[at:at + k]
            at += k
        dt, shape = DT[cache], (n, kv, page, d)
        rows = []
        for _ in range(2):
            r = torch.full((n, kv * page * d + spread), float("nan"), dtype=dt)
            x = r[:, :kv * page * d].view(shape)
            for b, l in enumerate(lens):
                for i0 in range(0, l, page):
                    m = min(page, l - i0)
                    x[table[b, i0 // page], :, :m] = torch.randn(kv, m, d, generator=g).to(dt)
            rows.append(r.to(dev)[:, :kv * page * d].view(shape))
        self.k, self.v = rows
        self.table, self.lens, self.page, self.kv, self.d = table.to(dev), list(lens), page, kv, d
        self.weight = torch.full((n, kv, page), float("nan"))
        self.order = torch.full((n, kv, page), -99, dtype=torch.int32)
        for b, l in enumerate(lens):
            for h in range(kv):
                p, s = self.at(b, l)
                self.weight[p, h, s] = torch.randn(l, generator=g).exp()
                self.order[p, h, s] = torch.randperm(l, generator=g).to(torch.int32)
        self.weight, self.order = self.weight.to(dev), self.order.to(dev)
        self.dlens = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.handle = ofb.KvCache(self.k, self.v, self.table, weight=self.weight if meta else None, order=self.order if meta else None)

    def at(self, b, n, table=None):
        """(pages, slots) of the first n entries of sequence b."""
        i = torch.arange(n)
        t = (self.table if table is None else table)[b].cpu().long()
        return t[i // self.page] if n else i, i % self.page

    def rows(self, name, b, n):
        """[n, kv, ...] of the first n entries of sequence b."""
        p, s = self.at(b, n)
        t = getattr(self, name)
        return t[p.to(t.device), :, s.to(t.device)]


def attend(q, k, v, scale):
    """q [H, d], k, v [n, kv, d] float64 -> (out [H, d], weights [n, kv], bound on |z|'s terms [H])."""
    H, d = q.shape
    n, kv = k.shape[:2]
    if not n:
        return np.zeros((H, d)), np.zeros((0, kv)), np.zeros(H)
    kh, vh = np.repeat(k, H // kv, 1), np.repeat(v, H // kv, 1)
    z = scale * np.einsum("hd,nhd->hn", q, kh)
    size = abs(scale) * np.einsum("hd,nhd->hn", np.abs(q), np.abs(kh)).max(1)
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    return np.einsum("hn,nhd->hd", p, vh), p.reshape(kv, H // kv, n).sum(1).T, size


def attend_tol(size, d):
    """Bound on the relative error of a probability before its split: a score's
    terms are summed 16 at a time by the tensor core, which may cut off a whole
    step (2^-23) at each of d/16 additions, and by 4 f32 additions; a query's
    parts leave 2^-22 of it (fp16, the coarser); the score is scaled (2^-23).
    exp doubles a score's error at most for errors this small, numerator and
    denominator each have it; exp2f and the sums add 2^-20."""
    return 4 * size * ((d / 16 + 6) * 2.0 ** -23 + 2.0 ** -22) + 2.0 ** -20


def evict(weight, order, keep, recent):
    """weight, order [n] -> source place of each of the first min(n, keep) entries."""
    n = len(weight)
    src = np.arange(min(n, keep))
    if n <= keep:
        return src
    young = order.astype(np.int64) > int(order.max()) - recent if recent else np.zeros(n, bool)
    ranked = sorted(range(n), key=lambda i: (not young[i], 0 if young[i] else -weight[i] if weight[i] == weight[i] else np.inf, i))
    stays = np.zeros(n, bool)
    stays[ranked[:keep]] = True
    src[~stays[:keep]] = np.flatnonzero(stays[keep:]) + keep
    return src

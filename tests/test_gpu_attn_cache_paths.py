"""The attention cache's launches by size: calls at either side of each rule that
chooses a launch, each of which says which one it is for."""
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

from attn_cache_paths import GpuCache, check_attention, check_eviction, evict_path, launches
from attn_cache_ref import DT

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:DEBUG. ")]


def one_long(seqs, bound, short=700):
    """Lengths of which the second (or only) one is `bound`."""
    lens = [(short - 37 * b) % short for b in range(seqs)]
    lens[min(1, seqs - 1)] = bound
    return lens


# ---- eviction ----------------------------------------------------------------------

# Lengths at which keys and order numbers together are close to all the shared memory
# that a CTA can have (232448 bytes): chunks of 26840 entries take 222912 and, with the
# kernel's own arrays, less than that; 27392 are the last whose order numbers stay.
EDGES = [  # sequences, kv heads, largest length, whether order numbers stay
    (5, 8, 80520, True), (5, 8, 80521, True), (5, 8, 82176, True), (5, 8, 82177, False),
    (1, 2, 214720, True), (1, 2, 215040, True), (1, 2, 219136, True), (1, 2, 219137, False),
    (16, 8, 27008, True), (16, 8, 27392, True), (16, 8, 27396, False), (12, 2, 135000, True), (10, 3, 108000, True),
    (20, 4, 54000, True),
]


@pytest.mark.parametrize("seqs,kv,bound,stay", EDGES)
def test_eviction_near_all_shared_memory(ofb, cuda, seqs, kv, bound, stay):
    keep, recent = 500, 20
    assert evict_path(seqs * kv, bound, keep, recent)[3] == stay
    c = GpuCache(ofb, one_long(seqs, bound), kv, 64, 64, seed=bound)
    check_eviction(ofb, c, keep, recent, max_len=bound)


def test_eviction_by_the_tables_reach(ofb, cuda):
    # no max_len: the table's reach bounds the lengths, here 81920 whatever they are
    c = GpuCache(ofb, [3000] * 5, 8, 64, 64, reach=81920)
    check_eviction(ofb, c, 1024, 64)


# sequences, kv heads, largest length, how many are that long, page, keep, recent, CTAs of a
# cluster, whether order numbers stay in shared memory
EVICT_PATHS = [
    (64, 8, 6000, 3, 16, 700, 50, 1, False),        # order numbers read a second time: many rows ...
    (64, 8, 6000, 3, 7, 700, 50, 1, False),
    (64, 8, 5504, 2, 16, 700, 50, 1, True),         # (the last length at which they stay)
    (16, 8, 28000, 2, 64, 3000, 100, 1, False),
    (1, 1, 260000, 1, 64, 9000, 1000, 8, False),    # ... and long ones, in clusters
    (1, 1, 260000, 1, 7, 9000, 1000, 8, False),
    (3, 2, 30000, 2, 7, 2000, 100, 7, True),        # clusters, pages of no multiple of 4
    (3, 2, 30000, 2, 10, 2000, 0, 7, False),
    (1, 1, 393216, 1, 64, 300000, 5000, 8, False),  # the longest there is, most of it kept
    (80, 8, 2000, 4, 16, 300, 20, 1, True),         # more rows than have room at once
    (80, 8, 60000, 1, 7, 300, 20, 2, False),        # a cluster because a CTA cannot hold the keys
    (25, 4, 100000, 1, 32, 1000, 20, 3, False),
    (25, 4, 150000, 1, 32, 1000, 0, 4, False),
]


@pytest.mark.parametrize("few_values", [False, True])
@pytest.mark.parametrize("seqs,kv,bound,long,page,keep,recent,ctas,stay", EVICT_PATHS)
def test_eviction_paths(ofb, cuda, tmp_path, seqs, kv, bound, long, page, keep, recent, ctas, stay, few_values):
    if torch.cuda.get_device_properties(cuda).multi_processor_count != 148:
        pytest.skip("sizes chosen for 148 SMs")
    lens = [(keep + 200 - 11 * b) % (keep + 200) for b in range(seqs)]
    lens[-long:] = [bound - 13 * i for i in range(long)]
    c = GpuCache(ofb, lens, kv, 64, page, "f16" if page % 2 else "bf16", seed=bound + page, reach=bound)
    if few_values:  # equals, zeros and NaN across the CTAs of a cluster
        vals = torch.tensor([0.0, -0.0, 1.0, 1.0, float("nan"), float("inf"), 1e-42, 0.25], device=cuda)
        c.weight.copy_(torch.where(c.live, vals[torch.randint(0, 8, c.weight.shape, device=cuda)], c.weight))
    C, threads, chunk, kept, _ = path = evict_path(seqs * kv, bound, keep, recent)
    assert (C, kept) == (ctas, stay), path
    first = launches(lambda: ofb.kv_evict(c.handle, c.dlens, keep=keep, recent=recent, max_len=bound), tmp_path)[0]
    assert "evict_kernel" in first[0] and first[1:] == ((seqs * kv * C,), threads, 4 * (2048 + (2 if kept else 1) * chunk)), first
    check_eviction(ofb, c, keep, recent, max_len=bound)


# ---- attention -----------------------------------------------------------------------

def attention(ofb, c, G, io, tmp_path, acc, path):
    """One call with its launches' names and CTAs: (part of the name, CTAs or None) each."""
    q = (torch.randn(len(c.lens), c.kv * G, c.d, generator=torch.Generator().manual_seed(G)) * 2).to(DT[io]).to(c.k.device)
    before = c.weight.clone()
    call = lambda: ofb.attn_decode(c.handle, q, c.dlens, max_len=max(c.lens), accumulate=acc)  # noqa: E731
    found = launches(call, tmp_path)
    assert len(found) == len(path), found
    for f, (name, ctas) in zip(found, path):
        assert name in f[0] and (ctas is None or f[1] == ctas), (f, name, ctas)
    check_attention(c, q, call(), io, c.d ** -0.5, before if acc else None)


def passes(G, d, io):
    """(heads of a pass, passes)"""
    rows = 16 if G > 8 and (io != "f32" or d <= 128) else 8
    return rows, -(-G // rows)


JOINED = [  # head_dim, query heads of a kv head, cache, activations
    (64, 8, "bf16", "f32"), (64, 12, "f16", "f16"), (64, 20, "bf16", "bf16"), (96, 8, "f16", "f32"), (96, 12, "bf16", "f32"),
    (96, 20, "f16", "f32"), (128, 8, "bf16", "f32"), (128, 12, "f16", "f32"), (128, 20, "bf16", "bf16"), (192, 8, "f16", "f16"),
    (192, 12, "bf16", "f32"), (192, 12, "bf16", "bf16"), (256, 4, "f16", "f32"), (256, 8, "bf16", "f32"), (256, 12, "bf16", "f32"),
    (256, 20, "f16", "f16")]


@pytest.mark.parametrize("acc", [False, True])
@pytest.mark.parametrize("d,G,cache,io", JOINED)
def test_attention_joins_few_parts_of_many_heads(ofb, cuda, tmp_path, d, G, cache, io, acc):
    # 40 ragged sequences x 8 kv heads: a head has a few parts, which a warp joins
    lens = np.random.default_rng(G).integers(1, 1500, size=40).tolist()
    lens[3:9] = 0, 1, 31, 32, 33, 3000
    c = GpuCache(ofb, lens, 8, d, 20 if d == 96 else 16, cache, seed=d, stale=float("inf") if acc else float("nan"))
    R, NB = passes(G, d, io)
    path = [("attn_split_kernelILi%dELi%dE" % (d, R), None), ("attn_join_kernel", (8 * NB * R // 8, 1, 40))]
    attention(ofb, c, G, io, tmp_path, acc, path + [("attn_weight_kernel", (40 * 8 * 3,))] * acc)


@pytest.mark.parametrize("acc", [False, True])
@pytest.mark.parametrize("seqs,kv,G,d,cache,io", [
    (300, 2, 8, 128, "bf16", "f32"), (1536, 1, 8, 64, "f16", "f16"), (1000, 1, 12, 256, "bf16", "bf16"), (700, 3, 20, 96, "bf16", "f32"),
    (1536, 2, 2, 192, "f16", "f32"), (129, 8, 9, 256, "f16", "f32")])
def test_attention_runs_over_many_sequences(ofb, cuda, tmp_path, seqs, kv, G, d, cache, io, acc):
    # many short sequences and a few of several hundred entries: runs that hold many whole parts
    lens = np.random.default_rng(seqs).integers(0, 90, size=seqs).tolist()
    lens[0], lens[seqs // 2], lens[-1] = 5, 700, 333
    c = GpuCache(ofb, lens, kv, d, 16 if seqs % 2 else 24, cache, seed=seqs)
    R, NB = passes(G, d, io)
    path = [("attn_split_kernelILi%dELi%dE" % (d, R), (148 * (2 if d <= 128 else 1),)), ("attn_join_kernel", (kv * NB * R // 8, 1, seqs))]
    attention(ofb, c, G, io, tmp_path, acc, path + [("attn_weight_kernel", (seqs * kv,))] * acc)


# ---- host threads --------------------------------------------------------------------

def test_threads_with_calls_of_different_sizes(ofb, cuda):
    # each raises the kernels' shared-memory limits to what its sizes need, at the same time
    def work(lens, keep):
        c = GpuCache(ofb, lens, 2, 64, 16, seed=keep)
        q = torch.randn(len(lens), 4, 64, device=cuda)
        state = [t.clone() for t in (c.k, c.v, c.weight, c.order)]

        def step():
            for t, s in zip((c.k, c.v, c.weight, c.order), state):
                t.copy_(s)
            out = ofb.attn_decode(c.handle, q, c.dlens)
            return [out, *ofb.kv_evict(c.handle, c.dlens, keep=keep, recent=10), c.k.clone(), c.order.clone()]
        return step

    works = [work([20000, 40], 700), work([9000] * 3, 800), work([300] * 400, 100), work([50] * 900 + [500], 40)]
    want = [w() for w in works]
    torch.cuda.synchronize()

    def loop(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(8):
                got = works[i]()
                torch.cuda.current_stream().synchronize()
                bits = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
                assert all(torch.equal(bits(a), bits(b)) for a, b in zip(got, want[i]))

    with ThreadPoolExecutor(len(works)) as pool:
        list(pool.map(loop, range(len(works))))

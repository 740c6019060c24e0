"""The attention cache's launches by size: calls at either side of each rule that
chooses a launch, each of which says which one it is for."""
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from attn_cache_paths import GpuCache, check_eviction, evict_path

pytestmark = pytest.mark.gpu


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

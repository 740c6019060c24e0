// evict.cu — ofb_kv_evict: a sequence's cache brought down to `keep` entries
// per kv head, those with the largest accumulated attention weight.
//
// One cluster of CTAs per (sequence, kv head), one launch. Bound by the bytes
// it must touch: 8 per entry (weight and order number), and for the kept
// entries that lie behind place `keep` their K and V rows, read and written.
// Filling the places that fall free instead of closing the ranks moves the
// fewest rows there can be, and sources (behind `keep`) and targets (before it)
// never meet, so the copies need no order among each other.
//
// 1. Each CTA takes a run of the entries and turns weights into 32-bit keys in
//    shared memory whose unsigned order is the order of eviction: NaN, then the
//    weights, then the youngest (order number above the highest - recent)
//    as all ones.
// 2. The keep-th largest key by three rounds of histograms over 11, 11 and 10
//    bits, each CTA's in its own shared memory, summed over the cluster through
//    distributed shared memory. Of the entries with just that key the first
//    `need` in place order are kept.
// 3. Warps own consecutive runs of the CTA's entries, so that ranks (of equal
//    keys where not all of them stay, of holes, of spares) come from ballots and
//    one exchange of counts.
// 4. The k-th hole and the k-th spare meet in the scratch; the warps of the
//    cluster then copy rows, 4 KB in flight per warp.
//
// A CTA's steps wait on each other, so what counts is that all CTAs run at
// once: the fewer rows, the more CTAs per cluster and threads per CTA.
#include <cooperative_groups.h>

#include "kv_cache.cuh"

namespace cg = cooperative_groups;

namespace ofb {

constexpr int EV_THREADS = 1024;  // at most
constexpr int EV_WARPS = EV_THREADS / 32;
constexpr int EV_BINS = 2048;
constexpr int EV_KEYS = 49152;  // keys a CTA holds at most: OFB_EVICT_MAX_LEN / 8
static_assert(OFB_EVICT_MAX_LEN == 8 * EV_KEYS, "eviction length limit");

struct EvictArgs {
    void *k, *v;
    float *weight;
    int32_t *order;
    const int32_t *table, *lens;
    int32_t *lens_out, *kept, *lists;
    uint32_t *errors;
    int64_t page_stride;
    FastDiv page, row2;  // by page_size; by the 16-byte chunks of a K and a V row
    int KVH, d, page_size, n_pages, max_pages, max_len, keep, recent, chunk;
    int order_kept;  // order numbers fit beside the keys (else they are read again)
};

// Unsigned order of f32: NaN lowest, -0 as 0; 0 itself is left for entries that
// are not there.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 1u;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(EV_THREADS) evict_kernel(const __grid_constant__ EvictArgs a) {
    extern __shared__ int hist[];  // [2][EV_BINS], then keys, then order numbers
    uint32_t *keys = reinterpret_cast<uint32_t *>(hist + 2 * EV_BINS);  // [chunk]
    int *orders = hist + 2 * EV_BINS + a.chunk;
    __shared__ int s_max, s_bin, s_need, s_ties;
    __shared__ int s_cnt[3][EV_WARPS];  // equal keys, holes, spares per warp
    __shared__ int s_tot[2];            // holes, spares of this CTA
    __shared__ int scan[EV_WARPS];
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nthr = blockDim.x, nwarp = nthr >> 5;
    const int u = blockIdx.x / C, b = u / a.KVH, h = u - b * a.KVH;
    auto sync_all = [&]() {
        if (C == 1) __syncthreads();
        else cl.sync();
    };
    for (int i = tid; i < 2 * EV_BINS; i += nthr) hist[i] = 0;
    if (tid == 0) s_max = INT32_MIN;
    pdl_wait();
    pdl_trigger();

    const int raw = a.lens[b], n = min(max(raw, 0), a.max_len), K = a.keep, n_out = min(n, K);
    if (rank == 0 && tid == 0) {
        if (raw > a.max_len) report(a.errors, OFB_CACHE_ELEN);
        if (h == 0) a.lens_out[b] = n_out;
    }
    int32_t *kept = a.kept ? a.kept + (int64_t)u * K : nullptr;
    if (n <= K) {  // nothing leaves (the whole cluster returns)
        if (kept)
            for (int i = rank * nthr + tid; i < K; i += C * nthr) kept[i] = i < n ? i : -1;
        return;
    }
    const int32_t *table = a.table + (int64_t)b * a.max_pages;
    // row of entry i in page p (-1: no such page) among a kv head's rows [n_pages][KVH][page_size]
    auto row_of = [&](int i, int p) -> int64_t {
        if (p < 0 || p >= a.n_pages) return -1;
        return ((int64_t)p * a.KVH + h) * a.page_size + (i - a.page.div(i) * a.page_size);
    };
    const int i0 = min(rank * a.chunk, n), i1 = min(i0 + a.chunk, n), m = i1 - i0;

    __syncthreads();
    int top = INT32_MIN;
    for (int base = tid; base < m; base += 4 * nthr) {
        int p[4], o[4];
        int64_t e[4];
        float w[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (base + k * nthr < m) p[k] = table[a.page.div(i0 + base + k * nthr)];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            e[k] = base + k * nthr < m ? row_of(i0 + base + k * nthr, p[k]) : -1;
            if (e[k] >= 0) {
                w[k] = a.weight[e[k]];
                if (a.recent) o[k] = a.order[e[k]];
            }
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = base + k * nthr;
            if (i >= m) break;
            if (e[k] < 0) report(a.errors, OFB_CACHE_EPAGE);
            keys[i] = e[k] < 0 ? 0u : weight_key(w[k]);
            if (a.recent) {
                const int v = e[k] < 0 ? INT32_MIN : o[k];
                top = max(top, v);
                if (a.order_kept) orders[i] = v;
            }
        }
    }
    int64_t above = INT64_MAX;  // wide: the difference may leave 32 bits
    if (a.recent) {
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) atomicMax(&s_max, top);
        sync_all();
        for (int r = 0; r < C; r++) top = max(top, *cl.map_shared_rank(&s_max, r));
        above = (int64_t)top - a.recent;
    }

    // the K-th largest key, by digits from the top
    uint32_t found = 0;
    int need = K;
#pragma unroll 1
    for (int round = 0; round < 3; round++) {
        const int shift = round == 0 ? 21 : round == 1 ? 10 : 0, bits = round == 2 ? 10 : 11;
        const uint32_t mask = (1u << bits) - 1, high = round == 0 ? 0u : ~0u << (shift + bits);
        int *hr = hist + (round & 1) * EV_BINS;
        for (int i = tid; i < m; i += nthr) {
            uint32_t key = keys[i];
            if (round == 0 && a.recent) {
                int v;
                if (a.order_kept) {
                    v = orders[i];
                } else {
                    const int64_t e = row_of(i0 + i, table[a.page.div(i0 + i)]);
                    v = e < 0 ? INT32_MIN : a.order[e];
                }
                // (an entry that is not there stays 0)
                if (v > above && key) keys[i] = key = 0xffffffffu;
            }
            if ((key & high) == found) atomicAdd(&hr[(key >> shift) & mask], 1);
        }
        sync_all();
        if (round == 1)  // all have read round 0's: room for round 2's
            for (int i = tid; i < EV_BINS; i += nthr) hist[i] = 0;
        // this thread's bins, counted from the top
        const int per = EV_BINS / nthr, hi = EV_BINS - 1 - tid * per;
        int c[EV_BINS / 256], s = 0;
#pragma unroll
        for (int k = 0; k < EV_BINS / 256; k++) {
            c[k] = 0;
            if (k < per)
                for (int r = 0; r < C; r++) c[k] += (C == 1 ? hr : cl.map_shared_rank(hr, r))[hi - k];
            s += c[k];
        }
        const int mine = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += v;
        }
        if (lane == 31) scan[warp] = s;
        __syncthreads();
        int before = s - mine;  // keys in the bins above
        for (int w = 0; w < warp; w++) before += scan[w];
        if (before < need && need <= before + mine) {
#pragma unroll
            for (int k = 0; k < EV_BINS / 256; k++) {
                if (k >= per) break;
                if (need <= before + c[k]) {
                    s_bin = hi - k, s_need = need - before, s_ties = c[k];
                    break;
                }
                before += c[k];
            }
        }
        __syncthreads();
        found |= (uint32_t)s_bin << shift;
        need = s_need;
        if (round < 2) __syncthreads();
    }
    // each warp's consecutive run of this CTA's entries
    const int per = ((m + nwarp - 1) / nwarp + 31) / 32 * 32;
    const int w0 = min(warp * per, m), w1 = min(w0 + per, m);
    const uint32_t lt = (1u << lane) - 1;
    const bool all_ties = s_ties == need;
    int ties_before = 0;  // equal keys before this warp's run, where not all of them stay
    if (!all_ties) {
        // the last round's bin counted exactly them
        for (int r = 0; r < rank; r++) ties_before += cl.map_shared_rank(hist, r)[found & 1023u];
        int ties = 0;
        for (int i = w0 + lane; i < w0 + per; i += 32) ties += __popc(__ballot_sync(0xffffffffu, i < w1 && keys[i] == found));
        if (lane == 0) s_cnt[0][warp] = ties;
        __syncthreads();
        for (int w = 0; w < warp; w++) ties_before += s_cnt[0][w];
    }
    int holes = 0, spares = 0;
    for (int i = w0 + lane; i < w0 + per; i += 32) {
        const uint32_t key = i < w1 ? keys[i] : 0u;
        bool stays = i < w1 && key >= found;
        if (!all_ties) {
            const bool tie = stays && key == found;
            const uint32_t tb = __ballot_sync(0xffffffffu, tie);
            if (tie && ties_before + __popc(tb & lt) >= need) stays = false;
            ties_before += __popc(tb);
        }
        const int at = i0 + i;
        const bool hole = i < w1 && at < K && !stays, spare = stays && at >= K;
        holes += __popc(__ballot_sync(0xffffffffu, hole));
        spares += __popc(__ballot_sync(0xffffffffu, spare));
        if (i < w1) {
            keys[i] = hole ? 1u : spare ? 2u : 0u;
            if (kept && at < K && stays) kept[at] = at;
        }
    }
    if (lane == 0) s_cnt[1][warp] = holes, s_cnt[2][warp] = spares;
    __syncthreads();
    if (warp == 0) {
        const int x = __reduce_add_sync(0xffffffffu, lane < nwarp ? s_cnt[1][lane] : 0);
        const int y = __reduce_add_sync(0xffffffffu, lane < nwarp ? s_cnt[2][lane] : 0);
        if (lane == 0) s_tot[0] = x, s_tot[1] = y;
    }
    sync_all();
    int hole_at = 0, spare_at = 0, moves = 0;
    for (int r = 0; r < C; r++) {
        const int *t = cl.map_shared_rank(&s_tot[0], r);
        const int x = t[0], y = t[1];
        if (r < rank) hole_at += x, spare_at += y;
        moves += x;
    }
    for (int w = 0; w < warp; w++) hole_at += s_cnt[1][w], spare_at += s_cnt[2][w];
    int32_t *hole_list = a.lists + (int64_t)u * 2 * K, *spare_list = hole_list + K;
    for (int i = w0 + lane; i < w0 + per; i += 32) {
        const uint32_t f = i < w1 ? keys[i] : 0u;
        const uint32_t hb = __ballot_sync(0xffffffffu, f == 1u), sb = __ballot_sync(0xffffffffu, f == 2u);
        if (f == 1u) hole_list[hole_at + __popc(hb & lt)] = i0 + i;
        if (f == 2u) spare_list[spare_at + __popc(sb & lt)] = i0 + i;
        hole_at += __popc(hb);
        spare_at += __popc(sb);
    }
    sync_all();  // the lists are complete and visible; no CTA's shared memory is read after this

    // rows: a warp takes `batch` moves, its lanes look them up, then copy one after another
    const int warps = C * nwarp, batch = min(32, (moves + warps - 1) / warps), row = a.d / 8;
    for (int m0 = (warp * C + rank) * batch; m0 < moves; m0 += warps * batch) {
        const int cnt = min(batch, moves - m0);
        int64_t from = -1, to = -1;
        if (lane < cnt) {
            const int hole = hole_list[m0 + lane], spare = spare_list[m0 + lane];
            const int cs = a.page.div(spare), ch = a.page.div(hole), ps = table[cs], ph = table[ch];
            const int ss = spare - cs * a.page_size, sh = hole - ch * a.page_size;
            if (kept) kept[hole] = spare;
            if (ps >= 0 && ps < a.n_pages && ph >= 0 && ph < a.n_pages) {
                const int64_t ms = ((int64_t)ps * a.KVH + h) * a.page_size + ss, mh = ((int64_t)ph * a.KVH + h) * a.page_size + sh;
                a.weight[mh] = a.weight[ms];
                a.order[mh] = a.order[ms];
                from = ps * a.page_stride + ((int64_t)h * a.page_size + ss) * a.d;
                to = ph * a.page_stride + ((int64_t)h * a.page_size + sh) * a.d;
            }
        }
        // 16-byte chunks of K and V rows, element type of 2 bytes
        const int total = cnt * 2 * row;
        for (int c0 = 0; c0 < total; c0 += 8 * 32) {
            uint4 x[8];
            char *dst[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int c = c0 + j * 32 + lane, mv = a.row2.div(c), q = c - mv * 2 * row;
                const int64_t f = __shfl_sync(0xffffffffu, from, mv & 31), t = __shfl_sync(0xffffffffu, to, mv & 31);
                dst[j] = nullptr;
                if (c < total && f >= 0) {
                    char *base = static_cast<char *>(q < row ? a.k : a.v) + (int64_t)(q < row ? q : q - row) * 16;
                    x[j] = *reinterpret_cast<const uint4 *>(base + f * 2);
                    dst[j] = base + t * 2;
                }
            }
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (dst[j]) *reinterpret_cast<uint4 *>(dst[j]) = x[j];
        }
    }
}

// CTAs per (sequence, kv head): enough that a CTA's keys fit, and more while
// the GPU has room for them and runs stay above 1024 entries.
static int evict_cluster(int rows, int max_len) {
    int c = 1;
    while (c < 8 && ((max_len + c - 1) / c > EV_KEYS || (2 * c * rows <= 2 * sm_count() && max_len / (2 * c) >= 1024))) c *= 2;
    return c;
}

// Threads per CTA: as many as leave all CTAs on the GPU at once (an SM runs
// 1024 threads of this kernel), and no more than one for two entries.
static int evict_threads(int ctas, int chunk) {
    int t = EV_THREADS;
    while (t > 256 && (ctas > sm_count() * (1024 / t) || t > chunk / 2)) t /= 2;
    return t;
}

static int check_evict(const ofb_kv_cache *c, int n_seqs, int keep) {
    int st = check_cache(c, "ofb_kv_evict");
    if (st != OFB_OK) return st;
    if (n_seqs < 0 || n_seqs > c->n_seqs || keep < 1 || keep > OFB_EVICT_MAX_LEN) {
        set_error("ofb_kv_evict: %d sequences of %d, keep %d", n_seqs, c->n_seqs, keep);
        return OFB_EINVAL;
    }
    return OFB_OK;
}

}  // namespace ofb

using namespace ofb;

extern "C" size_t ofb_kv_evict_scratch_size(const ofb_kv_cache *cache, int n_seqs, int keep) {
    if (check_evict(cache, n_seqs, keep) != OFB_OK) return 0;
    return (size_t)(n_seqs ? n_seqs : 1) * cache->n_kv_heads * 2 * keep * sizeof(int32_t);
}

extern "C" int ofb_kv_evict(const ofb_kv_cache *cache, const int32_t *lens, int n_seqs, int max_len, int keep, int recent,
                            int32_t *lens_out, int32_t *kept, void *scratch, size_t scratch_bytes, void *stream) {
    int st = check_evict(cache, n_seqs, keep);
    if (st != OFB_OK) return st;
    if (!cache->weight || !cache->order) { set_error("ofb_kv_evict: the cache has no weight or order"); return OFB_EINVAL; }
    if (recent < 0 || recent > keep || max_len < 0) {
        set_error("ofb_kv_evict: recent %d of keep %d, max_len %d", recent, keep, max_len);
        return OFB_EINVAL;
    }
    const int reach = cache_reach(cache), bound = max_len && max_len < reach ? max_len : reach;
    if (bound > OFB_EVICT_MAX_LEN) {
        set_error("ofb_kv_evict: %d entries, %d at most", bound, OFB_EVICT_MAX_LEN);
        return OFB_ETOOLARGE;
    }
    if (!n_seqs) return OFB_OK;
    if (!lens || !lens_out || misaligned(lens, 4) || misaligned(lens_out, 4) || misaligned(kept, 4) ||
        (lens_out < lens + n_seqs && lens < lens_out + n_seqs)) {
        set_error("ofb_kv_evict: lens or lens_out is NULL, misaligned, or they overlap");
        return OFB_EINVAL;
    }
    if (!scratch || misaligned(scratch, 16)) { set_error("ofb_kv_evict: scratch is NULL or not 16-byte aligned"); return OFB_EINVAL; }
    const size_t want = (size_t)n_seqs * cache->n_kv_heads * 2 * keep * sizeof(int32_t);
    if (scratch_bytes < want) { set_error("ofb_kv_evict: scratch of %zu bytes, %zu needed", scratch_bytes, want); return OFB_ETOOLARGE; }
    const int64_t rows = (int64_t)n_seqs * cache->n_kv_heads;
    if (rows > INT32_MAX / 8) { set_error("ofb_kv_evict: too many sequences"); return OFB_ETOOLARGE; }

    EvictArgs a = {};
    a.k = cache->k, a.v = cache->v, a.weight = cache->weight, a.order = cache->order, a.table = cache->page_table;
    a.lens = lens, a.lens_out = lens_out, a.kept = kept, a.lists = static_cast<int32_t *>(scratch), a.errors = cache->errors;
    a.page_stride = cache_page_stride(cache);
    a.KVH = cache->n_kv_heads, a.d = cache->head_dim, a.page_size = cache->page_size, a.n_pages = cache->n_pages;
    a.page = fast_div(a.page_size), a.max_pages = cache->max_pages, a.max_len = bound, a.keep = keep, a.recent = recent;
    const int C = evict_cluster((int)rows, bound);
    a.chunk = (bound + C - 1) / C;
    const int threads = evict_threads((int)rows * C, a.chunk);
    a.row2 = fast_div(2 * (a.d / 8));
    // order numbers stay in shared memory where that leaves room for the SM's other CTAs
    size_t smem = (size_t)(2 * EV_BINS + 2 * a.chunk) * 4;
    a.order_kept = smem <= (size_t)200 * 1024 * threads / 1024;
    if (!a.order_kept) smem = (size_t)(2 * EV_BINS + a.chunk) * 4;
    static size_t attr[64];
    // with room for the kernel's static arrays, which count against the default limit too
    cudaError_t e = ensure_dyn_smem(evict_kernel, smem + 1024, attr);
    if (e != cudaSuccess) return cuda_status(e, "ofb_kv_evict smem attribute");
    e = launch_pdl_cluster(evict_kernel, dim3((unsigned)(rows * C)), dim3(threads), C, smem, static_cast<cudaStream_t>(stream), a);
    return e == cudaSuccess ? OFB_OK : cuda_status(e, "ofb_kv_evict launch");
}

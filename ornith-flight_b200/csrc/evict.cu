// evict.cu — ofb_kv_evict: a sequence's cache brought down to `keep` entries
// per kv head, those with the largest accumulated attention weight.
//
// One cluster of CTAs per (sequence, kv head). Bound by the bytes
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
// 2. The last entry that stays, by place in the order (key down, place up): a
//    histogram of even steps between the smallest and the largest weight, each
//    CTA's in its own shared memory, summed over the cluster through distributed
//    shared memory, leaves the entries of one step. Up to EV_CAND of them are
//    ranked against each other directly (usual: a step of 4096 weights holds two
//    dozen); more take another histogram within the step, down to a single key,
//    of which the first `need` in place order stay. Weights of 0 are counted by
//    themselves: there are many, entries not attended to yet among them.
// 3. A bit per entry says whether it stays; places in the lists of holes (zeros
//    before `keep`) and spares (ones behind) come from counts of bits, a scan over
//    the CTA and one exchange over the cluster.
// 4. The k-th hole and the k-th spare meet in the scratch and rows are copied,
//    4 KB in flight per warp: by the same cluster where few rows can move, else
//    by a second launch whose CTAs take 16 or 32 moves each, since one (sequence, kv
//    head) has many more than another.
//
// A CTA's steps wait on each other, so what counts is that all CTAs run at
// once: the fewer rows, the more CTAs per cluster and threads per CTA.
#include <cooperative_groups.h>

#include "kv_cache.cuh"

namespace cg = cooperative_groups;

namespace ofb {

constexpr int EV_THREADS = 1024;  // at most
constexpr int EV_WARPS = EV_THREADS / 32;
constexpr int EV_CLUSTER = 8;   // CTAs of a cluster at most
constexpr int EV_BINS = 1024;
// moves of one CTA of the second launch: 32, or 16 where so short ones have room at
// once, EV_ROOM per SM (8 rows of 32000, 4000 moves each: 24.6 us with 32, 26.1 with
// 16, 27.1 with 64; 2 rows of 2000, 250 moves each: 11.2, 10.8 and 12.2; 512 rows of up
// to 512 moves: 40.9, 45.4 and 41.0; 24 rows of 8192: 71.4, 76.3 and 70.8)
constexpr int EV_SLICE = 32, EV_ROOM = 8;
// moves per row that may be, up to which there is no second launch: 48 with up to
// EV_FEW rows, whose clusters leave most of the GPU idle, else 128 (8 rows of 1072
// entries down to 1024 take 9.6 us without and 9.8 with it, of 4160 to 4096 14.4 and
// 13.1; 128 rows of 1152 to 1024 11.9 and 13.6)
constexpr int EV_FUSED_FEW = 48, EV_FUSED = 128, EV_FEW = 64;
// entries per CTA from which a cluster is worth its barriers: 2 rows of 8000 take
// 17.2 us with one CTA each and 20.1 with seven, of 16000 19.3 with three and 22.1
// with one
constexpr int EV_RUN = 4096;
constexpr int EV_CAND = 256;    // entries ranked directly (at most one per thread)
constexpr int EV_STATIC = 5120;  // the kernel's static arrays (4416 bytes), rounded up
constexpr int EV_KEYS = 49152;  // keys a CTA holds at most: OFB_EVICT_MAX_LEN / EV_CLUSTER
static_assert(EV_KEYS < 1 << 16, "counts of a CTA's holes and spares share a word");
static_assert(OFB_EVICT_MAX_LEN == EV_CLUSTER * EV_KEYS, "eviction length limit");

struct EvictArgs {
    void *k, *v;
    float *weight;
    int32_t *order;
    const int32_t *table, *lens;
    int32_t *lens_out, *kept, *counts;  // counts: moves per (sequence, kv head)
    int32_t *lists;                     // per (sequence, kv head): holes [keep], spares [keep]
    uint32_t *errors;
    int64_t page_stride;
    FastDiv page, row2;  // by page_size; by the 16-byte chunks of a K and a V row
    FastDiv kvh, slices; // by KVH; by the second launch's CTAs per row
    int slice;           // moves of such a CTA
    int KVH, d, page_size, n_pages, max_pages, max_len, keep, recent, chunk;
    int kept_quads;  // keep is a multiple of 4 and kept 16-byte aligned
    int fused;       // rows are copied by this launch
    int order_kept;  // order numbers fit beside the keys (else they are read again)
};

// Unsigned order of f32: NaN lowest, -0 as 0; 0 itself is left for entries that
// are not there.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 1u;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One lane's move: places from the lists, pages, rows.
struct EvictMove {
    int hole, spare, ps, ph;
    int64_t from, to;  // first elements of the rows, -1: nothing to copy
    int at;            // row of the hole among all rows [n_pages][KVH][page_size]
    float weight;
    int order;
    __device__ __forceinline__ void pages(const EvictArgs &a, int b, bool on) {
        ps = ph = -1;
        if (on) {
            const int32_t *table = a.table + (int64_t)b * a.max_pages;
            ps = table[a.page.div(spare)];
            ph = table[a.page.div(hole)];
        }
    }
    __device__ __forceinline__ void rows(const EvictArgs &a, int h) {
        from = to = -1;
        // (rows of pages that are none stay as they are)
        if (ps >= 0 && ps < a.n_pages && ph >= 0 && ph < a.n_pages) {
            const int ss = spare - a.page.div(spare) * a.page_size, sh = hole - a.page.div(hole) * a.page_size;
            const int of = (ps * a.KVH + h) * a.page_size + ss;
            at = (ph * a.KVH + h) * a.page_size + sh;
            weight = a.weight[of];
            order = a.order[of];
            from = ps * a.page_stride + ((int64_t)h * a.page_size + ss) * a.d;
            to = ph * a.page_stride + ((int64_t)h * a.page_size + sh) * a.d;
        }
    }
};

// Copies the rows of the lanes' first cnt moves, one after another, and puts
// weight, order number and `kept` in place.
__device__ __forceinline__ void evict_copy(const EvictArgs &a, int u, const EvictMove &mv, int cnt, int lane) {
    const int row = a.d / 8, total = cnt * 2 * row;  // 16-byte chunks of K and V rows, element type of 2 bytes
    for (int c0 = 0; c0 < total; c0 += 8 * 32) {
        uint4 x[8];
        char *dst[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int c = c0 + j * 32 + lane, k = a.row2.div(c), q = c - k * 2 * row;
            const int64_t f = __shfl_sync(0xffffffffu, mv.from, k & 31), t = __shfl_sync(0xffffffffu, mv.to, k & 31);
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
    if (lane < cnt) {
        if (a.kept) a.kept[(int64_t)u * a.keep + mv.hole] = mv.spare;
        if (mv.from >= 0) {
            a.weight[mv.at] = mv.weight;
            a.order[mv.at] = mv.order;
        }
    }
}

__device__ __forceinline__ uint32_t cluster_index() {  // blockIdx.x over the cluster's size
    uint32_t i;
    asm("mov.u32 %0, %%clusterid.x;" : "=r"(i));
    return i;
}

// NT threads. QUAD: four consecutive entries lie in one page, 16-byte aligned.
template <int NT, bool QUAD> __global__ void __launch_bounds__(NT, EV_THREADS / NT) evict_kernel(const __grid_constant__ EvictArgs a) {
    extern __shared__ __align__(16) int hist[];  // [2][EV_BINS], then keys, then order numbers
    uint32_t *keys = reinterpret_cast<uint32_t *>(hist + 2 * EV_BINS);  // [chunk]
    int *orders = hist + 2 * EV_BINS + a.chunk;
    __shared__ int s_max;
    __shared__ uint32_t s_low, s_high;  // keys of the smallest and the largest positive finite weight
    __shared__ int s_bin, s_need, s_ties, s_cands, s_zeros;
    __shared__ uint2 s_last;            // key and place of the last entry that stays
    __shared__ int s_cnt[EV_WARPS];     // equal keys per warp
    __shared__ uint32_t s_tot;          // holes and spares of this CTA
    __shared__ int scan[EV_WARPS];
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int nthr = NT, nwarp = NT / 32;
    const int u = (int)cluster_index(), b = a.kvh.div(u), h = u - b * a.KVH;
    // sum of x[w] over the warps before this one (x: one value per warp)
    auto warps_before = [&](const int *x) { return __reduce_add_sync(0xffffffffu, lane < warp ? x[lane] : 0); };
    auto sync_all = [&]() {
        if (C == 1) __syncthreads();
        else cl.sync();
    };
    for (int i = tid; i < 2 * EV_BINS; i += nthr) hist[i] = 0;
    if (tid == 0) s_max = INT32_MIN, s_low = 0xffffffffu, s_high = 0u, s_cands = s_zeros = 0;
    pdl_wait();
    pdl_trigger();

    // page numbers of the first entries, asked for beside the length, and then always
    // those of the next ones (2 rows of 1040 8.55 -> 8.3 us, 24 of 131072 70.9 -> 70.5)
    constexpr int V = QUAD ? 4 : 1, UN = QUAD ? 3 : 8;  // entries read together, groups in flight
    const int32_t *table = a.table + (int64_t)b * a.max_pages;
    const int start = rank * a.chunk;
    int page[UN];
    auto look_up = [&](int base, int end) {
#pragma unroll
        for (int k = 0; k < UN; k++)
            if (base + k * nthr * V < end) page[k] = table[a.page.div(start + base + k * nthr * V)];
    };
    look_up(tid * V, min(a.chunk, a.max_len - start));
    const int raw = a.lens[b], n = min(max(raw, 0), a.max_len), K = a.keep, n_out = min(n, K);
    if (rank == 0 && tid == 0) {
        if (raw > a.max_len) report(a.errors, OFB_CACHE_ELEN);
        if (h == 0) a.lens_out[b] = n_out;
    }
    int32_t *kept = a.kept ? a.kept + (int64_t)u * K : nullptr;
    if (n <= K) {  // nothing leaves (the whole cluster returns)
        if (kept)
            for (int i = rank * nthr + tid; i < K; i += C * nthr) kept[i] = i < n ? i : -1;
        if (rank == 0 && tid == 0) a.counts[u] = 0;
        return;
    }
    // row of entry i in page p (-1: no such page) among all rows [n_pages][KVH][page_size]
    auto row_of = [&](int i, int p) {
        if (p < 0 || p >= a.n_pages) return -1;
        return (p * a.KVH + h) * a.page_size + (i - a.page.div(i) * a.page_size);
    };
    const int i0 = min(start, n), i1 = min(i0 + a.chunk, n), m = i1 - i0;

    __syncthreads();
    constexpr uint32_t ZERO = 0x80000000u, INF = 0xff800000u;  // keys of 0 and of infinity
    int top = INT32_MIN;
    uint32_t low = 0xffffffffu, high = 0u;
    for (int base = tid * V; base < m; base += UN * nthr * V) {
        int e[UN], o[UN][V];
        float w[UN][V];
#pragma unroll
        for (int k = 0; k < UN; k++) {
            const int i = base + k * nthr * V;
            e[k] = i < m ? row_of(i0 + i, page[k]) : -1;
            if (e[k] < 0) continue;
            if constexpr (QUAD) {  // (what lies behind the last entry is read with it, and not used)
                *reinterpret_cast<float4 *>(w[k]) = *reinterpret_cast<const float4 *>(a.weight + e[k]);
                if (a.recent) *reinterpret_cast<int4 *>(o[k]) = *reinterpret_cast<const int4 *>(a.order + e[k]);
            } else {
                w[k][0] = a.weight[e[k]];
                if (a.recent) o[k][0] = a.order[e[k]];
            }
        }
        look_up(base + UN * nthr * V, m);
#pragma unroll
        for (int k = 0; k < UN; k++) {
            const int i = base + k * nthr * V;
            if (i >= m) break;
            if (e[k] < 0) report(a.errors, OFB_CACHE_EPAGE);
            uint32_t key[V];
            int v[V];
#pragma unroll
            for (int x = 0; x < V; x++) {  // (behind the last entry: as if not there)
                const bool there = e[k] >= 0 && (V == 1 || i + x < m);
                key[x] = there ? weight_key(w[k][x]) : 0u;
                v[x] = there && a.recent ? o[k][x] : INT32_MIN;
                if (key[x] - (ZERO + 1u) < INF - (ZERO + 1u)) low = min(low, key[x]), high = max(high, key[x]);
                top = max(top, v[x]);
            }
            if constexpr (QUAD) {
                *reinterpret_cast<uint4 *>(keys + i) = make_uint4(key[0], key[1], key[2], key[3]);
                if (a.order_kept) *reinterpret_cast<int4 *>(orders + i) = make_int4(v[0], v[1], v[2], v[3]);
            } else {
                keys[i] = key[0];
                if (a.order_kept) orders[i] = v[0];
            }
        }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    if (lane == 0) atomicMax(&s_max, top), atomicMin(&s_low, low), atomicMax(&s_high, high);
    sync_all();
#pragma unroll
    for (int r = 0; r < EV_CLUSTER; r++)
        if (r < C) {
            top = max(top, *cl.map_shared_rank(&s_max, r));
            low = min(low, *cl.map_shared_rank(&s_low, r));
            high = max(high, *cl.map_shared_rank(&s_high, r));
        }
    if (low > high) low = high = ZERO + 1u;
    // above this order number an entry is protected (wide: the difference may leave 32 bits)
    const int64_t above = a.recent ? (int64_t)top - a.recent : INT64_MAX;

    if (a.recent && !a.order_kept) {
        constexpr int UO = QUAD ? 6 : 8;
        for (int base = tid * V; base < m; base += UO * nthr * V) {
            int e[UO], o[UO][V];
#pragma unroll
            for (int k = 0; k < UO; k++) {
                const int i = base + k * nthr * V;
                e[k] = i < m ? row_of(i0 + i, table[a.page.div(i0 + i)]) : -1;
                if (e[k] < 0) continue;
                if constexpr (QUAD) *reinterpret_cast<int4 *>(o[k]) = *reinterpret_cast<const int4 *>(a.order + e[k]);
                else o[k][0] = a.order[e[k]];
            }
#pragma unroll
            for (int k = 0; k < UO; k++)
#pragma unroll
                for (int x = 0; x < V; x++) {
                    const int i = base + k * nthr * V + x;
                    if (i < m && e[k] >= 0 && o[k][x] > above) keys[i] = 0xffffffffu;
                }
        }
        __syncthreads();
    }

    // [key_lo, key_hi] holds the key of the last entry that stays, the need-th
    // from the top of those within
    uint32_t key_lo = 0u, key_hi = 0xffffffffu;
    int need = K;
    bool ranked = false;    // s_last is found
    bool tie_break = false; // all of [key_lo, key_hi] = one key: its first `need` stay
#pragma unroll 1
    for (int round = 0;; round++) {
        // even steps: in the first round from the smallest to the largest weight,
        // bin 0 for all below (0 among them); then over the interval
        const uint32_t base = round ? key_lo : low, width = (round ? key_hi : high) - base, off = round ? 0u : 1u;
        const int shift = max(0, 32 - __clz(width) - 10);
        int *hr = hist + (round & 1) * EV_BINS;
        int zeros = 0;
        for (int i = 4 * tid; i < m; i += 4 * nthr) {
            uint4 q = *reinterpret_cast<const uint4 *>(keys + i);
            uint32_t key[4] = {q.x, q.y, q.z, q.w};
            if (round == 0 && a.order_kept) {  // (an entry that is not there stays 0)
                const int4 o = *reinterpret_cast<const int4 *>(orders + i);
                const int v[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                for (int x = 0; x < 4; x++)
                    if (v[x] > above && key[x]) key[x] = 0xffffffffu;
                *reinterpret_cast<uint4 *>(keys + i) = make_uint4(key[0], key[1], key[2], key[3]);
            }
#pragma unroll
            for (int x = 0; x < 4; x++) {
                if (i + x >= m || key[x] - key_lo > key_hi - key_lo) continue;
                if (round == 0 && key[x] == ZERO) zeros++;
                else atomicAdd(&hr[key[x] < base ? 0u : min(((key[x] - base) >> shift) + off, EV_BINS - 1u)], 1);
            }
        }
        if (round == 0) {
            zeros = __reduce_add_sync(0xffffffffu, zeros);
            if (lane == 0 && zeros) atomicAdd(&s_zeros, zeros), atomicAdd(&hr[0], zeros);
        }
        sync_all();
        if (round)  // all have read the round before: room for the next
            for (int i = tid; i < EV_BINS; i += nthr) hist[((round & 1) ^ 1) * EV_BINS + i] = 0;
        // this thread's bins, counted from the top
        constexpr int per = EV_BINS / NT;
        const int hi = EV_BINS - (tid + 1) * per;
        int c[per], s = 0;
#pragma unroll
        for (int k = 0; k < per; k++) c[k] = 0;
        if (C == 1) {
#pragma unroll
            for (int k = 0; k < per; k++) c[k] = hr[hi + k];
        } else {
#pragma unroll
            for (int r = 0; r < EV_CLUSTER; r++)
                if (r < C) {
                    const int *x = cl.map_shared_rank(hr, r) + hi;
#pragma unroll
                    for (int k = 0; k < per; k++) c[k] += x[k];
                }
        }
#pragma unroll
        for (int k = 0; k < per; k++) s += c[k];
        const int mine = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += v;
        }
        if (lane == 31) scan[warp] = s;
        __syncthreads();
        int before = s - mine + warps_before(scan);  // entries in the bins above
        if (before < need && need <= before + mine) {
#pragma unroll
            for (int k = per - 1; k >= 0; k--) {
                if (need <= before + c[k]) {
                    s_bin = hi + k, s_need = need - before, s_ties = c[k];
                    break;
                }
                before += c[k];
            }
        }
        __syncthreads();
        const uint32_t bin = (uint32_t)s_bin;
        int count = s_ties;
        need = s_need;
        // the bin's keys (the outer bins of the first round hold what lies outside, too)
        const uint32_t b_lo = base + ((bin - off) << shift), span = (1u << shift) - 1u;
        if (bin < off) {
            key_hi = low - 1u;
        } else {
            key_lo = b_lo;
            if (bin < EV_BINS - 1u && key_hi - b_lo > span) key_hi = b_lo + span;
        }
        if (bin < off) {  // the zeros come first of these
            int n0 = 0;
            for (int r = 0; r < C; r++) n0 += *cl.map_shared_rank(&s_zeros, r);
            if (need <= n0) {
                key_lo = key_hi = ZERO;
                tie_break = need < n0;
                break;
            }
            need -= n0, count -= n0;
            key_hi = ZERO - 1u;
        }
        if (count == need) break;  // all of them stay
        if (count <= EV_CAND) {
            ranked = true;
            break;
        }
        if (key_lo == key_hi) {
            tie_break = true;
            break;
        }
        __syncthreads();  // s_bin is written again
    }
    if (ranked) {
        // (key, place) of every candidate of the cluster, ranked by each CTA
        __shared__ __align__(16) uint2 cand[EV_CAND], all[EV_CAND + 1];
        for (int i = 4 * tid; i < m; i += 4 * nthr) {
            const uint4 q = *reinterpret_cast<const uint4 *>(keys + i);
            const uint32_t key[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int x = 0; x < 4; x++)
                if (i + x < m && key[x] - key_lo <= key_hi - key_lo)
                    cand[atomicAdd(&s_cands, 1)] = make_uint2(key[x], (uint32_t)(i0 + i + x));
        }
        sync_all();
        int n_all = 0, from = -1, nth = 0;  // thread i brings candidate i of the cluster's row of them
#pragma unroll
        for (int r = 0; r < EV_CLUSTER; r++)
            if (r < C) {
                const int cnt = *cl.map_shared_rank(&s_cands, r);
                if (tid >= n_all && tid < n_all + cnt) from = r, nth = tid - n_all;
                n_all += cnt;
            }
        if (from >= 0) all[tid] = cl.map_shared_rank(cand, from)[nth];
        if (tid == 0) all[n_all] = make_uint2(0u, 0xffffffffu);  // ranks behind all
        __syncthreads();
        // each CTA ranks its own, `team` lanes to a candidate
        const int own = s_cands;
        int shift = 0;
        while (shift < 5 && (2 * own << shift) <= nthr) shift++;
        const int team = 1 << shift, c = tid >> shift, part = tid & (team - 1);
        const uint2 x = c < own ? cand[c] : make_uint2(0u, 0u);
        int r = 0;
        if (c < own) {
#pragma unroll 4
            for (int j = 2 * part; j < n_all; j += 2 * team) {
                const uint4 y = *reinterpret_cast<const uint4 *>(all + j);  // two at a time
                r += y.x > x.x || (y.x == x.x && y.y < x.y);
                r += y.z > x.x || (y.z == x.x && y.w < x.y);
            }
        }
        for (int o = 1; o < team; o <<= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
        if (c < own && part == 0 && r == need - 1)
            for (int q = 0; q < C; q++) *cl.map_shared_rank(&s_last, q) = x;
        sync_all();
    }
    // an entry stays whose key is above last.x, or equal with a place up to last.y
    const uint2 last = ranked ? s_last : make_uint2(tie_break ? max(key_lo, 1u) : key_lo, 0xffffffffu);

    if (tie_break) {  // of equal keys the first `need` stay: each warp ranks those of a consecutive run
        const int per = ((m + nwarp - 1) / nwarp + 31) / 32 * 32, w0 = min(warp * per, m), w1 = min(w0 + per, m);
        const uint32_t lt = (1u << lane) - 1;
        int ties_before = 0;
        int ties = 0;
        for (int i = w0 + lane; i < w1; i += 32) ties += keys[i] == key_lo;
        ties = __reduce_add_sync(0xffffffffu, ties);
        if (lane == 0) s_cnt[warp] = ties;
        __syncthreads();
        if (tid == 0) {
            int x = 0;
            for (int w = 0; w < nwarp; w++) x += s_cnt[w];
            s_ties = x;
        }
        sync_all();
        for (int r = 0; r < rank; r++) ties_before += *cl.map_shared_rank(&s_ties, r);
        ties_before += warps_before(s_cnt);
        // from here on an equal key that stays is above all, one that leaves below
        for (int base = w0; base < w1; base += 32) {
            const int i = base + lane;
            const bool tie = i < w1 && keys[i] == key_lo;
            const uint32_t tb = __ballot_sync(0xffffffffu, tie);
            if (tie) keys[i] = ties_before + __popc(tb & lt) < need ? 0xffffffffu : 0u;
            ties_before += __popc(tb);
        }
        __syncthreads();
    }
    if (kept) {  // each comes from its own place; the moves' are written over
        const int k1 = min(K - i0, m);
        if (a.kept_quads) {
            for (int i = 4 * tid; i < k1; i += 4 * nthr)
                *reinterpret_cast<int4 *>(kept + i0 + i) = make_int4(i0 + i, i0 + i + 1, i0 + i + 2, i0 + i + 3);
        } else {
            for (int i = tid; i < k1; i += nthr) kept[i0 + i] = i0 + i;
        }
    }
    // a bit per entry that stays, 32 of them in the place of one of their keys
    // (word w in that of entry 33 w at most, so that threads read from all banks)
    const int words = (m + 31) / 32;
    auto word_at = [&](int w) -> uint32_t & { return keys[min(32 * w + (w & 31), m - 1)]; };
    for (int w = warp; w < words; w += nwarp) {
        const int i = 32 * w + lane;
        const uint32_t key = i < m ? keys[i] : 0u;
        const bool stays = i < m && (key > last.x || (key == last.x && (uint32_t)(i0 + i) <= last.y));
        const uint32_t bits = __ballot_sync(0xffffffffu, stays);
        if (lane == 0) word_at(w) = bits;
    }
    __syncthreads();
    // holes are the zeros below K, spares the ones from K on
    auto holes_spares = [&](int w, uint32_t &hole, uint32_t &spare) {
        const uint32_t bits = word_at(w);
        const int below = K - (i0 + 32 * w), there = m - 32 * w;
        const uint32_t head = below >= 32 ? ~0u : below <= 0 ? 0u : (1u << below) - 1u;
        hole = ~bits & head & (there >= 32 ? ~0u : (1u << there) - 1u);
        spare = bits & ~head;
    };
    // threads take consecutive words; counts of holes in the low half (a CTA has
    // less than 2^16 entries), of spares in the high half
    const int per_t = (words + nthr - 1) / nthr, wa = min(tid * per_t, words), wb = min(wa + per_t, words);
    uint32_t n2 = 0;
    for (int w = wa; w < wb; w++) {
        uint32_t hole, spare;
        holes_spares(w, hole, spare);
        n2 += __popc(hole) + (__popc(spare) << 16);
    }
    uint32_t s2 = n2;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, s2, o);
        if (lane >= o) s2 += v;
    }
    if (lane == 31) scan[warp] = (int)s2;
    __syncthreads();
    const uint32_t before2 = s2 - n2 + (uint32_t)warps_before(scan);
    if (tid == NT - 1) s_tot = before2 + n2;
    sync_all();
    int moves = 0, hole_at = (int)(before2 & 0xffffu), spare_at = (int)(before2 >> 16);  // as many holes as spares
#pragma unroll
    for (int r = 0; r < EV_CLUSTER; r++)
        if (r < C) {
            const uint32_t x = *cl.map_shared_rank(&s_tot, r);
            moves += (int)(x & 0xffffu);
            if (r < rank) hole_at += (int)(x & 0xffffu), spare_at += (int)(x >> 16);
        }
    int32_t *hole_list = a.lists + (int64_t)u * 2 * K, *spare_list = hole_list + K;
    int32_t *hole_out = hole_list + hole_at, *spare_out = spare_list + spare_at;
    for (int w = wa; w < wb; w++) {
        uint32_t hole, spare;
        holes_spares(w, hole, spare);
        for (; hole; hole &= hole - 1u) *hole_out++ = i0 + 32 * w + __ffs(hole) - 1;
        for (; spare; spare &= spare - 1u) *spare_out++ = i0 + 32 * w + __ffs(spare) - 1;
    }
    sync_all();  // the lists are complete and visible; no CTA's shared memory is read after this

    if (rank == 0 && tid == 0) a.counts[u] = moves;
    if (a.fused) {
        const int warps = C * nwarp, batch = min(32, (moves + warps - 1) / warps);
        for (int m0 = (warp * C + rank) * batch; m0 < moves; m0 += warps * batch) {
            const int k = min(m0 + lane, moves - 1), cnt = min(batch, moves - m0);
            EvictMove mv;
            mv.hole = hole_list[k], mv.spare = spare_list[k];
            mv.pages(a, b, lane < cnt);
            mv.rows(a, h);
            evict_copy(a, u, mv, cnt, lane);
        }
    }
}

// The second launch: CTA (row, s) makes moves slice * s and on.
// (Warps that go round over slices, looking the next ones up while they copy,
// took 10 to 15% longer: what counts is rows under way at once.)
constexpr int EV_MOVE_THREADS = 128;
__global__ void __launch_bounds__(EV_MOVE_THREADS) evict_move_kernel(const __grid_constant__ EvictArgs a) {
    const int u = a.slices.div(blockIdx.x), s = (int)(blockIdx.x - u * a.slices.d), lane = threadIdx.x & 31, b = a.kvh.div(u);
    const int each = a.slice / (EV_MOVE_THREADS / 32);
    const int m0 = s * a.slice + (threadIdx.x >> 5) * each, k = min(m0 + lane, a.keep - 1);
    pdl_wait();
    pdl_trigger();
    // the lists are asked for beside the count: places behind the last move are not used
    const int32_t *list = a.lists + (int64_t)u * 2 * a.keep;
    const int moves = a.counts[u];
    EvictMove mv;
    mv.hole = list[k], mv.spare = list[a.keep + k];
    if (m0 >= moves) return;
    const int cnt = min(each, moves - m0);
    mv.pages(a, b, lane < cnt);
    mv.rows(a, u - b * a.KVH);
    evict_copy(a, u, mv, cnt, lane);
}

// CTAs per (sequence, kv head) and threads per CTA: what brings the most threads
// onto the GPU with all CTAs there at once (an SM runs 1024 threads of this
// kernel), as long as a CTA has EV_RUN entries and a thread two; fewer, larger
// CTAs where that is nearly the same.
static void evict_shape(int rows, int max_len, int &ctas, int &threads) {
    ctas = 0;
    int64_t best = 0;
    for (int t = EV_THREADS; t >= 256; t /= 2) {
        if (t > 256 && t > max_len / 2) continue;
        const int per_sm = EV_THREADS / t, slots = sm_count() * per_sm;
        // a cluster lies within one of the GPU's eight groups of 16 SMs or more
        int c = slots / rows;
        while (c > 1 && 8 * (16 * per_sm / c) < rows) c--;
        if (c > max_len / EV_RUN) c = max_len / EV_RUN;
        c = c < 1 ? 1 : c > EV_CLUSTER ? EV_CLUSTER : c;
        while (c < EV_CLUSTER && (max_len + c - 1) / c > EV_KEYS) c++;
        const int64_t n = rows > slots ? 0 : (int64_t)rows * c * t;
        if (!ctas || n > best + best / 8) ctas = c, threads = t, best = n;
    }
    // more rows than fit at once: small CTAs, so that the last ones to run are short
    if (!best) threads = 256;
}

static size_t evict_scratch(int n_seqs, int kvh, int keep) {
    return (size_t)n_seqs * kvh * (2 * (size_t)keep + 1) * sizeof(int32_t);
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
    return evict_scratch(n_seqs ? n_seqs : 1, cache->n_kv_heads, keep);
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
    const size_t want = evict_scratch(n_seqs, cache->n_kv_heads, keep);
    if (scratch_bytes < want) { set_error("ofb_kv_evict: scratch of %zu bytes, %zu needed", scratch_bytes, want); return OFB_ETOOLARGE; }
    if ((int64_t)cache->n_pages * cache->n_kv_heads * cache->page_size > INT32_MAX) {
        set_error("ofb_kv_evict: the cache has more than 2^31 rows");
        return OFB_ETOOLARGE;
    }
    const int64_t rows = (int64_t)n_seqs * cache->n_kv_heads;
    if (rows > INT32_MAX / 8) { set_error("ofb_kv_evict: too many sequences"); return OFB_ETOOLARGE; }

    EvictArgs a = {};
    a.k = cache->k, a.v = cache->v, a.weight = cache->weight, a.order = cache->order, a.table = cache->page_table;
    a.lens = lens, a.lens_out = lens_out, a.kept = kept, a.errors = cache->errors;
    a.page_stride = cache_page_stride(cache);
    a.KVH = cache->n_kv_heads, a.d = cache->head_dim, a.page_size = cache->page_size, a.n_pages = cache->n_pages;
    a.page = fast_div(a.page_size), a.max_pages = cache->max_pages, a.max_len = bound, a.keep = keep, a.recent = recent;
    a.lists = static_cast<int32_t *>(scratch);
    a.counts = a.lists + rows * 2 * keep;
    const int most = bound <= keep ? 0 : bound - keep < keep ? bound - keep : keep;  // moves of a row
    a.kept_quads = keep % 4 == 0 && !misaligned(kept, 16);
    a.fused = most <= (rows <= EV_FEW ? EV_FUSED_FEW : EV_FUSED);
    a.slice = rows * ((most + EV_SLICE / 2 - 1) / (EV_SLICE / 2)) <= EV_ROOM * sm_count() ? EV_SLICE / 2 : EV_SLICE;
    const int slices = (most + a.slice - 1) / a.slice;
    a.slices = fast_div(slices > 1 ? slices : 1), a.kvh = fast_div(a.KVH);
    if (!a.fused && rows * slices > INT32_MAX) { set_error("ofb_kv_evict: too many moves"); return OFB_ETOOLARGE; }
    int C, threads = 256;
    evict_shape((int)rows, bound, C, threads);
    a.chunk = ((bound + C - 1) / C + 3) / 4 * 4;  // runs of the CTAs start at a multiple of 4
    a.row2 = fast_div(2 * (a.d / 8));
    // order numbers stay in shared memory where that leaves room for the SM's other CTAs (one
    // CTA of 1024 threads: 227328 bytes and the static arrays, the 227 KB that a CTA can have)
    size_t smem = (size_t)(2 * EV_BINS + 2 * a.chunk) * 4;
    a.order_kept = recent > 0 && (smem + EV_STATIC + 1024) * (1024 / threads) <= 228 * 1024;
    if (!a.order_kept) smem = (size_t)(2 * EV_BINS + a.chunk) * 4;
    const bool quad = a.page_size % 4 == 0 && !misaligned(a.weight, 16) && !misaligned(a.order, 16);
    const int vi = (threads == 256 ? 0 : threads == 512 ? 1 : 2) * 2 + quad;
    const auto kernel = vi == 0   ? evict_kernel<256, false>
                        : vi == 1 ? evict_kernel<256, true>
                        : vi == 2 ? evict_kernel<512, false>
                        : vi == 3 ? evict_kernel<512, true>
                        : vi == 4 ? evict_kernel<1024, false>
                                  : evict_kernel<1024, true>;
    static size_t attr[6][64];
    cudaError_t e = ensure_dyn_smem(kernel, smem, attr[vi], EV_STATIC);
    if (e != cudaSuccess) return cuda_status(e, "ofb_kv_evict smem attribute");
    e = launch_pdl_cluster(kernel, dim3((unsigned)(rows * C)), dim3(threads), C, smem, static_cast<cudaStream_t>(stream), a);
    if (e == cudaSuccess && !a.fused)
        e = launch_pdl(evict_move_kernel, dim3((unsigned)(rows * slices)), dim3(EV_MOVE_THREADS), 0, static_cast<cudaStream_t>(stream), a);
    return e == cudaSuccess ? OFB_OK : cuda_status(e, "ofb_kv_evict launch");
}

// attn.cuh — attention of one new token over the paged cache: the split
// kernel (attn_d*.cu hold its instances, attn.cu the join and the entry point).
//
//   z_n = scale * q.k_n,  p_n = exp(z_n - m) / l,  out = sum_n p_n v_n
//
// HBM-bound: 4 * head_dim bytes per cached entry and kv head against
// 4 * head_dim operations per query head.
//
// Work: the entries of each (sequence, kv head) are cut into tiles of 32, and
// the tiles of all of them, laid end to end, are dealt to the CTAs in equal runs,
// whatever the lengths. A run holds parts of one or more (sequence, kv head)s; a
// part that is not whole goes to the scratch (sums, maximum, sum of exponentials)
// and attn.cu joins it with the others. (Runs of three quarters and the rest
// taken in smaller ones by CTAs that finish early gained 4% on 48 ragged
// sequences with head_dim 128 and lost 3% on 24 with 256: not kept.)
//
// Inside a CTA the warps take the tiles of a part in turn, each by itself: its own
// ring of tiles in shared memory filled by 16-byte asynchronous copies (page
// by page, a tile or two ahead and across parts, the page numbers one tile
// before that), its own running maximum and sums, no barrier but one merge at
// the end of a part. The 6 to 8 warps that an SM's shared memory has room for
// leave latencies open, so a tile is 32 entries: its four chains of products, and
// one softmax step for all, keep a warp busier than two tiles of 16 would (24
// sequences of head_dim 256: 193 -> 184 us). Rows are padded by 16 bytes, so that
// ldmatrix meets no bank twice.
//
// Short sequences take a cluster of CTAs each instead of runs (CLUSTER): its
// CTAs share the tiles of one (sequence, kv head) and join their sums through
// distributed shared memory, which saves the second launch.
//
// Measured: 24 sequences of 8 to 40 thousand entries, 2 kv heads of 256, fp16
// (1.11 GB): 180 to 190 us, 5.8 to 6.1 TB/s; a plain sum over as many bytes takes 183.
// The copies alone, without the products, take 178.
//
// The products run on mma.sync m16n8k16 (bf16 or fp16, f32 sums): 16 rows of A
// by 8 entries or 8 output columns. Neither an f32 query nor a probability is
// rounded to the cache's type; both go in as parts of that type:
//   query: in the cache's type one part, exact. f32: bf16 hi + mid + low (24
//     bits) or fp16 hi + low (22 bits) of q scaled by a power of two into fp16's
//     range.
//   probability: bf16 hi + low (16 bits) or, for f32 output, + lowest (24 bits);
//     fp16 hi + low of 2^14 p (22 bits).
// Up to 8 query heads of a kv head fill 8 rows; the other 8 rows take the next
// part of the same numbers, so that two parts cost one product. 9 to 16 heads
// (R = 16) fill all rows, with a product per part; more take several passes, a part
// of the work each, which read K and V again: ceil(G / 16), or ceil(G / 8) with f32
// heads of 192 or 256, of which 16 have more queries and sums than one warp's registers
// hold. 24 sequences of 8 to 40 thousand entries in bf16: 2 x 8 f32 heads of 256 203 us,
// 2 x 16 417; 1 x 16 bf16 heads of 128 60 us, 1 x 128 324. (Warps of a CTA that share
// tiles and take a pass each have not been tried.)
// A number's parts end in the same thread, which adds them in f32. With f32 output
// each tile's product starts at zero and is added to the running sum by an FFMA,
// since the tensor core's own accumulation cuts off where an addition rounds; with
// 16-bit output, whose own rounding is coarser than that by far, the tensor core
// accumulates up to head_dim 128.
#pragma once
#include <cooperative_groups.h>

#include <type_traits>

#include "async.cuh"
#include "kv_cache.cuh"

namespace cg = cooperative_groups;

namespace ofb {

constexpr int ATT_TILE = 32;  // entries per tile, one per lane
constexpr int ATT_MAX_SEQS = OFB_ATTN_MAX_SEQS;
constexpr int ATT_MAX_CTAS = 2;  // per SM, of any instance

struct AttnArgs {
    const void *k, *v, *q;
    void *out;
    const int32_t *table, *lens;
    int64_t page_stride, q_stride, out_stride;
    int B, KVH, G, NB, H;  // NB: passes of at most R heads per kv head
    FastDiv page;  // by page_size
    int page_size, max_pages, n_pages, max_len;
    int halves;       // page_size is a multiple of 16: each half of a tile lies in one page
    int quads;        // page_size is a multiple of 4 and weight 16-byte aligned
    float scale;      // times log2(e)
    uint32_t *errors;
    // scratch
    int *prefix;      // [B + 1] places before each sequence, per pass
    float2 *ml;       // [B][H] maximum (log2) and sum
    float *part_o;    // [2 * CTAs][R][d]
    float2 *part_ml;  // [2 * CTAs][R]
    float *z;         // [B][H][z_stride] scores in log2, or NULL
    int64_t z_stride;
    float *weight;
    FastDiv ctas;     // by the number of runs
};

__device__ __forceinline__ float exp2_fast(float x) {  // 2 steps at most; below 2^-126 it gives 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// How many entries of sequence b are attended to.
__device__ __forceinline__ int attn_len(const AttnArgs &a, int b) { return min(max(a.lens[b], 0), a.max_len); }
// The row of all places: each (sequence, pass) with entries has ATT_PART places
// that stand for the time a part costs besides its tiles (queries, the warps'
// merge), then one per tile. It is cut into runs, one per CTA: at least a tile
// per warp, so that few tiles do not leave many parts to join.
// (8: 48 ragged sequences with weights 194 us without such places, 186 with 4, 182
// with 8, 183 with 16.)
constexpr int ATT_PART = 8;
struct AttnSplit {
    int total, run;
    static __device__ __forceinline__ AttnSplit make(int total, const FastDiv &ctas, int warps) {
        return {total, max(ctas.div(total + (int)ctas.d - 1), warps)};
    }
    __device__ __forceinline__ int first(int id) const { return (int)min((int64_t)id * run, (int64_t)total); }
};

// How the queries of an instance go in (see the top): parts, fragments of A, and
// whether the fragments are in shared memory, one copy for all warps, instead of
// each warp's registers. That is where registers cannot hold them beside the
// sums: 8 heads of 256, f32, bf16 cache (24 sequences of 8 to 40 thousand entries
// 268 -> 209 us).
template <int D, int R, typename CT, typename IO> struct AttnQuery {
    static constexpr bool F32 = sizeof(IO) == 4, BF = std::is_same<CT, __nv_bfloat16>::value;
    static constexpr int NQ = F32 ? (BF ? 3 : 2) : 1;
    static constexpr int QF = R == 8 ? (NQ + 1) / 2 : NQ;
    static constexpr bool QS = F32 && BF && R == 8 && D == 256;
    static constexpr int QB = QS ? D / 16 * 32 * 24 : 0;  // bytes
};
template <int D, int QB> struct AttnShape {
    static constexpr int PITCH = D * 2 + 16;                 // bytes of a row in shared memory
    static constexpr int TILE_BYTES = 2 * ATT_TILE * PITCH;  // K, then V
    static constexpr int W = D == 128 || D == 256 ? 3 : 4;   // warps per CTA
    static constexpr int S = D <= 64 ? 3 : 2;                // ring slots
    static constexpr int CTAS = D <= 128 ? 2 : 1;            // per SM
    static constexpr int THREADS = W * 32;
    // behind the rings: the warps' and the cluster's (maximum, sum), the queries'
    // fragments, then per sequence the places before it and the entries of its last
    // tile
    static __host__ __device__ constexpr int ring(int w) { return w * S * TILE_BYTES; }
    static __host__ __device__ constexpr int head(int w) { return ring(w) + (W + 1) * 16 * 8 + QB; }
    // (head_dim 64: beside more than 869 sequences' an SM has room for one CTA, not two; 1400
    // sequences of 100 to 300 entries, 2 kv heads: 103 us, 860 43)
    static constexpr int smem(int B) { return head(W) + (B + 1) * 4 + (B + 3) / 4 * 4; }
    static_assert(CTAS <= ATT_MAX_CTAS, "parts in the scratch");
    static_assert(TILE_BYTES >= 16 * (D + 4) * 4, "a warp's sums must fit one ring slot");
    static_assert(CTAS * (smem(384) + 2048) <= 228 * 1024, "shared memory of an SM");
    static_assert(smem(ATT_MAX_SEQS) + 1024 <= 227 * 1024, "shared memory of a CTA");
};

template <typename T> struct Mma;
template <> struct Mma<__nv_bfloat16> {
    static __device__ __forceinline__ void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <> struct Mma<__half> {
    static __device__ __forceinline__ void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// 16 bytes, or 16 zero bytes when `bytes` is 0 (the source is then not read). K and
// V are read once: the policy lets L2 give them up before the scores and the parts (48
// ragged sequences with weights 180 -> 177 us, one of 131071 entries 34.1 -> 33.1). It
// is formed here, by one instruction that the compiler may merge or repeat: kept in
// registers throughout it cost 8 f32 heads of 256 in a bf16 cache 8%.
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, int bytes) {
    uint64_t pol;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(pol));
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes), "l"(pol)
                 : "memory");
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float x, float y);  // x in the low half
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t p);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t p) {
    return make_float2(__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t p) {
    __half2 h;
    memcpy(&h, &p, 4);
    return __half22float2(h);
}
// Splits (x, y) into parts of T: p[i] holds part i of x (low half) and y.
template <typename T, int N> __device__ __forceinline__ void split2(float x, float y, uint32_t (&p)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        p[i] = pack2<T>(x, y);
        if (i + 1 < N) {
            const float2 f = unpack2<T>(p[i]);
            x -= f.x, y -= f.y;
        }
    }
}

// A part: tiles [t, end) of (sequence b, pass vh), of nt tiles that hold len
// entries; f_end: the place behind it in the row of all places.
struct AttnPart {
    int b, vh, t, end, nt, len, f_end;
};
// The part that begins at place f, cut at f1 (it may then be without tiles).
__device__ __forceinline__ AttnPart attn_part(const int *prefix, const uint8_t *last, int B, int nvh, int f, int f1) {
    int lo = 0, hi = B - 1;  // the last sequence that begins at or before f (and has places)
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (prefix[mid] * nvh <= f) lo = mid;
        else hi = mid - 1;
    }
    AttnPart p;
    const int places = prefix[lo + 1] - prefix[lo], r = f - prefix[lo] * nvh;
    p.b = lo;
    p.nt = places - ATT_PART;
    p.len = (p.nt - 1) * ATT_TILE + last[lo];
    p.vh = r / places;
    const int off = r - p.vh * places, n = min(f1 - f, places - off);
    p.t = max(off - ATT_PART, 0);
    p.end = max(off + n - ATT_PART, 0);
    p.f_end = f + n;
    return p;
}

template <int D, int R, typename CT, typename IO, bool CLUSTER>
__global__ void __launch_bounds__(AttnShape<D, AttnQuery<D, R, CT, IO>::QB>::THREADS,
                                  AttnShape<D, AttnQuery<D, R, CT, IO>::QB>::CTAS) attn_split_kernel(const __grid_constant__ AttnArgs a) {
    using Q = AttnQuery<D, R, CT, IO>;
    using SH = AttnShape<D, Q::QB>;
    constexpr bool F32 = Q::F32, BF = Q::BF, QS = Q::QS;
    constexpr int NQ = Q::NQ, QF = Q::QF;            // parts of a query; fragments
    constexpr int NP = BF && F32 ? 3 : 2;            // parts of a probability
    constexpr float PSCALE = BF ? 1.0f : 16384.0f;   // fp16 holds 2^14 p
    constexpr int NR = R / 8;                        // query heads of a thread: g, g + 8
    constexpr int PF = R == 8 ? (NP + 1) / 2 : NP;   // fragments: two parts of 8 heads, or a part of 16
    constexpr bool DIRECT = !F32 && D <= 128;        // the tensor core accumulates (registers allow no more)
    constexpr int NO = DIRECT || R == 16 ? 4 : 2;    // accumulators of 8 columns
    constexpr int KS = D / 16, CH = D / 8;           // k steps; 16-byte chunks of a row
    // CLUSTER: fewer warps where there are fewer tiles
    const int W = CLUSTER ? (int)blockDim.x >> 5 : SH::W, THREADS = W * 32;
    // the next part's queries are asked for while registers hold them beside the sums
    constexpr bool AHEAD = NR * D * sizeof(IO) <= 512;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c2 = (lane & 3) * 2;
    uint8_t *ring = smem + warp * SH::S * SH::TILE_BYTES;
    float2 *mml = reinterpret_cast<float2 *>(smem + SH::ring(W));  // [W][R]
    float2 *cml = mml + SH::W * R;                          // [R]: the cluster's
    int *prefix = reinterpret_cast<int *>(smem + SH::head(W));  // [B + 1]
    uint8_t *last = reinterpret_cast<uint8_t *>(prefix + a.B + 1);
    // fragments: [KS][32] of four registers, then [KS][32] of the two of the second
    // fragment that are not zero
    uint4 *const q4 = reinterpret_cast<uint4 *>(smem + SH::ring(W) + (SH::W + 1) * 16 * 8);
    uint2 *const q2 = reinterpret_cast<uint2 *>(q4 + KS * 32);
    __shared__ uint32_t valid[SH::W][4];  // per ring slot: which of the 32 entries are there
    __shared__ int wsum[SH::W];
    __shared__ float *mo[SH::W];  // each warp's sums at the end of a part, [R][D + 4]
    __shared__ float2 all_ml[8][R];  // CLUSTER: every CTA's (maximum, sum) ...
    __shared__ int all_at[8];            // ... and where its sums are in its shared memory
    cg::cluster_group cl = cg::this_cluster();
    const int C = CLUSTER ? (int)cl.num_blocks() : 1, rank = CLUSTER ? (int)cl.block_rank() : 0;

    pdl_wait();
    pdl_trigger();

    const int nvh = a.KVH * a.NB;
    int f0 = 0, f1 = 1;
    AttnPart first;
    if constexpr (CLUSTER) {
        if (C > 1) cl.barrier_arrive();  // waited for before the others' shared memory is written
        const int u = blockIdx.x / C;
        first.b = u / nvh;
        first.vh = u - first.b * nvh;
        if (a.lens[first.b] > a.max_len && first.vh == 0 && rank == 0 && tid == 0) report(a.errors, OFB_CACHE_ELEN);
        first.len = attn_len(a, first.b);
        first.nt = (first.len + ATT_TILE - 1) / ATT_TILE;
        const int share = __ffs(C) - 1;  // (C is a power of two)
        first.t = (int)((int64_t)rank * first.nt >> share);
        first.end = (int)((int64_t)(rank + 1) * first.nt >> share);
        first.f_end = 1;
    } else {
        // places before each sequence; every CTA forms them for itself
        for (int base = 0; base < a.B; base += THREADS) {
            const int b = base + tid;
            int n = 0;
            if (b < a.B) {
                const int len = attn_len(a, b);
                if (a.lens[b] > a.max_len && blockIdx.x == 0) report(a.errors, OFB_CACHE_ELEN);
                n = (len + ATT_TILE - 1) / ATT_TILE;
                last[b] = (uint8_t)(len - (n - 1) * ATT_TILE);
                if (n) n += ATT_PART;
            }
            int s = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += u;
            }
            if (lane == 31) wsum[warp] = s;
            if (!base && !tid) prefix[0] = 0;
            __syncthreads();
            int before = prefix[base];
            for (int w = 0; w < warp; w++) before += wsum[w];
            if (b < a.B) prefix[b + 1] = before + s;
            __syncthreads();
        }
        if (blockIdx.x == 0)
            for (int b = tid; b <= a.B; b += THREADS) a.prefix[b] = prefix[b];
        // sequences without entries: zeros
        for (int b = blockIdx.x; b < a.B; b += gridDim.x)
            if (prefix[b + 1] == prefix[b])
                for (int i = tid; i < a.H * D; i += THREADS) static_cast<IO *>(a.out)[b * a.out_stride + i] = from_f32<IO>(0.0f);
        const AttnSplit sp = AttnSplit::make(prefix[a.B] * nvh, a.ctas, W);
        f0 = sp.first(blockIdx.x), f1 = sp.first(blockIdx.x + 1);
        if (f0 >= f1) return;
        first = attn_part(prefix, last, a.B, nvh, f0, f1);
        if (first.t >= first.end) return;
    }

    const uint32_t ring_s = ax::smem_u32(ring);
    // The tile that the ring is filled with next: its part, number, and each
    // lane's entry with the page number already asked for.
    AttnPart lp = first;
    int lf = f0;
    int lt = lp.t + warp, l_entry = 0, l_page = -1;
    bool more = true;
    auto look_up = [&]() {
        while (more && lt >= lp.end) {
            lf = lp.f_end;
            if (CLUSTER || lf >= f1) more = false;
            else lp = attn_part(prefix, last, a.B, nvh, lf, f1), lt = lp.t + warp;
        }
        if (more) {
            l_entry = lt * ATT_TILE + lane;
            if (l_entry < lp.len) l_page = a.table[(int64_t)lp.b * a.max_pages + a.page.div(l_entry)];
        }
    };
    auto fill = [&](int slot) {
        if (more) {
            const uint32_t dst = ring_s + slot * SH::TILE_BYTES;
            const CT *const k = static_cast<const CT *>(a.k), *const v = static_cast<const CT *>(a.v);
            const int kvh = a.NB == 1 ? lp.vh : lp.vh / a.NB, in = l_entry - a.page.div(l_entry) * a.page_size;
            const bool there = l_entry < lp.len, ok = there && l_page >= 0 && l_page < a.n_pages;
            if (there && !ok) report(a.errors, OFB_CACHE_EPAGE);
            const int64_t off = ok ? l_page * a.page_stride + ((int64_t)kvh * a.page_size + in) * D : -1;
            const uint32_t mask = __ballot_sync(0xffffffffu, ok);
            if (lane == 0) valid[warp][slot] = mask;
            if (a.halves && mask == 0xffffffffu) {  // two times 16 rows on end
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int64_t o = __shfl_sync(0xffffffffu, off, 16 * h) + lane * 8;
                    const CT *ks = k + o, *vs = v + o;
#pragma unroll
                    for (int j = 0; j < 16 * CH / 32; j++) {
                        const int c = j * 32 + lane, r = c / CH, x = c - r * CH;
                        cp16(dst + (16 * h + r) * SH::PITCH + x * 16, ks + j * 256, 16);
                        cp16(dst + (ATT_TILE + 16 * h + r) * SH::PITCH + x * 16, vs + j * 256, 16);
                    }
                }
            } else {
#pragma unroll 4
                for (int j = 0; j < ATT_TILE * CH / 32; j++) {
                    const int c = j * 32 + lane, r = c / CH, x = c - r * CH;
                    const int64_t o = __shfl_sync(0xffffffffu, off, r);
                    // a row that is not there is not read: its address need not exist
                    const int64_t e = o < 0 ? 0 : o + x * 8;
                    const int n = o < 0 ? 0 : 16;
                    cp16(dst + r * SH::PITCH + x * 16, k + e, n);
                    cp16(dst + (ATT_TILE + r) * SH::PITCH + x * 16, v + e, n);
                }
            }
            lt += W;
            look_up();
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    look_up();
    // Queries: row g of A, parts as told at the top. The first part's are asked
    // for before the rings fill, whose copies would keep them waiting.
    IO qx[NR][KS][2][2];
    auto ask_queries = [&](const AttnPart &p) {
        const int kvh = p.vh / a.NB, h0 = (p.vh - kvh * a.NB) * R;
#pragma unroll
        for (int n = 0; n < NR; n++) {
            const IO *qr = static_cast<const IO *>(a.q) + p.b * a.q_stride + (int64_t)(kvh * a.G + h0 + g + 8 * n) * D + c2;
            const bool there = g + 8 * n < min(R, a.G - h0);
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    qx[n][ks][u][0] = there ? qr[ks * 16 + u * 8] : from_f32<IO>(0.0f);
                    qx[n][ks][u][1] = there ? qr[ks * 16 + u * 8 + 1] : from_f32<IO>(0.0f);
                }
        }
    };
    ask_queries(first);
#pragma unroll
    for (int i = 0; i < SH::S - 1; i++) fill(i);
    int slot = 0;  // of the next tile to compute

    int npart = 0;
    AttnPart p = first;
    for (;;) {
        const int kvh = p.vh / a.NB, h0 = (p.vh - kvh * a.NB) * R, rows = min(R, a.G - h0);
        uint32_t qa[QS ? 1 : KS][2][QF][2];  // [k step][k half][fragment][row g, row g + 8]
        float qscale[NR];
        float up[NR];
#pragma unroll
        for (int n = 0; n < NR; n++) {
            up[n] = 1.0f;
            qscale[n] = a.scale;
            if constexpr (F32 && !BF) {
                // a power of two that brings the row's largest element to [2^13, 2^14)
                float m = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ks++)
#pragma unroll
                    for (int u = 0; u < 2; u++) m = fmaxf(m, fmaxf(fabsf(qx[n][ks][u][0]), fabsf(qx[n][ks][u][1])));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                const int e = (int)(__float_as_uint(m) >> 23);  // 0: zero or subnormal, 255: not finite
                if (e > 0 && e < 255) {
                    const int sh = min(max(13 + 127 - e, -100), 100);
                    up[n] = __uint_as_float((uint32_t)(127 + sh) << 23);
                    qscale[n] = a.scale * __uint_as_float((uint32_t)(127 - sh) << 23);
                }
            }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            if (QS && ks % W != warp) continue;
            uint32_t(&to)[2][QF][2] = qa[QS ? 0 : ks];
#pragma unroll
            for (int n = 0; n < NR; n++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    uint32_t part[NQ];
                    split2<CT, NQ>(to_f32(qx[n][ks][u][0]) * up[n], to_f32(qx[n][ks][u][1]) * up[n], part);
#pragma unroll
                    for (int f = 0; f < QF; f++) {
                        if (R == 8) {
                            to[u][f][0] = part[2 * f];
                            to[u][f][1] = 2 * f + 1 < NQ ? part[2 * f + 1 < NQ ? 2 * f + 1 : 0] : 0u;
                        } else {
                            to[u][f][n] = part[f];
                        }
                    }
                }
            if constexpr (QS) {
                q4[ks * 32 + lane] = make_uint4(to[0][0][0], to[0][0][1], to[1][0][0], to[1][0][1]);
                q2[ks * 32 + lane] = make_uint2(to[0][1][0], to[1][1][0]);
            }
        }
        if (QS) __syncthreads();
        float o[D / 8][NO], m[NR], l[NR];
#pragma unroll
        for (int n = 0; n < NR; n++) m[n] = -INFINITY, l[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 8; i++)
#pragma unroll
            for (int u = 0; u < NO; u++) o[i][u] = 0.0f;

        for (int t = p.t + warp; t < p.end; t += W) {
            asm volatile("cp.async.wait_group %0;" ::"n"(SH::S - 2) : "memory");
            __syncwarp();
            fill(slot == 0 ? SH::S - 1 : slot - 1);
            const uint32_t ks_s = ring_s + slot * SH::TILE_BYTES, vs_s = ks_s + ATT_TILE * SH::PITCH;
            const uint32_t ok = valid[warp][slot] >> c2;
            slot = slot == SH::S - 1 ? 0 : slot + 1;

            // scores of 8 entries each; the second fragment on apart, so that small
            // numbers are not cut off against large ones
            float s[4][4] = {}, sl[QF > 1 ? 4 : 1][4] = {};
            const uint32_t ka = ks_s + ((lane & 7) + ((lane >> 4) << 3)) * SH::PITCH + ((lane >> 3) & 1) * 16;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                uint4 x = {};
                uint2 y = {};
                if constexpr (QS) x = q4[ks * 32 + lane], y = q2[ks * 32 + lane];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t b[4];
                    ldmatrix4(b, ka + h * 16 * SH::PITCH + ks * 32);
#pragma unroll
                    for (int f = 0; f < QF; f++) {
                        const int k = QS ? 0 : ks;
                        const uint32_t af[4] = {QS ? (f ? y.x : x.x) : qa[k][0][f][0], QS ? (f ? 0u : x.y) : qa[k][0][f][1],
                                                QS ? (f ? y.y : x.z) : qa[k][1][f][0], QS ? (f ? 0u : x.w) : qa[k][1][f][1]};
                        Mma<CT>::run(f ? sl[QF > 1 ? 2 * h : 0] : s[2 * h], af, b[0], b[1]);
                        Mma<CT>::run(f ? sl[QF > 1 ? 2 * h + 1 : 0] : s[2 * h + 1], af, b[2], b[3]);
                    }
                }
            }
            // rows g (and g + 8), entries 8j + c2 + {0, 1}, in log2
            float z[NR][4][2], alpha[NR];
            uint32_t pa[4][PF][2];  // [8 entries][fragment][row g, row g + 8]
            bool grown = false;
#pragma unroll
            for (int n = 0; n < NR; n++) {
                float mt = -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        float x = s[j][2 * n + u];
                        if (R == 8 && NQ > 1) x += s[j][2 + u];
                        if constexpr (QF > 1) x += sl[j][2 * n + u];
                        z[n][j][u] = (ok >> (8 * j + u)) & 1 ? x * qscale[n] : -INFINITY;
                        mt = fmaxf(mt, z[n][j][u]);
                    }
                if (a.z && g + 8 * n < rows) {
                    float *zr = a.z + ((int64_t)p.b * a.H + kvh * a.G + h0 + g + 8 * n) * a.z_stride + t * ATT_TILE + c2;
#pragma unroll
                    for (int j = 0; j < 4; j++) *reinterpret_cast<float2 *>(zr + 8 * j) = make_float2(z[n][j][0], z[n][j][1]);
                }
                mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
                mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
                const float mn = fmaxf(m[n], mt), ref = mn == -INFINITY ? 0.0f : mn;
                alpha[n] = exp2_fast(m[n] - ref);  // 0 at the first tile
                grown |= mn != m[n];
                m[n] = mn;
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float x = exp2_fast(z[n][j][0] - ref), y = exp2_fast(z[n][j][1] - ref);
                    sum += x + y;
                    uint32_t part[NP];
                    split2<CT, NP>(x * PSCALE, y * PSCALE, part);
#pragma unroll
                    for (int f = 0; f < PF; f++) {
                        if (R == 8) {
                            pa[j][f][0] = part[2 * f];
                            pa[j][f][1] = 2 * f + 1 < NP ? part[2 * f + 1 < NP ? 2 * f + 1 : 0] : 0u;
                        } else {
                            pa[j][f][n] = part[f];
                        }
                    }
                }
                l[n] = l[n] * alpha[n] + sum;
            }
            if (DIRECT && __any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int i = 0; i < D / 8; i++)
#pragma unroll
                    for (int u = 0; u < NO; u++) o[i][u] *= alpha[R == 8 ? 0 : u / 2];
            }
            const uint32_t va = vs_s + ((lane & 7) + ((lane >> 3) & 1) * 8) * SH::PITCH + (lane >> 4) * 16;
#pragma unroll
            for (int n = 0; n < D / 16; n++) {
                float x[2][4] = {};  // of 8 columns each
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t b[4];
                    ldmatrix4_t(b, va + h * 16 * SH::PITCH + n * 32);
#pragma unroll
                    for (int f = 0; f < PF; f++) {
                        const uint32_t af[4] = {pa[2 * h][f][0], pa[2 * h][f][1], pa[2 * h + 1][f][0], pa[2 * h + 1][f][1]};
                        if constexpr (DIRECT) {
                            Mma<CT>::run(o[2 * n], af, b[0], b[1]);
                            Mma<CT>::run(o[2 * n + 1], af, b[2], b[3]);
                        } else {
                            Mma<CT>::run(x[0], af, b[0], b[1]);
                            Mma<CT>::run(x[1], af, b[2], b[3]);
                        }
                    }
                }
                if constexpr (!DIRECT) {
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int u = 0; u < NO; u++) {
                            const float y = R == 8 ? x[i][u] + x[i][u + 2 < 4 ? u + 2 : 0] : x[i][u];
                            o[2 * n + i][u] = o[2 * n + i][u] * alpha[R == 8 ? 0 : u / 2] + y;
                        }
                }
            }
        }
        // merge the warps: their sums, maxima and sums of exponentials. A warp
        // leaves its sums in the ring slot it computed last, which the next
        // fill is for (at the start: the one not filled yet).
#pragma unroll
        for (int n = 0; n < NR; n++) {
            l[n] += __shfl_xor_sync(0xffffffffu, l[n], 1);
            l[n] += __shfl_xor_sync(0xffffffffu, l[n], 2);
        }
        __syncwarp();
        float *const mslot = reinterpret_cast<float *>(ring + (slot == 0 ? SH::S - 1 : slot - 1) * SH::TILE_BYTES);
        float *mw = mslot + g * (D + 4);
        if (lane == 0) mo[warp] = mslot;
        if (CLUSTER && C > 1) {
            cl.barrier_wait();
            if (tid < C)  // tell every CTA where warp 0's sums are
                *cl.map_shared_rank(&all_at[rank], tid) = (int)(reinterpret_cast<uint8_t *>(mslot) - smem);
        }
#pragma unroll
        for (int i = 0; i < D / 8; i++) {
            if (R == 16) {
                *reinterpret_cast<float2 *>(mw + i * 8 + c2) = make_float2(o[i][0], o[i][1]);
                *reinterpret_cast<float2 *>(mw + 8 * (D + 4) + i * 8 + c2) = make_float2(o[i][NO - 2], o[i][NO - 1]);
            } else {
                *reinterpret_cast<float2 *>(mw + i * 8 + c2) =
                    DIRECT ? make_float2(o[i][0] + o[i][NO - 2], o[i][1] + o[i][NO - 1]) : make_float2(o[i][0], o[i][1]);
            }
        }
        if ((lane & 3) == 0)
#pragma unroll
            for (int n = 0; n < NR; n++) mml[warp * R + g + 8 * n] = make_float2(m[n], l[n]);
        // the next part and its queries, on their way while the warps merge
        AttnPart next = p;
        bool go_on = false;
        if (!CLUSTER && p.f_end < f1) {
            next = attn_part(prefix, last, a.B, nvh, p.f_end, f1);
            go_on = next.t < next.end;
            if (AHEAD && go_on) ask_queries(next);
        }
        __syncthreads();
        const bool whole = CLUSTER ? C == 1 : p.t == 0 && p.end == p.nt;
        const int64_t slot_id = 2 * (int64_t)blockIdx.x + (npart ? 1 : 0);
        for (int i = tid; i < rows * (D / 4); i += THREADS) {
            const int r = i / (D / 4), x = (i - r * (D / 4)) * 4;
            float mm = -INFINITY;
#pragma unroll
            for (int w = 0; w < SH::W; w++)
                if (w < W) mm = fmaxf(mm, mml[w * R + r].x);
            const float ref = mm == -INFINITY ? 0.0f : mm;
            float ll = 0.0f;
            float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < SH::W; w++) {
                if (w >= W) break;
                const float2 e = mml[w * R + r];
                const float s = exp2_fast(e.x - ref);
                const float4 y = *reinterpret_cast<const float4 *>(mo[w] + r * (D + 4) + x);
                ll += s * e.y;
                acc.x += s * y.x, acc.y += s * y.y, acc.z += s * y.z, acc.w += s * y.w;
            }
            const int64_t head = kvh * a.G + h0 + r;
            if (CLUSTER && C > 1) {  // in place of warp 0's sums, whose elements only this thread reads
                *reinterpret_cast<float4 *>(mo[0] + r * (D + 4) + x) = acc;
                if (x < 4 * C) cl.map_shared_rank(&all_ml[0][0], x / 4)[rank * R + r] = make_float2(mm, ll);  // to CTA x / 4
            } else if (whole) {
                // no entry attended to (all on bad pages): zeros
                const float inv = ll > 0.0f || ll != ll ? 1.0f / (ll * PSCALE) : 0.0f;
                IO *dst = static_cast<IO *>(a.out) + p.b * a.out_stride + head * D + x;
                dst[0] = from_f32<IO>(acc.x * inv), dst[1] = from_f32<IO>(acc.y * inv);
                dst[2] = from_f32<IO>(acc.z * inv), dst[3] = from_f32<IO>(acc.w * inv);
                if (x == 0) {
                    if (CLUSTER) cml[r] = make_float2(ref, inv * PSCALE);
                    if (!CLUSTER || a.NB > 1) a.ml[(int64_t)p.b * a.H + head] = make_float2(mm, ll);
                }
            } else {
                const float u = 1.0f / PSCALE;
                *reinterpret_cast<float4 *>(a.part_o + (slot_id * R + r) * D + x) = make_float4(acc.x * u, acc.y * u, acc.z * u, acc.w * u);
                if (x == 0) a.part_ml[slot_id * R + r] = make_float2(mm, ll);
            }
        }
        if constexpr (CLUSTER) {
            // join the cluster's CTAs, whose maxima and sums have been told to
            // all; each writes some of the columns
            if (C > 1) cl.sync();
            for (int i = rank * THREADS + tid; C > 1 && i < rows * (D / 4); i += C * THREADS) {
                const int r = i / (D / 4), x = (i - r * (D / 4)) * 4;
                float4 y[8];
                float mm = -INFINITY, ll = 0.0f;
#pragma unroll
                for (int c = 0; c < 8; c++)
                    if (c < C) {
                        y[c] = *reinterpret_cast<const float4 *>(cl.map_shared_rank(smem, c) + all_at[c] + (r * (D + 4) + x) * 4);
                        mm = fmaxf(mm, all_ml[c][r].x);
                    }
                const float ref = mm == -INFINITY ? 0.0f : mm;
                float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
                for (int c = 0; c < 8; c++)
                    if (c < C) {
                        const float2 e = all_ml[c][r];
                        const float s = exp2_fast(e.x - ref);
                        ll += s * e.y;
                        acc.x += s * y[c].x, acc.y += s * y[c].y, acc.z += s * y[c].z, acc.w += s * y[c].w;
                    }
                const float inv = ll > 0.0f || ll != ll ? 1.0f / (ll * PSCALE) : 0.0f;
                IO *dst = static_cast<IO *>(a.out) + p.b * a.out_stride + (int64_t)(kvh * a.G + h0 + r) * D + x;
                dst[0] = from_f32<IO>(acc.x * inv), dst[1] = from_f32<IO>(acc.y * inv);
                dst[2] = from_f32<IO>(acc.z * inv), dst[3] = from_f32<IO>(acc.w * inv);
            }
            // weights: with one pass per kv head this CTA's entries are its own; with more
            // a launch of its own adds them (attn.cu)
            if (a.z) {
                if (C > 1 && tid < rows) {
                    float mm = -INFINITY, ll = 0.0f;
                    for (int c = 0; c < C; c++) mm = fmaxf(mm, all_ml[c][tid].x);
                    const float ref = mm == -INFINITY ? 0.0f : mm;
                    for (int c = 0; c < C; c++) ll += exp2_fast(all_ml[c][tid].x - ref) * all_ml[c][tid].y;
                    cml[tid] = make_float2(ref, ll > 0.0f || ll != ll ? 1.0f / ll : 0.0f);
                    if (a.NB > 1 && rank == 0) a.ml[(int64_t)p.b * a.H + kvh * a.G + h0 + tid] = make_float2(mm, ll);
                }
                __syncthreads();
                const int i1 = a.NB > 1 ? 0 : min(p.end * ATT_TILE, p.len);
                for (int i = p.t * ATT_TILE + tid; i < i1; i += THREADS) {
                    const float *z = a.z + ((int64_t)p.b * a.H + kvh * a.G) * a.z_stride + i;
                    float add = 0.0f;
                    for (int r = 0; r < rows; r++) add += exp2_fast(z[r * a.z_stride] - cml[r].x) * cml[r].y;
                    const int col = a.page.div(i), page = a.table[(int64_t)p.b * a.max_pages + col];
                    if (page >= 0 && page < a.n_pages) a.weight[((int64_t)page * a.KVH + kvh) * a.page_size + (i - col * a.page_size)] += add;
                }
            }
            if (C > 1) cl.sync();  // no CTA leaves while its sums are read
            break;
        }
        if (!go_on) break;
        npart++;
        __syncthreads();  // the slots may be filled again
        p = next;
        if (!AHEAD) ask_queries(p);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

using AttnKernel = void (*)(AttnArgs);
struct AttnVariant {
    AttnKernel run, cluster;
    int ctas, warps;            // CTAs per SM, warps per CTA
    int ring, head;             // shared memory: a warp's ring; all rings and what follows, but for the per-sequence part
};
// Whether there are instances for 16 heads per pass: not where registers cannot
// hold 16 f32 queries and sums.
constexpr bool attn_wide_rows(int d, bool f32) { return !f32 || d <= 128; }
// The instances for a head width: cache type bf16 or fp16, activations f32 or the
// cache's, 8 or 16 query heads per pass.
AttnVariant attn_variant_64(bool bf16, bool f32, int rows);
AttnVariant attn_variant_96(bool bf16, bool f32, int rows);
AttnVariant attn_variant_128(bool bf16, bool f32, int rows);
AttnVariant attn_variant_192(bool bf16, bool f32, int rows);
AttnVariant attn_variant_256(bool bf16, bool f32, int rows);

template <int D, int R, typename CT, typename IO> AttnVariant attn_instance() {
    if constexpr (R == 8 || attn_wide_rows(D, sizeof(IO) == 4)) {
        using SH = AttnShape<D, AttnQuery<D, R, CT, IO>::QB>;
        return {attn_split_kernel<D, R, CT, IO, false>, attn_split_kernel<D, R, CT, IO, true>, SH::CTAS, SH::W,
                SH::ring(1), SH::head(SH::W)};
    } else {
        return {};
    }
}
template <int D, typename CT, typename IO> AttnVariant attn_instances(int rows) {
    return rows == 8 ? attn_instance<D, 8, CT, IO>() : attn_instance<D, 16, CT, IO>();
}

}  // namespace ofb

#define OFB_ATTN_INSTANCES(D)                                                                                   \
    namespace ofb {                                                                                             \
    AttnVariant attn_variant_##D(bool bf16, bool f32, int rows) {                                               \
        if (bf16)                                                                                               \
            return f32 ? attn_instances<D, __nv_bfloat16, float>(rows) : attn_instances<D, __nv_bfloat16, __nv_bfloat16>(rows); \
        return f32 ? attn_instances<D, __half, float>(rows) : attn_instances<D, __half, __half>(rows);          \
    }                                                                                                           \
    }

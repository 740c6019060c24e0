// attn.cu — ofb_attn_decode: the join of the split kernel's parts (attn.cuh)
// and the entry point.
//
// Second launch (programmatic, its CTAs come up as the split kernel's leave): the
// parts of a head that more than one run holds are joined in the order of the runs,
//   M = max m_i, out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i,
// so the result does not depend on which CTA took which run, nor on when. Where a
// head has many parts, a CTA takes 32 columns of it and a quarter of a warp every
// 32nd part (one sequence of 131071 entries, 16 heads of 128 in some 150 parts each:
// 30.7 us in all, with all columns in one CTA 33.1); where it has few, a CTA takes
// eight heads of a kv head, a warp each.
//
// Third launch, with `accumulate` (the second behind clusters of several passes; with
// one pass they do it themselves): each entry's probability, summed over the query
// heads of its kv head in their order, is added to the cache's weight, four
// entries per thread. It reads the scores the split kernel left (4 bytes per entry
// and query head, a sixteenth of the entry's K and V at 8 heads of 128; forming them
// again would read all of K a second time). Of 176 us for 48 ragged sequences, 32 heads
// over 8 kv heads of 128, the scores' way through HBM takes some 15 and this launch
// 10. Asking L2 to keep them, whole lines per store, or weights and join in one launch
// did not make it less.
#include "attn.cuh"

namespace ofb {

constexpr int AJ_THREADS = 256;  // 8 warps, a row each where a CTA joins 8 rows
constexpr int AJ_COLUMNS = 32;  // of a CTA that has one head's parts
constexpr int AJ_CHUNK = 4 * AJ_THREADS;  // entries of one weight CTA

struct AttnJoinArgs {
    AttnArgs a;
    int warps, rows, d;       // of the split kernel: warps of a CTA, heads per pass (8 or 16); head_dim
    FastDiv group;            // by G
    int wide, chunks;         // one head per CTA; weight CTAs per (sequence, kv head)
};

// The runs that hold parts of (sequence b, pass vh): n of them from CTA c0's on.
struct PartRange {
    AttnSplit sp;
    int f0, n, c0;
    __device__ __forceinline__ int slot(int i) const { return 2 * (c0 + i) + (i == 0 && sp.first(c0) < f0 ? 1 : 0); }
};
__device__ __forceinline__ PartRange part_range(const AttnJoinArgs &j, int b, int vh, int nt) {
    const int nvh = j.a.KVH * j.a.NB, places = nt + ATT_PART;
    PartRange r;
    r.sp = AttnSplit::make(j.a.prefix[j.a.B] * nvh, j.a.ctas, j.warps);
    r.f0 = j.a.prefix[b] * nvh + vh * places;
    r.c0 = (r.f0 + ATT_PART) / r.sp.run;
    r.n = (r.f0 + places - 1) / r.sp.run - r.c0 + 1;
    return r;
}

// Sums over parts w, w + step, ... of row r of 4 N columns x on, x + 128 on, for one
// lane; columns from d on are not there.
template <int N> struct JoinSum {
    float m, l;
    float4 o[N];
    __device__ __forceinline__ void add(const AttnJoinArgs &j, const PartRange &pr, int r, int w, int step, int x) {
        m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int h = 0; h < N; h++) o[h] = make_float4(0, 0, 0, 0);
        constexpr int UN = 4;
        for (int i0 = w; i0 < pr.n; i0 += UN * step) {
            float2 e[UN];
            float4 y[UN][N];
#pragma unroll
            for (int k = 0; k < UN; k++) {
                const int i = i0 + k * step;
                e[k] = make_float2(-INFINITY, 0.0f);
#pragma unroll
                for (int h = 0; h < N; h++) y[k][h] = make_float4(0, 0, 0, 0);
                if (i < pr.n) {
                    const int p = pr.slot(i) * j.rows + r;
                    const float *src = j.a.part_o + (int64_t)p * j.d;
                    e[k] = j.a.part_ml[p];
#pragma unroll
                    for (int h = 0; h < N; h++)
                        if (128 * h + x < j.d) y[k][h] = *reinterpret_cast<const float4 *>(src + 128 * h + x);
                }
            }
            float mn = m;
#pragma unroll
            for (int k = 0; k < UN; k++) mn = fmaxf(mn, e[k].x);
            rescale(mn);
            const float ref = mn == -INFINITY ? 0.0f : mn;
#pragma unroll
            for (int k = 0; k < UN; k++) {
                const float f = exp2_fast(e[k].x - ref);
                l += f * e[k].y;
#pragma unroll
                for (int h = 0; h < N; h++)
                    o[h].x += f * y[k][h].x, o[h].y += f * y[k][h].y, o[h].z += f * y[k][h].z, o[h].w += f * y[k][h].w;
            }
        }
    }
    __device__ __forceinline__ void rescale(float mn) {  // to the maximum mn
        const float f = exp2_fast(m - (mn == -INFINITY ? 0.0f : mn));
        m = mn;
        l *= f;
#pragma unroll
        for (int h = 0; h < N; h++) o[h].x *= f, o[h].y *= f, o[h].z *= f, o[h].w *= f;
    }
};

template <typename IO> __global__ void __launch_bounds__(AJ_THREADS) attn_join_kernel(const __grid_constant__ AttnJoinArgs j) {
    constexpr int W = AJ_THREADS / 32;
    __shared__ __align__(16) float acc[W][AJ_COLUMNS];
    __shared__ float2 ml[W];
    const AttnArgs &a = j.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // grid: wide: head, columns, sequence; else eight heads, -, sequence
    const int b = blockIdx.z, shift = j.rows == 16 ? 4 : 3;
    int kvh, g, x;
    if (j.wide) {
        kvh = j.group.div(blockIdx.x), g = (int)blockIdx.x - kvh * a.G;
        x = blockIdx.y * AJ_COLUMNS + lane % 8 * 4;
    } else {
        const int vh = blockIdx.x * W >> shift;
        kvh = a.NB == 1 ? vh : vh / a.NB, g = blockIdx.x * W + warp - (kvh * a.NB << shift);
        x = 4 * lane;
    }
    const int vh = kvh * a.NB + (g >> shift), r = g & (j.rows - 1);
    pdl_wait();
    pdl_trigger();
    const int nt = a.prefix[b + 1] - a.prefix[b] - ATT_PART;
    if (nt < 0) return;
    const PartRange pr = part_range(j, b, vh, nt);
    if (pr.n == 1 || g >= a.G) return;  // (`wide`: the CTA's only head, so all leave)
    IO *const out = static_cast<IO *>(a.out) + b * a.out_stride + (int64_t)(kvh * a.G + g) * j.d + x;
    float2 *const joined = a.ml + (int64_t)b * a.H + kvh * a.G + g;  // for the weights
    if (!j.wide) {
        JoinSum<2> s;
        s.add(j, pr, r, 0, 1, x);
        if (lane == 0) *joined = make_float2(s.m, s.l);
        const float inv = s.l > 0.0f || s.l != s.l ? 1.0f / s.l : 0.0f;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (128 * h + x >= j.d) break;
            out[128 * h] = from_f32<IO>(s.o[h].x * inv), out[128 * h + 1] = from_f32<IO>(s.o[h].y * inv);
            out[128 * h + 2] = from_f32<IO>(s.o[h].z * inv), out[128 * h + 3] = from_f32<IO>(s.o[h].w * inv);
        }
        return;
    }
    // four parts side by side in a warp, joined by shuffles, then the warps
    JoinSum<1> s;
    s.add(j, pr, r, warp * 4 + lane / 8, W * 4, x);
#pragma unroll
    for (int o = 8; o < 32; o <<= 1) {
        s.rescale(fmaxf(s.m, __shfl_xor_sync(0xffffffffu, s.m, o)));
        s.l += __shfl_xor_sync(0xffffffffu, s.l, o);
        s.o[0].x += __shfl_xor_sync(0xffffffffu, s.o[0].x, o);
        s.o[0].y += __shfl_xor_sync(0xffffffffu, s.o[0].y, o);
        s.o[0].z += __shfl_xor_sync(0xffffffffu, s.o[0].z, o);
        s.o[0].w += __shfl_xor_sync(0xffffffffu, s.o[0].w, o);
    }
    if (lane == 0) ml[warp] = make_float2(s.m, s.l);
    if (lane < 8) *reinterpret_cast<float4 *>(&acc[warp][4 * lane]) = s.o[0];
    __syncthreads();
    if (tid >= AJ_COLUMNS) return;
    float m = -INFINITY, l = 0.0f, v = 0.0f;
#pragma unroll
    for (int w = 0; w < W; w++) m = fmaxf(m, ml[w].x);
    const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int w = 0; w < W; w++) {
        const float f = exp2_fast(ml[w].x - ref);
        l += f * ml[w].y;
        v += f * acc[w][tid];
    }
    out[tid - x % AJ_COLUMNS] = from_f32<IO>(l > 0.0f || l != l ? v / l : 0.0f);
    if (x == 0) *joined = make_float2(m, l);
}

constexpr int AW_HEADS = 128;  // heads whose maximum and sum are in shared memory at a time
__global__ void __launch_bounds__(AJ_THREADS) attn_weight_kernel(const __grid_constant__ AttnJoinArgs j) {
    __shared__ float2 ml[AW_HEADS];  // (maximum, 1 / sum)
    const AttnArgs &a = j.a;
    const int tid = threadIdx.x;
    const int u = blockIdx.x / j.chunks, b = u / a.KVH, kvh = u - b * a.KVH, i0 = (blockIdx.x - u * j.chunks) * AJ_CHUNK;
    pdl_wait();
    pdl_trigger();
    const int len = attn_len(a, b), i = i0 + 4 * tid;
    if (i0 >= len) return;
    // the entries' weights, asked for beside the scores
    const bool quad = a.quads && i + 3 < len;  // four entries in one page, 16-byte aligned
    float *at[4] = {nullptr, nullptr, nullptr, nullptr};
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int x = 0; x < 4; x++) {
        if (i + x >= len || (quad && x)) break;
        const int col = a.page.div(i + x), page = a.table[(int64_t)b * a.max_pages + col];
        if (page < 0 || page >= a.n_pages) continue;
        at[x] = a.weight + ((int64_t)page * a.KVH + kvh) * a.page_size + (i + x - col * a.page_size);
        if (quad) {
            const float4 y = *reinterpret_cast<const float4 *>(at[0]);
            v[0] = y.x, v[1] = y.y, v[2] = y.z, v[3] = y.w;
        } else {
            v[x] = *at[x];
        }
    }
    float4 add = make_float4(0, 0, 0, 0);
    for (int g0 = 0; g0 < a.G; g0 += AW_HEADS) {
        const int ng = min(a.G - g0, AW_HEADS);
        if (tid < ng) {
            const float2 e = a.ml[(int64_t)b * a.H + kvh * a.G + g0 + tid];
            ml[tid] = make_float2(e.x == -INFINITY ? 0.0f : e.x, e.y > 0.0f || e.y != e.y ? 1.0f / e.y : 0.0f);
        }
        // scores are there up to the end of the last tile
        const float *z = a.z + ((int64_t)b * a.H + kvh * a.G + g0) * a.z_stride + i;
        float4 x[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (i < len && k < ng) x[k] = *reinterpret_cast<const float4 *>(z + k * a.z_stride);
        __syncthreads();
        for (int g = 0; i < len && g < ng; g += 4) {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (g + k >= ng) break;
                const float2 e = ml[g + k];
                add.x += exp2_fast(x[k].x - e.x) * e.y, add.y += exp2_fast(x[k].y - e.x) * e.y;
                add.z += exp2_fast(x[k].z - e.x) * e.y, add.w += exp2_fast(x[k].w - e.x) * e.y;
                if (g + 4 + k < ng) x[k] = *reinterpret_cast<const float4 *>(z + (g + 4 + k) * a.z_stride);
            }
        }
        __syncthreads();
    }
    if (quad) {
        if (at[0]) *reinterpret_cast<float4 *>(at[0]) = make_float4(v[0] + add.x, v[1] + add.y, v[2] + add.z, v[3] + add.w);
    } else {
        if (at[0]) *at[0] = v[0] + add.x;
        if (at[1]) *at[1] = v[1] + add.y;
        if (at[2]) *at[2] = v[2] + add.z;
        if (at[3]) *at[3] = v[3] + add.w;
    }
}

// Tiles per warp up to which a sequence is left to a cluster: 2 heads of 16 over one
// sequence of 1500 entries (two tiles) 7.9 us, as runs and a join 8.6; of 2500 10.9
// and 9.2. CTAs of one warp, up to 4 tiles: 64 x 8 kv heads of 100 entries with
// weights 18.0 us against 21.7, 95 x 3 of 15 entries (256) 12.4 against 27.7.
constexpr int ATT_SHORT = 3, ATT_ONE_WARP = 4;

struct AttnPlan {
    AttnVariant v;
    int max_len, ctas, NB, rows;
    int warps;    // of a CTA of those
    int cluster;  // CTAs per (sequence, pass) that join by themselves, or 0: runs and a second launch
    int64_t z_stride;
    size_t prefix, ml, part_o, part_ml, z, total;
};

// Checks the call's sizes and lays out its scratch.
static int attn_plan(const ofb_kv_cache *c, int n_heads, int n_seqs, int max_len, int accumulate, bool f32, AttnPlan &p) {
    int st = check_cache(c, "ofb_attn_decode");
    if (st != OFB_OK) return st;
    if (n_heads < 1 || n_heads % c->n_kv_heads || n_heads > 65536 || n_seqs < 0 || n_seqs > c->n_seqs || max_len < 0 ||
        (accumulate != 0 && accumulate != 1)) {
        set_error("ofb_attn_decode: %d heads over %d kv heads, %d sequences of %d, max_len %d", n_heads, c->n_kv_heads, n_seqs,
                  c->n_seqs, max_len);
        return OFB_EINVAL;
    }
    if (accumulate && !c->weight) { set_error("ofb_attn_decode: accumulate needs the cache's weight"); return OFB_EINVAL; }
    if (n_seqs > ATT_MAX_SEQS) { set_error("ofb_attn_decode: %d sequences, %d at most", n_seqs, ATT_MAX_SEQS); return OFB_ETOOLARGE; }
    const int reach = cache_reach(c);
    p.max_len = max_len && max_len < reach ? max_len : reach;
    const int64_t tiles = ((int64_t)p.max_len + ATT_TILE - 1) / ATT_TILE;
    const int group = n_heads / c->n_kv_heads;
    p.rows = group > 8 && attn_wide_rows(c->head_dim, f32) ? 16 : 8;
    p.NB = (group + p.rows - 1) / p.rows;
    if ((tiles + ATT_PART) * n_seqs > (1 << 30) / ((int64_t)c->n_kv_heads * p.NB)) {  // (sums of tile numbers stay within 31 bits)
        set_error("ofb_attn_decode: %d sequences of %d entries are too many tiles", n_seqs, p.max_len);
        return OFB_ETOOLARGE;
    }
    const bool bf = c->type == OFB_TYPE_BF16;
    switch (c->head_dim) {
    case 64: p.v = attn_variant_64(bf, f32, p.rows); break;
    case 96: p.v = attn_variant_96(bf, f32, p.rows); break;
    case 128: p.v = attn_variant_128(bf, f32, p.rows); break;
    case 192: p.v = attn_variant_192(bf, f32, p.rows); break;
    default: p.v = attn_variant_256(bf, f32, p.rows); break;
    }
    const int64_t runs = (int64_t)n_seqs * c->n_kv_heads * p.NB * ((tiles + p.v.warps - 1) / p.v.warps);
    const int most = sm_count() * p.v.ctas;
    const int64_t units = (int64_t)n_seqs * c->n_kv_heads * p.NB;
    // Short sequences: clusters of as many CTAs as give each warp a tile, while all
    // have room at once and no warp more than ATT_SHORT; for so many sequences that
    // they have no room at once a CTA of one warp each, of which an SM holds more.
    // Weights they add themselves, but for a kv head's query heads in several passes
    // (80 sequences of 9 to 13 entries, 16 f32 heads of 256 in two: 23.1 us, as runs 33.7).
    p.cluster = 0;
    int n = 1;
    while (n < 8 && tiles > n * p.v.warps && 2 * n * units <= most) n *= 2;
    if (units <= most && tiles <= (int64_t)n * p.v.warps * ATT_SHORT) {
        p.cluster = n;
        p.warps = p.v.warps;
    } else if (units > most && tiles <= ATT_ONE_WARP) {
        p.cluster = p.warps = 1;
    }
    p.ctas = runs < 1 ? 1 : runs < most ? (int)runs : most;
    const size_t parts = 2 * (size_t)ATT_MAX_CTAS * sm_count();  // whatever the type: one scratch serves both
    p.z_stride = tiles * ATT_TILE;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t o = at; at += (bytes + 255) / 256 * 256; return o; };
    p.prefix = take((size_t)(n_seqs + 1) * 4);
    p.ml = take((size_t)n_seqs * n_heads * 8);
    // sized for a full grid, so that the size grows with n_seqs and max_len
    p.part_ml = take(parts * 16 * 8);
    p.part_o = take(parts * 16 * c->head_dim * 4);
    p.z = accumulate ? take((size_t)n_seqs * n_heads * p.z_stride * 4) : 0;
    p.total = at;
    return OFB_OK;
}

}  // namespace ofb

using namespace ofb;

extern "C" size_t ofb_attn_scratch_size(const ofb_kv_cache *cache, int n_heads, int n_seqs, int max_len, int accumulate) {
    AttnPlan p;
    return attn_plan(cache, n_heads, n_seqs, max_len, accumulate, true, p) == OFB_OK ? p.total : 0;
}

extern "C" int ofb_attn_decode(const ofb_kv_cache *cache, const void *q, int type, int64_t q_stride, int n_heads,
                               float scale, const int32_t *lens, int n_seqs, int max_len, int accumulate, void *out,
                               int64_t out_stride, void *scratch, size_t scratch_bytes, void *stream) {
    AttnPlan p;
    int st = attn_plan(cache, n_heads, n_seqs, max_len, accumulate, type == OFB_TYPE_F32, p);
    if (st != OFB_OK) return st;
    if (type != OFB_TYPE_F32 && type != cache->type) {
        set_error("ofb_attn_decode: type %d is neither F32 nor the cache's", type);
        return OFB_EUNSUPPORTED;
    }
    if (!n_seqs) return OFB_OK;
    const int64_t width = (int64_t)n_heads * cache->head_dim;
    if (!q || !lens || !out || q == out || misaligned(q, type_size(type)) || misaligned(out, type_size(type)) ||
        misaligned(lens, 4) || (n_seqs > 1 && (q_stride < width || out_stride < width)) || !(scale == scale)) {
        set_error("ofb_attn_decode: bad arguments (q stride %lld, out stride %lld)", (long long)q_stride, (long long)out_stride);
        return OFB_EINVAL;
    }
    if (!scratch || misaligned(scratch, 16)) { set_error("ofb_attn_decode: scratch is NULL or not 16-byte aligned"); return OFB_EINVAL; }
    if (scratch_bytes < p.total) {
        set_error("ofb_attn_decode: scratch of %zu bytes, %zu needed", scratch_bytes, p.total);
        return OFB_ETOOLARGE;
    }
    uint8_t *w = static_cast<uint8_t *>(scratch);
    AttnJoinArgs j = {};
    AttnArgs &a = j.a;
    a.k = cache->k, a.v = cache->v, a.q = q, a.out = out, a.table = cache->page_table, a.lens = lens;
    a.page_stride = cache_page_stride(cache), a.q_stride = q_stride, a.out_stride = out_stride;
    a.B = n_seqs, a.KVH = cache->n_kv_heads, a.G = n_heads / a.KVH, a.NB = p.NB, a.H = n_heads;
    a.page_size = cache->page_size, a.max_pages = cache->max_pages, a.n_pages = cache->n_pages, a.max_len = p.max_len;
    a.page = fast_div(a.page_size), a.ctas = fast_div(p.ctas), a.halves = a.page_size % 16 == 0;
    a.scale = scale * 1.4426950408889634f;
    a.errors = cache->errors;
    a.prefix = reinterpret_cast<int *>(w + p.prefix), a.ml = reinterpret_cast<float2 *>(w + p.ml);
    a.part_o = reinterpret_cast<float *>(w + p.part_o), a.part_ml = reinterpret_cast<float2 *>(w + p.part_ml);
    a.z = accumulate ? reinterpret_cast<float *>(w + p.z) : nullptr;
    a.z_stride = p.z_stride, a.weight = cache->weight;
    a.quads = a.page_size % 4 == 0 && !misaligned(a.weight, 16);
    j.group = fast_div(a.G), j.warps = p.v.warps, j.rows = p.rows, j.d = cache->head_dim;
    // parts of a head, about, when all sequences are of the largest length
    j.wide = p.ctas >= 4 * n_seqs * a.KVH * a.NB;
    j.chunks = (p.max_len + AJ_CHUNK - 1) / AJ_CHUNK;
    const int64_t weight_ctas = (int64_t)n_seqs * a.KVH * j.chunks;
    if (accumulate && weight_ctas > INT32_MAX) { set_error("ofb_attn_decode: too many weight blocks"); return OFB_ETOOLARGE; }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // a raised shared-memory limit per kernel and device
    static size_t attr[80][64];
    const int vi = (cache->head_dim == 64 ? 0 : cache->head_dim == 96 ? 1 : cache->head_dim == 128 ? 2 : cache->head_dim == 192 ? 3 : 4) * 16 +
                   (cache->type == OFB_TYPE_BF16 ? 8 : 0) + (type == OFB_TYPE_F32 ? 4 : 0) + (p.rows == 16 ? 2 : 0);
    auto weights = [&]() {
        const cudaError_t e = launch_pdl(attn_weight_kernel, dim3((unsigned)weight_ctas), dim3(AJ_THREADS), 0, s, j);
        return e == cudaSuccess ? OFB_OK : cuda_status(e, "ofb_attn_decode weight launch");
    };
    if (p.cluster) {
        const size_t smem = p.v.head - (size_t)(p.v.warps - p.warps) * p.v.ring;
        cudaError_t e = ensure_dyn_smem(p.v.cluster, p.v.head, attr[vi + 1]);
        if (e != cudaSuccess) return cuda_status(e, "ofb_attn_decode smem attribute");
        e = launch_pdl_cluster(p.v.cluster, dim3((unsigned)(n_seqs * a.KVH * a.NB * p.cluster)), dim3(p.warps * 32), p.cluster,
                               smem, s, a);
        if (e != cudaSuccess) return cuda_status(e, "ofb_attn_decode launch");
        return accumulate && p.NB > 1 ? weights() : OFB_OK;
    }
    const size_t smem = p.v.head + (size_t)(n_seqs + 1) * 4 + (n_seqs + 3) / 4 * 4;
    cudaError_t e = ensure_dyn_smem(p.v.run, smem, attr[vi]);
    if (e != cudaSuccess) return cuda_status(e, "ofb_attn_decode smem attribute");
    e = launch_pdl(p.v.run, dim3(p.ctas), dim3(p.v.warps * 32), smem, s, a);
    if (e != cudaSuccess) return cuda_status(e, "ofb_attn_decode launch");
    if (p.ctas == 1 && !accumulate) return OFB_OK;  // every part is whole
    const dim3 block(AJ_THREADS), grid = j.wide ? dim3(n_heads, j.d / AJ_COLUMNS, n_seqs) : dim3(a.KVH * a.NB * p.rows / (AJ_THREADS / 32), 1, n_seqs);
    e = type == OFB_TYPE_F32              ? launch_pdl(attn_join_kernel<float>, grid, block, 0, s, j)
        : cache->type == OFB_TYPE_BF16 ? launch_pdl(attn_join_kernel<__nv_bfloat16>, grid, block, 0, s, j)
                                       : launch_pdl(attn_join_kernel<__half>, grid, block, 0, s, j);
    if (e != cudaSuccess) return cuda_status(e, "ofb_attn_decode join launch");
    return accumulate ? weights() : OFB_OK;
}

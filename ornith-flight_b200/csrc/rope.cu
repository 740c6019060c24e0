// rope.cu — rotary positions with several axes, and the entry of new tokens
// into the paged cache (ofb_rope, ofb_rope_append).
//
//   y[u] = x[u] cos a - x[v] sin a,  y[v] = x[v] cos a + x[u] sin a,
//   a = pos[axis(i)] * f(i) for pair i = (u, v)
//
// HBM-bound: every element is read and written once, in one launch for q, k
// and v. A CTA owns a few tokens. It first forms the cosine and sine of each
// (token, pair) once in shared memory, for all heads. A far position times a
// frequency would lose its place in the turn in f32; here f(i) / 2 pi comes as a
// 64-bit fraction of a turn, and since positions are integers, the product's low
// 64 bits are that fraction's exact place: its top word, as f32 half turns within
// [-1, 1], is off by at most 2^-25 + 2^-31. The fraction itself comes from up to 127
// products in 64 bits of mantissa, from one powl (per axis with pairs when those have
// frequencies of their own), and is cut off after 64 bits: for a base of 1 or more,
// whose frequencies are 1 at most, off by less than 62 * 2^-64 turns, which at position
// 2^31 is less than 2^-26 half turns (base 10000, 128 pairs: some 2^-32). A base below
// 1 has frequencies above 1, and so much larger an error. The fractions are 1 KB of
// arguments. Then each thread takes items of two 8-element chunks (the two halves of 8
// pairs, or 16 neighbours), read and written 16 bytes at a time. Sizes or addresses
// that do not allow it (head_dim or rot_dim no multiple of 16, strides no
// multiple of 8, pointers off 16 bytes) take the second kernel, a pair per
// item.
#include <math.h>

#include "kv_cache.cuh"

namespace ofb {

constexpr int RP_THREADS = 256;
constexpr int RP_PAIRS = 128;
constexpr int RP_TOKENS = 1 << 30;

struct RopeArgs {
    int T, H, KVH, d, rot, tpb;  // heads of q; kv heads (0: no cache); tokens of a group
    // first kernel: rows of a CTA under way, CTAs that share a group's rows
    int slots, split;
    int n_pages, page_size, n_seqs, max_pages;
    FastDiv page, rows, per_row, pairs;  // by page_size, by H + 2 KVH, by chunk pairs of a row, by rot / 2
    const void *q, *k, *v;
    void *q_out, *ck, *cv;
    int64_t qs, ks, vs, qos, page_stride, pos_stride;
    const int32_t *pos, *seq, *index, *number, *table;
    float *weight;
    int32_t *order;
    uint32_t *errors;
    uint64_t turns[RP_PAIRS];     // f(i) / 2 pi, a fraction of 2^64
    uint8_t axis[RP_PAIRS];
};

// Where a CTA's tokens go (a page below 0: nowhere) and their order numbers.
struct RopeEntry {
    int page, slot, number;
};
// Cosine and sine of position pos at a frequency.
__device__ __forceinline__ float2 rope_angle(int pos, uint64_t turns) {
    const uint64_t place = (uint64_t)(int64_t)pos * turns;
    float s, c;
    sincospif((float)(int)(place >> 32) * 0x1p-31f, &s, &c);
    return make_float2(c, s);
}

// The place of token t's rows; reports what is wrong with it.
__device__ __forceinline__ RopeEntry rope_entry(const RopeArgs &a, int t) {
    const int b = a.seq[t], i = a.index[t];
    RopeEntry e = {-1, 0, a.number ? a.number[t] : i};
    if (b < 0) return e;
    const int col = i < 0 ? 0 : a.page.div(i);
    if (b >= a.n_seqs || i < 0 || col >= a.max_pages) {
        report(a.errors, OFB_CACHE_EINDEX);
        return e;
    }
    const int p = a.table[(int64_t)b * a.max_pages + col];
    if (p < 0 || p >= a.n_pages) {
        report(a.errors, OFB_CACHE_EPAGE);
        return e;
    }
    e.page = p;
    e.slot = i - col * a.page_size;
    return e;
}

// Shared memory of the second kernel: cosines [tpb][rot/2], sines [tpb][rot/2], entries [tpb].
struct RopeShared {
    float *c, *s;
    RopeEntry *entry;
    __device__ __forceinline__ RopeShared(const RopeArgs &a, float *base)
        : c(base), s(base + a.tpb * (a.rot / 2)), entry(reinterpret_cast<RopeEntry *>(base + (a.tpb * a.rot + 3) / 4 * 4)) {}
};

__device__ __forceinline__ void rope_setup(const RopeArgs &a, int t0, int nt, const RopeShared &sh) {
    const int pairs = a.rot / 2;
    // read through a plain address: lanes want different pairs, which the
    // constant bank would serve one at a time
    const uint64_t *freq = a.turns;
    const uint8_t *axis = a.axis;
    asm("" : "+l"(freq), "+l"(axis));
    for (int i = threadIdx.x; i < nt * pairs; i += RP_THREADS) {
        const int t = a.pairs.div(i), p = i - t * pairs;
        const float2 cs = rope_angle(a.pos[axis[p] * a.pos_stride + t0 + t], freq[p]);
        sh.c[i] = cs.x;
        sh.s[i] = cs.y;
    }
    if (a.KVH && threadIdx.x < nt) sh.entry[threadIdx.x] = rope_entry(a, t0 + threadIdx.x);
    __syncthreads();
}

// Weight 0 and the order number of the CTA's new entries.
__device__ __forceinline__ void rope_meta(const RopeArgs &a, int nt, const RopeEntry *entry) {
    if (!a.weight && !a.order) return;
    for (int i = threadIdx.x; i < nt * a.KVH; i += RP_THREADS) {
        const int t = i / a.KVH, h = i - t * a.KVH;
        const RopeEntry e = entry[t];
        if (e.page < 0) continue;
        const int64_t m = ((int64_t)e.page * a.KVH + h) * a.page_size + e.slot;
        if (a.weight) a.weight[m] = 0.0f;
        if (a.order) a.order[m] = e.number;
    }
}

// A row of the launch: row `row` of token t of the group, the queries first,
// then the keys and the values.
struct RopeRow {
    int t, row;
};
__device__ __forceinline__ RopeRow rope_row(const RopeArgs &a, int vr) {
    const int t = a.rows.div(vr);
    return {t, vr - t * (int)a.rows.d};
}
template <typename IO> __device__ __forceinline__ const IO *rope_src(const RopeArgs &a, const RopeRow &r, int t0) {
    const bool is_q = r.row < a.H, is_v = r.row >= a.H + a.KVH;
    const void *p = is_q ? a.q : is_v ? a.v : a.k;
    const int64_t stride = is_q ? a.qs : is_v ? a.vs : a.ks;
    const int h = r.row - (is_q ? 0 : is_v ? a.H + a.KVH : a.H);
    return static_cast<const IO *>(p) + (t0 + r.t) * stride + (int64_t)h * a.d;
}
__device__ __forceinline__ int64_t rope_cache_at(const RopeArgs &a, const RopeEntry &e, int h) {
    return e.page * a.page_stride + ((int64_t)h * a.page_size + e.slot) * a.d;
}

// Sixteen elements of a row as loaded.
template <typename IO> struct RopeRaw {
    uint4 x[sizeof(IO) / 2], y[sizeof(IO) / 2];
    __device__ __forceinline__ void load(const IO *p, int at, int bt) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(IO) / 2; i++) {
            x[i] = reinterpret_cast<const uint4 *>(p + at)[i];
            y[i] = reinterpret_cast<const uint4 *>(p + bt)[i];
        }
    }
};

// A CTA has tpb tokens (most often one). Thread (slot, j) takes chunk pair j of rows
// slot, slot + slots, ...: it asks for its first three (f32: two) items at once;
// while they are on their way the last threads find the tokens' places in the cache
// and the first ones form the cosines, so that the three waits are one. Measured on
// 8190 tokens with 32 + 2 x 8 heads of 128, bf16: 38.7 us, 5.2 TB/s, where adding a
// number to as many bytes takes 32 (16383 tokens x 16 heads alone: 23.9 and 21.7).
// A plain division by the pairs where the cosines are formed cost 5% of that, with
// all CTAs waiting on it: 40.5. Against 39.5 for 7 CTAs per SM then, 8 took 39.8, 6
// 41.2, 4 items at once 43, 2 x 192 threads 42, 3 x 256 41; CTAs that stay and ask for
// the next group's loads, positions and pages ahead 45.
constexpr int RV_THREADS = 128, RV_CTAS = 7;  // CTAs per SM that registers allow
template <typename IO> constexpr int RV_BATCH = sizeof(IO) == 2 ? 3 : 2;  // items asked for at once
template <typename IO, typename CT, bool ADJ, bool CACHE>
__global__ void __launch_bounds__(RV_THREADS, RV_CTAS) rope_vec_kernel(const __grid_constant__ RopeArgs a) {
    constexpr int BATCH = RV_BATCH<IO>;
    extern __shared__ __align__(16) float rope_smem[];  // cosines, sines [tpb][rot/2], places [tpb]
    const int half = a.rot / 2, tid = threadIdx.x, part = blockIdx.x % a.split;
    const int t0 = blockIdx.x / a.split * a.tpb, nt = min(a.tpb, a.T - t0);
    float *const cosines = rope_smem, *const sines = rope_smem + a.tpb * half;
    RopeEntry *const entry = reinterpret_cast<RopeEntry *>(rope_smem + a.tpb * a.rot);
    const int in = a.per_row.div(tid), j = tid - in * (int)a.per_row.d, total = in < a.slots ? nt * (int)a.rows.d : 0;
    const int slot = part * a.slots + in, step = a.split * a.slots;  // first row, from one item to the next
    // The thread's two chunks of 8 elements and where their cosines are. HALVES:
    // the two halves of 8 pairs, or two chunks behind rot; ADJACENT: 4 pairs
    // each, half a row apart. Neighbouring threads have neighbouring chunks.
    int ta, tb;
    bool turn_a, turn_b;
    if (ADJ) {
        ta = 8 * j, tb = a.d / 2 + 8 * j;
        turn_a = ta < a.rot, turn_b = tb < a.rot;
    } else {
        const int pr = a.rot / 16, rest = (a.d - a.rot) / 2;
        turn_a = turn_b = j < pr;
        ta = turn_a ? 8 * j : a.rot + 8 * (j - pr), tb = ta + (turn_a ? half : rest);
    }
    pdl_wait();
    pdl_trigger();
    RopeRaw<IO> raw[BATCH];
    auto fetch = [&](int vr) {
#pragma unroll
        for (int k = 0; k < BATCH; k++)
            if (vr + k * step < total) {
                const RopeRow r = rope_row(a, vr + k * step);
                if constexpr (CACHE) raw[k].load(rope_src<IO>(a, r, t0), ta, tb);
                else raw[k].load(static_cast<const IO *>(a.q) + (t0 + r.t) * a.qs + (int64_t)r.row * a.d, ta, tb);
            }
    };
    fetch(slot);
    // (by the last threads: the first ones have the cosines)
    if (CACHE && RV_THREADS - 1 - tid < nt) entry[RV_THREADS - 1 - tid] = rope_entry(a, t0 + RV_THREADS - 1 - tid);
    {
        const uint64_t *freq = a.turns;  // see rope_setup
        const uint8_t *axis = a.axis;
        asm("" : "+l"(freq), "+l"(axis));
#pragma unroll 1
        for (int i = tid; i < nt * half; i += RV_THREADS) {
            const int t = a.pairs.div(i), p = i - t * half;
            const float2 cs = rope_angle(a.pos[axis[p] * a.pos_stride + t0 + t], freq[p]);
            cosines[i] = cs.x;
            sines[i] = cs.y;
        }
    }
    __syncthreads();
    for (int vr = slot; vr < total; vr += BATCH * step) {
        if (vr > slot) fetch(vr);
#pragma unroll
        for (int k = 0; k < BATCH; k++) {
            if (vr + k * step >= total) break;
            const RopeRow r = rope_row(a, vr + k * step);
            const bool is_q = !CACHE || r.row < a.H, is_v = CACHE && r.row >= a.H + a.KVH;
            float x[8], y[8];
            load8(reinterpret_cast<const IO *>(raw[k].x), x);
            load8(reinterpret_cast<const IO *>(raw[k].y), y);
            const float *cs = cosines + r.t * half, *sn = sines + r.t * half;
            if (ADJ) {
                auto turn4 = [&](float(&z)[8], int at) {
                    const float4 c = *reinterpret_cast<const float4 *>(cs + at), s = *reinterpret_cast<const float4 *>(sn + at);
                    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float u = z[2 * i], v = z[2 * i + 1];
                        z[2 * i] = u * cc[i] - v * ss[i];
                        z[2 * i + 1] = v * cc[i] + u * ss[i];
                    }
                };
                if (turn_a && !is_v) turn4(x, ta / 2);
                if (turn_b && !is_v) turn4(y, tb / 2);
            } else if (turn_a && !is_v) {
                float c[8], s[8];
                load8(cs + 8 * j, c);
                load8(sn + 8 * j, s);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float u = x[i], v = y[i];
                    x[i] = u * c[i] - v * s[i];
                    y[i] = v * c[i] + u * s[i];
                }
            }
            if (is_q) {
                IO *dst = static_cast<IO *>(a.q_out) + (t0 + r.t) * a.qos + (int64_t)r.row * a.d;
                store8(dst + ta, x);
                store8(dst + tb, y);
            } else if (const RopeEntry e = entry[r.t]; e.page >= 0) {
                const int h = r.row - a.H - (is_v ? a.KVH : 0);
                CT *dst = static_cast<CT *>(is_v ? a.cv : a.ck) + rope_cache_at(a, e, h);
                store8(dst + ta, x);
                store8(dst + tb, y);
                if (!is_v && j == 0) {  // with its key row: weight 0 and the order number
                    const int64_t m = ((int64_t)e.page * a.KVH + h) * a.page_size + e.slot;
                    if (a.weight) a.weight[m] = 0.0f;
                    if (a.order) a.order[m] = e.number;
                }
            }
        }
    }
}

// Any sizes and strides: items are pairs (rot/2 per row), then single elements, with
// element loads and plain divisions per item, which bound it: 16383 tokens x 16 heads of
// 128 one element off take 85 us in bf16 and 83 in f32, where the first kernel takes 25
// and 43. Kept simple: rows of a projection start on 16 bytes.
template <typename IO, typename CT>
__global__ void __launch_bounds__(RP_THREADS) rope_any_kernel(const __grid_constant__ RopeArgs a, int adjacent) {
    extern __shared__ __align__(16) float rope_smem[];
    const RopeShared sh(a, rope_smem);
    pdl_wait();
    pdl_trigger();
    const int t0 = blockIdx.x * a.tpb, nt = min(a.tpb, a.T - t0), half = a.rot / 2;
    rope_setup(a, t0, nt, sh);
    const int per_row = a.d - half, total = nt * (int)a.rows.d * per_row;
    for (int it = threadIdx.x; it < total; it += RP_THREADS) {
        const int vr = it / per_row, j = it - vr * per_row;
        const RopeRow r = rope_row(a, vr);
        const bool is_q = r.row < a.H, is_v = r.row >= a.H + a.KVH;
        if (!is_q && sh.entry[r.t].page < 0) continue;
        const IO *src = rope_src<IO>(a, r, t0);
        // where this item's one or two elements are
        const int ea = j >= half ? half + j : adjacent ? 2 * j : j, eb = j >= half ? ea : adjacent ? 2 * j + 1 : half + j;
        float x = to_f32(src[ea]), y = to_f32(src[eb]);
        if (!is_v && j < half) {
            const float c = sh.c[r.t * half + j], s = sh.s[r.t * half + j], u = x, v = y;
            x = u * c - v * s;
            y = v * c + u * s;
        }
        if (is_q) {
            IO *dst = static_cast<IO *>(a.q_out) + (t0 + r.t) * a.qos + (int64_t)r.row * a.d;
            dst[ea] = from_f32<IO>(x);
            dst[eb] = from_f32<IO>(y);
        } else {
            CT *dst = static_cast<CT *>(is_v ? a.cv : a.ck) + rope_cache_at(a, sh.entry[r.t], r.row - a.H - (is_v ? a.KVH : 0));
            dst[ea] = from_f32<CT>(x);
            dst[eb] = from_f32<CT>(y);
        }
    }
    rope_meta(a, nt, sh.entry);
}

// Checks a rotary form and lays out its pairs: axis and frequency / 2 pi.
static int rope_tables(const ofb_rope_config *r, int head_dim, const char *who, RopeArgs &a) {
    if (r->rot_dim < 2 || r->rot_dim > 2 * RP_PAIRS || r->rot_dim % 2 || r->rot_dim > head_dim || r->n_axes < 1 ||
        r->n_axes > 4 || (r->pairing != OFB_ROPE_HALVES && r->pairing != OFB_ROPE_ADJACENT) ||
        (r->order != OFB_ROPE_BLOCKED && r->order != OFB_ROPE_DEALT) || (r->per_axis != 0 && r->per_axis != 1) ||
        !(r->base > 0) || !isfinite(r->base)) {
        set_error("%s: rotary form out of range (rot_dim %d, head_dim %d, axes %d, pairing %d, order %d, per_axis %d, base %g)", who,
                  r->rot_dim, head_dim, r->n_axes, r->pairing, r->order, r->per_axis, r->base);
        return OFB_EINVAL;
    }
    if (r->per_axis && r->order != OFB_ROPE_BLOCKED) {
        set_error("%s: per_axis frequencies need blocked sections", who);
        return OFB_EINVAL;
    }
    const int pairs = r->rot_dim / 2;
    int64_t sum = 0;
    for (int x = 0; x < r->n_axes; x++) {
        if (r->section[x] < 0) { set_error("%s: section %d is negative", who, x); return OFB_EINVAL; }
        sum += r->section[x];
        if (r->order == OFB_ROPE_DEALT && x && (int64_t)r->section[x] * r->n_axes > pairs + r->n_axes - 1 - x) {
            set_error("%s: section %d (%d pairs) cannot be dealt from %d pairs over %d axes", who, x, r->section[x], pairs, r->n_axes);
            return OFB_EINVAL;
        }
    }
    if (sum != pairs) { set_error("%s: the sections have %lld pairs, rot_dim/2 is %d", who, (long long)sum, pairs); return OFB_EINVAL; }
    a.rot = r->rot_dim;
    // powers by repeated products: with 64 bits of mantissa 127 of them stay
    // within 2^-55 of the frequency, for one powl per call (per_axis: per axis)
    const long double inv_2pi = 0.159154943091895335768883763372514362L;
    int x = 0, left = r->section[0];
    long double f = inv_2pi, step = powl(r->base, -1.0L / (r->per_axis && left ? left : pairs));
    for (int i = 0; i < pairs; i++) {
        if (r->order == OFB_ROPE_BLOCKED) {
            while (!left) {
                left = r->section[++x];
                if (r->per_axis && left) f = inv_2pi, step = powl(r->base, -1.0L / left);
            }
            left--;
            a.axis[i] = (uint8_t)x;
        } else {
            const int y = i % r->n_axes;
            a.axis[i] = (uint8_t)(i / r->n_axes < r->section[y] ? y : 0);
        }
        // whole turns (frequencies above 2 pi) leave no trace at integer positions
        const long double part = f < 1.0L ? f : f - floorl(f);
        a.turns[i] = (uint64_t)(part * 0x1p64L);
        f *= step;
    }
    return OFB_OK;
}

template <typename IO, typename CT> static cudaError_t rope_launch(RopeArgs &a, bool vec, bool adjacent, cudaStream_t s) {
    const int rows = a.H + 2 * a.KVH, threads = vec ? RV_THREADS : RP_THREADS;
    const int64_t per_tok = (int64_t)rows * (vec ? a.d / 16 : a.d - a.rot / 2);
    // one batch of items per thread where a token alone does not give them, at
    // most 8 tokens (2 KB of cosines and sines each), and two CTAs per SM first
    int tpb = (int)(RV_BATCH<IO> * threads / per_tok);
    tpb = tpb < 1 ? 1 : tpb > 8 ? 8 : tpb;
    while (tpb > 1 && (a.T + tpb - 1) / tpb < 2 * sm_count()) tpb--;
    a.tpb = tpb;
    a.rows = fast_div(rows);
    a.page = fast_div(a.page_size ? a.page_size : 1);
    a.per_row = fast_div(vec ? a.d / 16 : 1);
    a.pairs = fast_div(a.rot ? a.rot / 2 : 1);
    a.slots = RV_THREADS / (int)a.per_row.d;
    // few tokens with many rows: several CTAs share a token's rows
    const int groups = (a.T + tpb - 1) / tpb, batches = (tpb * rows + a.slots * RV_BATCH<IO> - 1) / (a.slots * RV_BATCH<IO>);
    a.split = 1;
    while (vec && 2 * a.split <= batches && (int64_t)2 * a.split * groups <= 2 * sm_count()) a.split *= 2;
    // (a.rot is a multiple of 4 for the first kernel)
    const size_t smem = ((size_t)tpb * a.rot + 3) / 4 * 16 + tpb * sizeof(RopeEntry);
    const dim3 grid(groups * a.split), block(threads);
    if (!vec) return launch_pdl(rope_any_kernel<IO, CT>, grid, block, smem, s, a, (int)adjacent);
    if (!a.KVH)
        return adjacent ? launch_pdl(rope_vec_kernel<IO, IO, true, false>, grid, block, smem, s, a)
                        : launch_pdl(rope_vec_kernel<IO, IO, false, false>, grid, block, smem, s, a);
    return adjacent ? launch_pdl(rope_vec_kernel<IO, CT, true, true>, grid, block, smem, s, a)
                    : launch_pdl(rope_vec_kernel<IO, CT, false, true>, grid, block, smem, s, a);
}

static bool row_ok(const void *p, int64_t stride) { return !misaligned(p, 16) && stride % 8 == 0; }

}  // namespace ofb

using namespace ofb;

extern "C" int ofb_rope(const ofb_rope_config *rope, const void *x, int type, int n_tokens, int n_heads, int head_dim,
                        int64_t x_stride, const int32_t *pos, int64_t pos_stride, void *out, int64_t out_stride,
                        void *stream) {
    if (!rope || n_tokens < 0 || n_heads < 1 || n_heads > 65536 || head_dim < 1 || head_dim > 1024 ||
        (n_tokens && (!x || !pos || !out))) {
        set_error("ofb_rope: bad arguments");
        return OFB_EINVAL;
    }
    if (type != OFB_TYPE_F32 && !cache_type(type)) {
        set_error("ofb_rope: type %d is not F32/BF16/F16", type);
        return OFB_EUNSUPPORTED;
    }
    const int64_t width = (int64_t)n_heads * head_dim;
    if ((n_tokens > 1 && (x_stride < width || out_stride < width)) || (rope->n_axes > 1 && pos_stride < n_tokens) ||
        (x == out && n_tokens > 1 && x_stride != out_stride) || misaligned(x, type_size(type)) ||
        misaligned(out, type_size(type)) || misaligned(pos, 4)) {
        set_error("ofb_rope: strides or alignment (x %lld, out %lld, pos %lld)", (long long)x_stride, (long long)out_stride,
                  (long long)pos_stride);
        return OFB_EINVAL;
    }
    if (n_tokens > RP_TOKENS) { set_error("ofb_rope: %d tokens, %d at most", n_tokens, RP_TOKENS); return OFB_ETOOLARGE; }
    RopeArgs a = {};
    int st = rope_tables(rope, head_dim, "ofb_rope", a);
    if (st != OFB_OK) return st;
    if (!n_tokens) return OFB_OK;
    a.T = n_tokens, a.H = n_heads, a.d = head_dim;
    a.q = x, a.q_out = out, a.qs = x_stride, a.qos = out_stride, a.pos = pos, a.pos_stride = pos_stride;
    const bool vec = head_dim % 16 == 0 && a.rot % 16 == 0 && row_ok(x, x_stride) && row_ok(out, out_stride);
    const bool adj = rope->pairing == OFB_ROPE_ADJACENT;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = type == OFB_TYPE_F32    ? rope_launch<float, __nv_bfloat16>(a, vec, adj, s)
                          : type == OFB_TYPE_BF16 ? rope_launch<__nv_bfloat16, __nv_bfloat16>(a, vec, adj, s)
                                                  : rope_launch<__half, __half>(a, vec, adj, s);
    return e == cudaSuccess ? OFB_OK : cuda_status(e, "ofb_rope launch");
}

extern "C" int ofb_rope_append(const ofb_kv_cache *cache, const ofb_rope_config *rope, int type, int n_tokens, int n_heads,
                               const void *q, int64_t q_stride, const void *k, int64_t k_stride, const void *v,
                               int64_t v_stride, const int32_t *pos, int64_t pos_stride, const int32_t *seq,
                               const int32_t *index, const int32_t *number, void *q_out, int64_t q_out_stride,
                               void *stream) {
    int st = check_cache(cache, "ofb_rope_append");
    if (st != OFB_OK) return st;
    if (type != OFB_TYPE_F32 && type != cache->type) {
        set_error("ofb_rope_append: type %d is neither F32 nor the cache's", type);
        return OFB_EUNSUPPORTED;
    }
    if (n_tokens < 0 || n_heads < 0 || n_heads > 65536 ||
        (n_tokens && (!k || !v || !seq || !index || (rope && !pos) || (q && (!q_out || n_heads < 1))))) {
        set_error("ofb_rope_append: bad arguments");
        return OFB_EINVAL;
    }
    const int d = cache->head_dim;
    const int64_t qw = (int64_t)n_heads * d, kw = (int64_t)cache->n_kv_heads * d;
    const size_t ts = type_size(type);
    if ((n_tokens > 1 && ((q && (q_stride < qw || q_out_stride < qw)) || k_stride < kw || v_stride < kw)) ||
        (rope && rope->n_axes > 1 && pos_stride < n_tokens) ||
        (q && q == q_out && n_tokens > 1 && q_stride != q_out_stride) || misaligned(q, ts) || misaligned(q_out, ts) ||
        misaligned(k, ts) || misaligned(v, ts) || misaligned(pos, 4) || misaligned(seq, 4) || misaligned(index, 4) ||
        misaligned(number, 4)) {
        set_error("ofb_rope_append: strides or alignment (q %lld, k %lld, v %lld, q_out %lld, pos %lld)", (long long)q_stride,
                  (long long)k_stride, (long long)v_stride, (long long)q_out_stride, (long long)pos_stride);
        return OFB_EINVAL;
    }
    if (n_tokens > RP_TOKENS) { set_error("ofb_rope_append: %d tokens, %d at most", n_tokens, RP_TOKENS); return OFB_ETOOLARGE; }
    RopeArgs a = {};
    if (rope && (st = rope_tables(rope, d, "ofb_rope_append", a)) != OFB_OK) return st;
    if (!n_tokens) return OFB_OK;
    a.T = n_tokens, a.H = q ? n_heads : 0, a.KVH = cache->n_kv_heads, a.d = d;
    a.n_pages = cache->n_pages, a.page_size = cache->page_size, a.n_seqs = cache->n_seqs, a.max_pages = cache->max_pages;
    a.q = q, a.k = k, a.v = v, a.q_out = q_out, a.ck = cache->k, a.cv = cache->v;
    a.qs = q_stride, a.ks = k_stride, a.vs = v_stride, a.qos = q_out_stride;
    a.page_stride = cache_page_stride(cache), a.pos = pos, a.pos_stride = pos_stride;
    a.seq = seq, a.index = index, a.number = number, a.table = cache->page_table;
    a.weight = cache->weight, a.order = cache->order, a.errors = cache->errors;
    const bool vec = a.rot % 16 == 0 && row_ok(k, k_stride) && row_ok(v, v_stride) &&
                     (!q || (row_ok(q, q_stride) && row_ok(q_out, q_out_stride)));
    const bool adj = rope && rope->pairing == OFB_ROPE_ADJACENT;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool bf = cache->type == OFB_TYPE_BF16;
    const cudaError_t e = type == OFB_TYPE_F32 ? (bf ? rope_launch<float, __nv_bfloat16>(a, vec, adj, s)
                                                     : rope_launch<float, __half>(a, vec, adj, s))
                          : bf                 ? rope_launch<__nv_bfloat16, __nv_bfloat16>(a, vec, adj, s)
                                               : rope_launch<__half, __half>(a, vec, adj, s);
    return e == cudaSuccess ? OFB_OK : cuda_status(e, "ofb_rope_append launch");
}

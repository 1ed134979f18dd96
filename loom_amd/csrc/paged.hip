// paged.hip -- norms and rotation of queries and keys, and the way of keys and
// values into the pages of a paged cache.
//
// A head x of hd values at position p:
//   y = x / sqrt(sum x^2 / hd + eps) * w          (where there is a norm)
//   (a, b) of pair i < rot / 2  ->  (a cos t - b sin t, b cos t + a sin t),
//   t = p * freqs[i]
// The angle is taken in 64 bits, as turns t / 2 pi without their whole part:
// a position of a million leaves an f32 angle no digits below 2^-4.  The rest,
// at most half a turn, is rounded to f32 (off by up to 2^-26 turns, an angle of
// 1e-7) for the library's sine and cosine: results are off by 8e-8 of their size
// in the mean square, 6.5e-8 with both in 64 bits.  Everything else is in f32;
// keys and values are rounded once, to the nearest, on their way into the cache.
//
// Bound by bytes.  Measured: 4096 tokens of 32 and 4 heads of 128 29.8 us (151
// MB, 5.1 TB/s: a large copy runs at 4.8), 4101 tokens with queries into the pages
// 31.1 (160 MB), one token 3.2, a launch.  With 100 values rotated, loaded and
// stored one by one, 67 where 128 take 35, in a graph.  Norm weights as loads of single values
// and pointers indexed by a lane's kind of head took 47; several tokens a work
// group, with loops over their heads, 33 to 35.
#include "runtime.hpp"

#include <type_traits>

namespace lh {

constexpr int RP_THREADS = 256;
constexpr size_t RP_MAX_HD = 256;
typedef float rp_f4 __attribute__((ext_vector_type(4)));
typedef rp_f4 rp_f4u __attribute__((aligned(4))); // at any float
typedef uint16_t rp_u4 __attribute__((ext_vector_type(4)));

struct RopeParams {
    // queries, keys, values (of 0 heads where there are none); out NULL: into the pages
    const float *x[3];
    size_t xs[3];
    float *out[2];
    size_t os[2];
    const float *norm[2];
    int heads[3];
    const int32_t *pos;
    const double *freqs;
    int rot, interleaved;
    float eps;
    int hd;
    size_t n;
    loomhip_pages c;
    const int32_t *lanes;
};

// Pair p's elements of a head.
__device__ __forceinline__ int rp_first(const RopeParams &P, int p) {
    return p < P.rot / 2 && !P.interleaved ? p : 2 * p;
}
__device__ __forceinline__ int rp_second(const RopeParams &P, int p) {
    return p < P.rot / 2 && !P.interleaved ? p + P.rot / 2 : 2 * p + 1;
}

__device__ __forceinline__ uint16_t rp_half(float v, bool bf16) {
    return bf16 ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (_Float16)v);
}

// The row of a token's cache rows that holds position `pos`, in elements; false where there is none.
__device__ __forceinline__ bool rp_slot(const RopeParams &P, size_t t, int pos, size_t &at) {
    const int64_t lane = P.lanes ? (int64_t)P.lanes[t] : (int64_t)t;
    const uint32_t ps = (uint32_t)P.c.page_size, page = (uint32_t)pos / ps;
    if (lane < 0 || lane >= (int64_t)P.c.n_lanes || page >= P.c.table_width)
        return false;
    const int32_t id = P.c.table[(size_t)lane * P.c.table_stride + page];
    if (id < 0 || (size_t)id >= P.c.n_pages)
        return false;
    at = (size_t)id * P.c.page_stride + (size_t)((uint32_t)pos - page * ps) * P.c.row_stride;
    return true;
}

// A work group takes RP_THREADS / GP heads of a token: GP lanes (a power of two, at least hd / 8 of them) a head, each
// four pairs.  The token's cosines and sines are formed once, by a thread a pair, while the heads are on their way.
// VEC: the four pairs are two times four consecutive values (rot a multiple of 8).
template <int GP, bool VEC>
__global__ __launch_bounds__(RP_THREADS) void rope_kernel(RopeParams P) {
    constexpr int PAIRS = GP * 4;
    __shared__ __attribute__((aligned(16))) float cosines[PAIRS], sines[PAIRS];
    const int tid = threadIdx.x, g = tid % GP;
    const size_t t = blockIdx.x;
    const int pos = P.pos[t];
    if (pos < 0) // padding
        return;
    // the group's head: its kind (0 query, 1 key, 2 value) and its number
    const int at = blockIdx.y * (RP_THREADS / GP) + tid / GP;
    const int kind = at < P.heads[0] ? 0 : at < P.heads[0] + P.heads[1] ? 1 : 2;
    const int h = at - (kind > 0 ? P.heads[0] : 0) - (kind > 1 ? P.heads[1] : 0);
    const int p0 = g * 4, half = P.rot / 2;
    const bool mine = g < P.hd / 8 && h < (kind == 0 ? P.heads[0] : kind == 1 ? P.heads[1] : P.heads[2]);
    const bool turn = kind < 2 && p0 < half;
    const bool split = VEC && turn && !P.interleaved; // values p0 .. and p0 + rot / 2 .., not 2 p0 ..
    const bool pairs = VEC || kind == 2;              // in two times four consecutive values
    const int at_a = split ? p0 : 2 * p0, at_b = split ? p0 + half : 2 * p0 + 4;

    rp_f4 va = {0.0f, 0.0f, 0.0f, 0.0f}, vb = va, wa = va, wb = va;
    const float *norm = kind == 0 ? P.norm[0] : kind == 1 ? P.norm[1] : nullptr;
    // f(x), for the group's values in memory: as they lie, or pair by pair
    const auto fetch = [&](const float *x, rp_f4 &a, rp_f4 &b) {
        if (pairs) {
            a = *(const rp_f4u *)(x + at_a);
            b = *(const rp_f4u *)(x + at_b);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                a[e] = x[rp_first(P, p0 + e)];
                b[e] = x[rp_second(P, p0 + e)];
            }
        }
    };
    // four consecutive pairs of neighbours as first and second ones, and back
    const auto part = [&](rp_f4 &a, rp_f4 &b) {
        if (pairs && !split) {
            const rp_f4 x = a, y = b;
            a = rp_f4{x[0], x[2], y[0], y[2]};
            b = rp_f4{x[1], x[3], y[1], y[3]};
        }
    };
    if (mine) {
        const float *x = kind == 0 ? P.x[0] : kind == 1 ? P.x[1] : P.x[2];
        fetch(x + t * (kind == 0 ? P.xs[0] : kind == 1 ? P.xs[1] : P.xs[2]) + (size_t)h * P.hd, va, vb);
        if (norm)
            fetch(norm, wa, wb);
    }
    const bool to_pages = kind && !P.out[1];
    size_t row = 0;
    const bool stored = !to_pages || rp_slot(P, t, pos, row);
    if (tid < half && (int)(blockIdx.y * (RP_THREADS / GP)) < P.heads[0] + P.heads[1]) {
        const double turns = (double)pos * (P.freqs[tid] * 0x1.45f306dc9c883p-3);
        float s, c;
        sincospif((float)(2.0 * (turns - __builtin_rint(turns))), &s, &c);
        cosines[tid] = c, sines[tid] = s;
    }
    __syncthreads();
    rp_f4 a = va, b = vb;
    part(a, b);
    if (norm) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; e++)
            ss += a[e] * a[e] + b[e] * b[e];
        ss += dpp_f<0xB1>(ss, ss);
        ss += dpp_f<0x4E>(ss, ss);
        ss += dpp_f<0x141>(ss, ss);
        if (GP > 8)
            ss += dpp_f<0x140>(ss, ss);
        if (GP > 16)
            ss += __shfl_xor(ss, 16);
        const float r = 1.0f / sqrtf(ss / (float)P.hd + P.eps);
        part(wa, wb);
        a = a * r * wa;
        b = b * r * wb;
    }
    if (turn) {
        const rp_f4 c = *(const rp_f4 *)(cosines + p0), s = *(const rp_f4 *)(sines + p0);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (!VEC && p0 + e >= half) // behind the last rotated pair: not by a cosine of 1, for infinity times 0 is NaN
                break;
            const float u = a[e];
            a[e] = __builtin_fmaf(u, c[e], -(b[e] * s[e]));
            b[e] = __builtin_fmaf(b[e], c[e], u * s[e]);
        }
    }
    if (!mine || !stored)
        return;
    if (pairs && !split) {
        const rp_f4 x = a, y = b;
        a = rp_f4{x[0], y[0], x[1], y[1]};
        b = rp_f4{x[2], y[2], x[3], y[3]};
    }
    if (to_pages) {
        uint16_t *out = (uint16_t *)(kind == 1 ? P.c.k : P.c.v) + row + (size_t)h * P.c.head_stride;
        rp_u4 x, y;
#pragma unroll
        for (int e = 0; e < 4; e++)
            x[e] = rp_half(a[e], P.c.type == LOOMHIP_BF16), y[e] = rp_half(b[e], P.c.type == LOOMHIP_BF16);
        if (pairs) {
            *(rp_u4 *)(out + at_a) = x;
            *(rp_u4 *)(out + at_b) = y;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                out[rp_first(P, p0 + e)] = x[e], out[rp_second(P, p0 + e)] = y[e];
        }
    } else {
        float *out = (kind ? P.out[1] : P.out[0]) + t * (kind ? P.os[1] : P.os[0]) + (size_t)h * P.hd;
        if (pairs) {
            *(rp_f4u *)(out + at_a) = a;
            *(rp_f4u *)(out + at_b) = b;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                out[rp_first(P, p0 + e)] = a[e], out[rp_second(P, p0 + e)] = b[e];
        }
    }
}

static int rope_run(const RopeParams &P, const char *what, void *stream) {
    if (int rc = require_device())
        return rc;
    hipStream_t st = stream_of(stream);
    const auto run = [&](auto gp, auto vec) {
        constexpr int GP = decltype(gp)::value, GROUPS = RP_THREADS / GP;
        const dim3 g(P.n, (P.heads[0] + P.heads[1] + P.heads[2] + GROUPS - 1) / GROUPS);
        hipLaunchKernelGGL((rope_kernel<GP, decltype(vec)::value>), g, dim3(RP_THREADS), 0, st, P);
    };
    const auto sized = [&](auto vec) {
        if (P.hd <= 64)
            run(std::integral_constant<int, 8>{}, vec);
        else if (P.hd <= 128)
            run(std::integral_constant<int, 16>{}, vec);
        else
            run(std::integral_constant<int, 32>{}, vec);
    };
    if (P.rot % 8 == 0)
        sized(std::true_type{});
    else
        sized(std::false_type{});
    note_launch();
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? LOOMHIP_OK : hip_fail(e, what);
}

constexpr size_t RP_MAX_TOKENS = 1 << 23, RP_MAX_HEADS = 4096; // a launch has fewer than 2^32 threads a dimension

// heads of the tokens and where they go (out NULL: into pages)
static int heads_check(const loomhip_heads *s, size_t n, size_t hd, bool out, const char *fn, const char *what) {
    if (!s->x || (out && !s->out))
        return fail(LOOMHIP_ERR_ARG, "%s: %s null", fn, what);
    if (s->n_heads > RP_MAX_HEADS)
        return fail(LOOMHIP_DECLINED, "%s: %zu heads not served", fn, s->n_heads);
    if (n > 1 && (s->x_stride < s->n_heads * hd || (out && s->out_stride < s->n_heads * hd)))
        return fail(LOOMHIP_ERR_ARG, "%s: %s tokens %zu / %zu apart, below %zu heads of %zu", fn, what, s->x_stride,
                    s->out_stride, s->n_heads, hd);
    if (s->x_stride > 0xffffffffu || (out && s->out_stride > 0xffffffffu))
        return fail(LOOMHIP_DECLINED, "%s: %s tokens %zu / %zu apart not served", fn, what, s->x_stride, s->out_stride);
    if (((uintptr_t)s->x | (uintptr_t)s->norm | (out ? (uintptr_t)s->out : 0)) % 4)
        return fail(LOOMHIP_ERR_ARG, "%s: %s not aligned to its elements", fn, what);
    return LOOMHIP_OK;
}
static int rope_check(const loomhip_rope *r, size_t n, size_t hd, const char *fn) {
    if (!r || !r->pos)
        return fail(LOOMHIP_ERR_ARG, "%s: no positions", fn);
    if (hd == 0 || hd % 8 || hd > RP_MAX_HD || n > RP_MAX_TOKENS)
        return fail(LOOMHIP_DECLINED, "%s: %zu tokens, head size %zu not served", fn, n, hd);
    if (r->rot % 2 || r->rot > hd || (r->rot && !r->freqs))
        return fail(LOOMHIP_ERR_ARG, "%s: %zu of %zu values rotated%s", fn, r->rot, hd, r->freqs ? "" : " without frequencies");
    if ((uintptr_t)r->pos % 4 || (uintptr_t)r->freqs % 8)
        return fail(LOOMHIP_ERR_ARG, "%s: positions or frequencies not aligned to their elements", fn);
    return LOOMHIP_OK;
}
// Whether `out` of a shares a value with b's input (other than being it) or output.
static bool heads_meet(const loomhip_heads *a, const loomhip_heads *b, size_t n, size_t hd) {
    const size_t aw = a->n_heads * hd, bw = b->n_heads * hd;
    const bool in_place = a == b && a->out == b->x && (a->out_stride == b->x_stride || n == 1);
    return (!in_place && rows_overlap(a->out, a->out_stride, aw, b->x, b->x_stride, bw, n)) ||
           (a != b && b->out && rows_overlap(a->out, a->out_stride, aw, b->out, b->out_stride, bw, n));
}
static void rope_set(RopeParams &P, const loomhip_rope *r, size_t n, size_t hd) {
    P.pos = r->pos;
    P.freqs = r->freqs;
    P.rot = (int)r->rot;
    P.interleaved = r->interleaved;
    P.eps = r->eps;
    P.hd = (int)hd;
    P.n = n;
}
static void heads_set(RopeParams &P, int kind, const loomhip_heads *s) {
    P.x[kind] = s->x;
    P.xs[kind] = s->x_stride;
    P.heads[kind] = (int)s->n_heads;
    if (kind < 2) {
        P.out[kind] = s->out;
        P.os[kind] = s->out_stride;
        P.norm[kind] = s->norm;
    }
}

// What every call over pages asks of them (paged_attn.hip too).
int pages_check(const loomhip_pages *c, size_t n_kv, size_t hd, const char *fn) {
    if (!c || !c->k || !c->v || !c->table)
        return fail(LOOMHIP_ERR_ARG, "%s: no pages or no table", fn);
    if (c->type != LH_F16 && c->type != LOOMHIP_BF16)
        return fail(LOOMHIP_DECLINED, "%s: cache type %d not served", fn, c->type);
    if (c->n_pages == 0 || c->page_size == 0 || c->n_lanes == 0 || c->table_width == 0)
        return fail(LOOMHIP_ERR_ARG, "%s: %zu pages of %zu rows, a table of %zu x %zu", fn, c->n_pages, c->page_size,
                    c->n_lanes, c->table_width);
    if (c->n_lanes > 1 && c->table_stride < c->table_width)
        return fail(LOOMHIP_ERR_ARG, "%s: table rows %zu apart, below their %zu pages", fn, c->table_stride, c->table_width);
    // rows and pages are counted in 31 bits, a page pool's 16-byte pieces in 32
    if (c->n_pages > 0x7fffffff || c->page_size > 0x7fffffff || c->table_width > 0x7fffffff ||
        c->page_size * c->table_width > 0x7fffffff || c->n_lanes > 0x7fffffff || c->table_stride > 0xffffffffu)
        return fail(LOOMHIP_DECLINED, "%s: %zu pages of %zu rows, a table of %zu x %zu not served", fn, c->n_pages,
                    c->page_size, c->n_lanes, c->table_width);
    constexpr size_t MOST = (size_t)1 << 35; // elements
    if (c->page_stride >= MOST || c->row_stride >= MOST || c->head_stride >= MOST ||
        (c->n_pages > 1 && c->page_stride > MOST / (c->n_pages - 1)) ||
        (c->page_size > 1 && c->row_stride > MOST / (c->page_size - 1)) ||
        (n_kv > 1 && c->head_stride > MOST / (n_kv - 1)) ||
        (c->n_pages - 1) * c->page_stride + (c->page_size - 1) * c->row_stride >= MOST)
        return fail(LOOMHIP_DECLINED, "%s: a pool of more than 2^35 values not served", fn);
    if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16 || (c->n_pages > 1 && c->page_stride % 8) ||
        (c->page_size > 1 && c->row_stride % 8) || (n_kv > 1 && c->head_stride % 8))
        return fail(LOOMHIP_DECLINED, "%s: rows of the pages not at multiples of 16 bytes", fn);
    // the rows of all heads apart: rows of one head at least a head apart, whichever of the strides is the smallest
    if ((c->page_size > 1 && c->row_stride < hd) || (n_kv > 1 && c->head_stride < hd) ||
        (c->n_pages > 1 && c->page_stride < hd))
        return fail(LOOMHIP_ERR_ARG, "%s: rows, heads or pages closer than a head of %zu", fn, hd);
    if ((uintptr_t)c->table % 4)
        return fail(LOOMHIP_ERR_ARG, "%s: the table is not aligned to its elements", fn);
    return LOOMHIP_OK;
}

} // namespace lh

using namespace lh;

extern "C" {

int loomhip_qk_norm_rope_dev(const loomhip_heads *q, const loomhip_heads *k, const loomhip_rope *r, size_t n,
                             size_t head_dim, void *stream) {
    const char *fn = "qk_norm_rope";
    if (n == 0)
        return LOOMHIP_OK;
    if (!q || q->n_heads == 0)
        return fail(LOOMHIP_ERR_ARG, "%s: no heads", fn);
    const bool keys = k && k->n_heads;
    if (int rc = rope_check(r, n, head_dim, fn))
        return rc;
    if (int rc = heads_check(q, n, head_dim, true, fn, "q"))
        return rc;
    if (keys)
        if (int rc = heads_check(k, n, head_dim, true, fn, "k"))
            return rc;
    if (heads_meet(q, q, n, head_dim) || (keys && (heads_meet(k, k, n, head_dim) || heads_meet(q, k, n, head_dim) ||
                                                   heads_meet(k, q, n, head_dim))))
        return fail(LOOMHIP_ERR_ARG, "%s: an output overlaps an input without being it, or the other output", fn);
    RopeParams P = {};
    rope_set(P, r, n, head_dim);
    heads_set(P, 0, q);
    if (keys)
        heads_set(P, 1, k);
    return rope_run(P, "qk_norm_rope launch", stream);
}

int loomhip_paged_append_dev(const loomhip_pages *c, const loomhip_heads *q, const loomhip_heads *k, const float *v,
                             size_t v_stride, const int32_t *lanes, const loomhip_rope *r, size_t n, size_t head_dim,
                             void *stream) {
    const char *fn = "paged_append";
    if (n == 0)
        return LOOMHIP_OK;
    if (!k || k->n_heads == 0 || !v)
        return fail(LOOMHIP_ERR_ARG, "%s: no keys or values", fn);
    const bool queries = q && q->n_heads;
    const loomhip_heads vh = {v, v_stride, nullptr, 0, nullptr, k->n_heads};
    if (int rc = rope_check(r, n, head_dim, fn))
        return rc;
    if (int rc = heads_check(k, n, head_dim, false, fn, "k"))
        return rc;
    if (int rc = heads_check(&vh, n, head_dim, false, fn, "v"))
        return rc;
    if (queries)
        if (int rc = heads_check(q, n, head_dim, true, fn, "q"))
            return rc;
    if (int rc = pages_check(c, k->n_heads, head_dim, fn))
        return rc;
    if ((uintptr_t)lanes % 4)
        return fail(LOOMHIP_ERR_ARG, "%s: lanes not aligned to their elements", fn);
    if (!lanes && n > c->n_lanes)
        return fail(LOOMHIP_ERR_ARG, "%s: %zu tokens without their lanes, a table of %zu", fn, n, c->n_lanes);
    if (c->k == c->v) // attention may read one pool as both
        return fail(LOOMHIP_ERR_ARG, "%s: keys and values go to one pool", fn);
    RopeParams P = {};
    rope_set(P, r, n, head_dim);
    heads_set(P, 1, k);
    P.out[1] = nullptr;
    heads_set(P, 2, &vh);
    if (queries) {
        loomhip_heads in_k = *k;
        in_k.out = nullptr;
        if (heads_meet(q, q, n, head_dim) || heads_meet(q, &in_k, n, head_dim) || heads_meet(q, &vh, n, head_dim))
            return fail(LOOMHIP_ERR_ARG, "%s: q's output overlaps an input without being q", fn);
        heads_set(P, 0, q);
    }
    P.c = *c;
    P.lanes = lanes;
    return rope_run(P, "paged_append launch", stream);
}

} // extern "C"

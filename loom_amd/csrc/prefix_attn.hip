// prefix_attn.hip -- attention of a batch that shares a long prefix: every
// lane's query rows over one prefix cache, joined with the lane's own rows.
#include "runtime.hpp"

namespace lh {

constexpr int PA_THREADS = 256;
constexpr int PA_MAX_HD = 256;

struct PrefixAttnParams {
    loomhip_kv_rows pre, own;
    const float *q;
    const int32_t *own_len, *q_len;
    int n, n_q, n_heads, n_kv, hd;
    float scale;
    float *out;
};

__device__ __forceinline__ int pa_clamp(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// One work group per (head, query token, lane): each wave takes every fourth
// cache row with a running maximum and sum, the four are merged at the end.
__global__ __launch_bounds__(PA_THREADS) void prefix_attn_kernel(PrefixAttnParams P) {
    constexpr int W = PA_THREADS / 64, DPL = PA_MAX_HD / 64;
    __shared__ float sm[W], sl[W], so[W][PA_MAX_HD];
    const int h = blockIdx.x, j = blockIdx.y, i = blockIdx.z;
    const int own_rows = (int)P.own.rows;
    const int L = P.q_len ? pa_clamp(P.q_len[i], 0, P.n_q) : P.n_q;
    if (j >= L)
        return;
    const int len = own_rows ? pa_clamp(P.own_len[i], 0, own_rows) : 0;
    const int seen = len - L + 1 + j < 0 || !own_rows ? 0 : len - L + 1 + j;
    const size_t row = ((size_t)i * P.n_q + j) * P.n_heads + h;
    const int kvh = h / (P.n_heads / P.n_kv);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float q[DPL], o[DPL], m = -__builtin_inff(), l = 0.0f;
    for (int d = 0; d < DPL; d++) {
        q[d] = d * 64 + lane < P.hd ? P.q[row * P.hd + d * 64 + lane] * P.scale : 0.0f;
        o[d] = 0.0f;
    }
    const size_t T = P.pre.rows + seen;
    for (size_t t = wave; t < T; t += W) {
        const bool shared = t < P.pre.rows;
        const loomhip_kv_rows &R = shared ? P.pre : P.own;
        const size_t at = (shared ? t * R.row_stride : (size_t)i * R.lane_stride + (t - P.pre.rows) * R.row_stride) +
                          (size_t)kvh * R.head_stride;
        float s = 0.0f;
        for (int d = 0; d < DPL; d++)
            if (d * 64 + lane < P.hd)
                s = __builtin_fmaf(q[d], half_bits_to_float(R.k[at + d * 64 + lane]), s);
        for (int x = 1; x < 64; x *= 2)
            s += __shfl_xor(s, x);
        const float m2 = fmaxf(m, s), c = m == m2 ? 1.0f : __expf(m - m2), p = __expf(s - m2);
        m = m2;
        l = l * c + p;
        for (int d = 0; d < DPL; d++)
            if (d * 64 + lane < P.hd)
                o[d] = o[d] * c + p * half_bits_to_float(R.v[at + d * 64 + lane]);
    }
    if (lane == 0)
        sm[wave] = m, sl[wave] = l;
    for (int d = 0; d < DPL; d++)
        so[wave][d * 64 + lane] = o[d];
    __syncthreads();
    if (tid >= P.hd)
        return;
    float M = sm[0];
    for (int w = 1; w < W; w++)
        M = fmaxf(M, sm[w]);
    float sum = 0.0f, v = 0.0f;
    for (int w = 0; w < W; w++)
        if (sm[w] != -__builtin_inff() || sl[w] != 0.0f) {
            const float c = __expf(sm[w] - M);
            sum += sl[w] * c;
            v += so[w][tid] * c;
        }
    P.out[row * P.hd + tid] = T ? v / sum : 0.0f;
}

} // namespace lh

using namespace lh;

static int kv_rows_check(const loomhip_kv_rows *r, size_t n_kv, size_t hd, bool lanes, const char *what) {
    if (!r || r->rows == 0)
        return LOOMHIP_OK;
    if (!r->k || !r->v)
        return fail(LOOMHIP_ERR_ARG, "prefix_attn: %s has no keys or values", what);
    if (r->rows > 0x3fffffff)
        return fail(LOOMHIP_DECLINED, "prefix_attn: %zu %s rows not served", r->rows, what);
    if (r->row_stride < hd && r->rows > 1)
        return fail(LOOMHIP_ERR_ARG, "prefix_attn: %s row stride %zu below a head", what, r->row_stride);
    if ((uintptr_t)r->k % 16 || (uintptr_t)r->v % 16 || r->row_stride % 8 || r->head_stride % 8 ||
        (lanes && r->lane_stride % 8))
        return fail(LOOMHIP_DECLINED, "prefix_attn: %s rows not at multiples of 16 bytes", what);
    return LOOMHIP_OK;
}

extern "C" {

size_t loomhip_prefix_attn_ws(size_t prefix_rows, size_t own_rows, size_t n, size_t n_q, size_t n_heads,
                              size_t n_kv_heads, size_t head_dim) {
    return 0;
}

int loomhip_prefix_attn_dev(const loomhip_kv_rows *prefix, const loomhip_kv_rows *own, const float *q,
                            const int32_t *own_len, const int32_t *q_len, size_t n, size_t n_q, size_t n_heads,
                            size_t n_kv_heads, size_t head_dim, float scale, float *out, void *ws, size_t ws_bytes,
                            void *stream) {
    if (n == 0 || n_q == 0)
        return LOOMHIP_OK;
    if (!q || !out || n_heads == 0 || n_kv_heads == 0 || n_heads % n_kv_heads)
        return fail(LOOMHIP_ERR_ARG, "prefix_attn: null argument, or %zu heads over %zu key heads", n_heads, n_kv_heads);
    if (head_dim == 0 || head_dim % 8 || head_dim > PA_MAX_HD)
        return fail(LOOMHIP_DECLINED, "prefix_attn: head size %zu not served", head_dim);
    if (n > 65535 || n_q > 4096 || n_heads > 65535)
        return fail(LOOMHIP_DECLINED, "prefix_attn: %zu lanes of %zu tokens, %zu heads not served", n, n_q, n_heads);
    if (int rc = kv_rows_check(prefix, n_kv_heads, head_dim, false, "prefix"))
        return rc;
    if (int rc = kv_rows_check(own, n_kv_heads, head_dim, true, "own"))
        return rc;
    if (own && own->rows && !own_len)
        return fail(LOOMHIP_ERR_ARG, "prefix_attn: own rows without their lengths");
    if ((uintptr_t)q % 16 || (uintptr_t)out % 16)
        return fail(LOOMHIP_DECLINED, "prefix_attn: q or out not at a multiple of 16 bytes");
    if (int rc = require_device())
        return rc;
    PrefixAttnParams P = {};
    if (prefix)
        P.pre = *prefix;
    if (own)
        P.own = *own;
    P.q = q;
    P.own_len = own_len;
    P.q_len = q_len;
    P.n = (int)n;
    P.n_q = (int)n_q;
    P.n_heads = (int)n_heads;
    P.n_kv = (int)n_kv_heads;
    P.hd = (int)head_dim;
    P.scale = scale;
    P.out = out;
    hipStream_t st = stream_of(stream);
    hipLaunchKernelGGL(prefix_attn_kernel, dim3(n_heads, n_q, n), dim3(PA_THREADS), 0, st, P);
    note_launch();
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? LOOMHIP_OK : hip_fail(e, "prefix_attn launch");
}

} // extern "C"

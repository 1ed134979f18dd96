// sampling.hip -- from logits to tokens for a batched serving step: token
// probabilities at a temperature, and the verification of drafted tokens
// against the target's probabilities from given random numbers.
#include "runtime.hpp"

namespace lh {

// The work groups a row of `vocab` values is split over: enough that the
// whole launch fills the chip, no more than SPLIT_MAX, none with less than
// SPLIT_MIN values.
constexpr int SMP_THREADS = 256;
constexpr int SPLIT_MAX = 64;
constexpr size_t SPLIT_MIN = 2048;
constexpr size_t SPLIT_GROUPS = 1024;

static int row_splits(size_t rows, size_t vocab) {
    size_t s = (SPLIT_GROUPS + rows - 1) / rows;
    const size_t most = (vocab + SPLIT_MIN - 1) / SPLIT_MIN;
    s = s > most ? most : s;
    return (int)(s > SPLIT_MAX ? SPLIT_MAX : s < 1 ? 1 : s);
}
// Values per split, a multiple of 4 so that splits of aligned rows start aligned.
static size_t split_len(size_t vocab, int splits) { return ((vocab + splits - 1) / splits + 3) / 4 * 4; }

// ---- token probabilities -------------------------------------------------------
// p_v = exp((x_v - m) / T) / sum_w exp((x_w - m) / T), m = max x.  Two launches:
// each (row, split) reduces its values to (max, sum of exponentials, first
// index of the max); then each (row, split) merges the row's records and
// writes its probabilities.  T not positive, NaN or so small that 1/T
// passes f32: 1 at the first maximum.
struct ProbRec {
    float m, l;
    int32_t at;
    int32_t pad;
};

// exp((x - m) / T) with c = 1/T * log2 e split into a float and its remainder,
// so that the exponent's rounding does not grow with |x - m| / T.
__device__ __forceinline__ float exp_scaled(float d, float c_hi, float c_lo) {
    const float h = d * c_hi;
    const float r = __builtin_fmaf(d, c_lo, __builtin_fmaf(d, c_hi, -h));
    const float e = __builtin_amdgcn_exp2f(h);
    // d = -inf: h = -inf, r = NaN, e = 0
    return h > -150.0f || h != h ? __builtin_fmaf(e, r * 0.69314718f, e) : 0.0f;
}

struct ProbScale {
    float hi, lo;
    bool greedy;
};
__device__ __forceinline__ ProbScale prob_scale(const float *temperature, size_t row) {
    const float t = temperature ? temperature[row] : 1.0f;
    const double c = 0x1.71547652b82fep+0 / (double)t;
    const float hi = (float)c;
    return {hi, (float)(c - (double)hi), !(t > 0.0f) || !(hi < __builtin_inff())};
}

__device__ __forceinline__ void max_first(float &m, int &at, float m2, int at2) {
    // the larger value; of equal ones the lower index; a NaN stays
    const bool take = m2 > m || (m2 == m && at2 < at) || (m2 != m2 && (m == m || at2 < at));
    m = take ? m2 : m;
    at = take ? at2 : at;
}

__global__ __launch_bounds__(SMP_THREADS) void probs_reduce_kernel(const float *__restrict__ logits, size_t vocab,
                                                                   size_t stride, const float *__restrict__ temperature,
                                                                   size_t len, ProbRec *__restrict__ rec) {
    __shared__ float sm[SMP_THREADS / 64], sl[SMP_THREADS / 64];
    __shared__ int sa[SMP_THREADS / 64];
    const size_t row = blockIdx.y;
    const float *x = logits + row * stride;
    const size_t v0 = blockIdx.x * len, v1 = v0 + len < vocab ? v0 + len : vocab;
    const ProbScale sc = prob_scale(temperature, row);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float m = -__builtin_inff();
    int at = 0x7fffffff;
    for (size_t v = v0 + tid; v < v1; v += SMP_THREADS)
        max_first(m, at, x[v], (int)v);
    for (int o = 1; o < 64; o *= 2)
        max_first(m, at, __shfl_xor(m, o), __shfl_xor(at, o));
    if (lane == 0)
        sm[wave] = m, sa[wave] = at;
    __syncthreads();
    m = sm[0], at = sa[0];
    for (int w = 1; w < SMP_THREADS / 64; w++)
        max_first(m, at, sm[w], sa[w]);
    float l = 0.0f;
    if (m != -__builtin_inff())
        for (size_t v = v0 + tid; v < v1; v += SMP_THREADS)
            l += exp_scaled(x[v] - m, sc.hi, sc.lo);
    for (int o = 1; o < 64; o *= 2)
        l += __shfl_xor(l, o);
    if (lane == 0)
        sl[wave] = l;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < SMP_THREADS / 64; w++)
            l += sl[w];
        rec[row * gridDim.x + blockIdx.x] = {m, l, at, 0};
    }
}

__global__ __launch_bounds__(SMP_THREADS) void probs_write_kernel(const float *__restrict__ logits, size_t vocab,
                                                                  size_t stride, const float *__restrict__ temperature,
                                                                  size_t len, const ProbRec *__restrict__ rec,
                                                                  float *__restrict__ probs, size_t out_stride) {
    const size_t row = blockIdx.y;
    const float *x = logits + row * stride;
    float *p = probs + row * out_stride;
    const size_t v0 = blockIdx.x * len, v1 = v0 + len < vocab ? v0 + len : vocab;
    const ProbScale sc = prob_scale(temperature, row);
    const int tid = threadIdx.x, lane = tid & 63, splits = gridDim.x;
    ProbRec r = {-__builtin_inff(), 0.0f, 0x7fffffff, 0};
    if (lane < splits)
        r = rec[row * splits + lane];
    float m = r.m;
    int at = r.at;
    for (int o = 1; o < 64; o *= 2)
        max_first(m, at, __shfl_xor(m, o), __shfl_xor(at, o));
    if (sc.greedy) {
        for (size_t v = v0 + tid; v < v1; v += SMP_THREADS)
            p[v] = v == (size_t)at ? 1.0f : 0.0f;
        return;
    }
    float l = r.m == -__builtin_inff() ? 0.0f : r.l * exp_scaled(r.m - m, sc.hi, sc.lo);
    for (int o = 1; o < 64; o *= 2)
        l += __shfl_xor(l, o);
    const float inv = 1.0f / l;
    const bool none = m == -__builtin_inff(); // every logit is -inf: no token has a probability
    for (size_t v = v0 + tid; v < v1; v += SMP_THREADS)
        p[v] = none ? 0.0f : exp_scaled(x[v] - m, sc.hi, sc.lo) * inv;
}

// ---- verification of drafted tokens ----------------------------------------------
// Lane i's drafted token j (x_j, drawn from q_j) is accepted while u_j * q_j(x_j) <
// p_j(x_j); after the first refusal, at row r, the next token comes from
// max(p_r - q_r, 0), after none from p_nd, by the inverse of the running sum
// at a given number u: the lowest v with c_v > u * c_last.  The products and
// the sums are in 64 bits: they decide a whole number.  Two launches: each
// (lane, split) finds r and sums its values; then one work group per lane
// scans the split sums and the one split that holds the token.
struct VerifyParams {
    const float *target, *draft; // [n][k+1][vocab], [n][k][vocab] or null
    const int32_t *tok, *n_draft;
    const float *u_accept, *u_sample;
    size_t n, k, vocab;
    size_t len;
    int splits;
    double *sums; // [n][splits][2]: of max(p - q, 0) and of p
    int32_t *out; // [n][k+1]
    int32_t *accepted;
};

// What counts as a probability: a positive finite number, anything else as 0.
__device__ __forceinline__ float as_prob(float p) { return p > 0.0f && p < __builtin_inff() ? p : 0.0f; }

// The drafted tokens of a lane and how many of them are accepted, by the first wave's lanes.
__device__ __forceinline__ int verify_accepted(const VerifyParams &P, size_t i, int nd) {
    const int lane = threadIdx.x & 63;
    int acc = 0;
    for (int j0 = 0; j0 < nd; j0 += 64) { // tokens j0 .. j0 + 63, a lane each
        const int j = j0 + lane;
        bool ok = true;
        if (j < nd) {
            const int64_t x = P.tok[i * P.k + j];
            ok = x >= 0 && x < (int64_t)P.vocab;
            if (ok) {
                const float p = as_prob(P.target[(i * (P.k + 1) + j) * P.vocab + x]);
                const float q = P.draft ? as_prob(P.draft[(i * P.k + j) * P.vocab + x]) : 1.0f;
                ok = (double)P.u_accept[i * P.k + j] * (double)q < (double)p;
            }
        }
        const unsigned long long bad = __ballot(!ok);
        if (bad)
            return j0 + __builtin_ctzll(bad);
        acc = j0 + 64;
    }
    return nd < acc ? nd : acc;
}

__device__ __forceinline__ int verify_nd(const VerifyParams &P, size_t i) {
    const int nd = P.n_draft ? P.n_draft[i] : (int)P.k;
    return nd < 0 ? 0 : nd > (int)P.k ? (int)P.k : nd;
}

// The row the next token comes from: p, q (null where every draft was accepted or the
// drafter gave no probabilities) and the token whose probability is taken out (-1: none).
struct VerifyRow {
    const float *p, *q;
    int64_t out;
};
__device__ __forceinline__ VerifyRow verify_row(const VerifyParams &P, size_t i, int nd, int acc) {
    VerifyRow r = {P.target + (i * (P.k + 1) + acc) * P.vocab, nullptr, -1};
    if (acc < nd) {
        if (P.draft)
            r.q = P.draft + (i * P.k + acc) * P.vocab;
        else
            r.out = P.tok[i * P.k + acc];
    }
    return r;
}
__device__ __forceinline__ double residual(const VerifyRow &r, size_t v, float p) {
    if (r.q) {
        const double d = (double)p - (double)as_prob(r.q[v]);
        return d > 0.0 ? d : 0.0;
    }
    return (int64_t)v == r.out ? 0.0 : (double)p;
}

__device__ __forceinline__ double wave_sum_f64(double v) {
    for (int o = 1; o < 64; o *= 2)
        v += __shfl_xor(v, o);
    return v;
}

__global__ __launch_bounds__(SMP_THREADS) void verify_sum_kernel(VerifyParams P) {
    __shared__ double sd[SMP_THREADS / 64], sp[SMP_THREADS / 64];
    const size_t i = blockIdx.y;
    const int nd = verify_nd(P, i), acc = verify_accepted(P, i, nd);
    const VerifyRow r = verify_row(P, i, nd, acc);
    const size_t v0 = blockIdx.x * P.len, v1 = v0 + P.len < P.vocab ? v0 + P.len : P.vocab;
    double d = 0.0, all = 0.0;
    for (size_t v = v0 + threadIdx.x; v < v1; v += SMP_THREADS) {
        const float p = as_prob(r.p[v]);
        d += residual(r, v, p);
        all += (double)p;
    }
    d = wave_sum_f64(d);
    all = wave_sum_f64(all);
    if ((threadIdx.x & 63) == 0)
        sd[threadIdx.x >> 6] = d, sp[threadIdx.x >> 6] = all;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < SMP_THREADS / 64; w++)
            d += sd[w], all += sp[w];
        double *o = P.sums + (i * P.splits + blockIdx.x) * 2;
        o[0] = d, o[1] = all;
    }
}

__global__ __launch_bounds__(SMP_THREADS) void verify_pick_kernel(VerifyParams P) {
    constexpr int W = SMP_THREADS / 64;
    __shared__ double sw[W];
    __shared__ int s_found[W], s_last[W];
    const size_t i = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int nd = verify_nd(P, i), acc = verify_accepted(P, i, nd);
    VerifyRow r = verify_row(P, i, nd, acc);
    // the running sum at each split's end (splits <= 64: a lane each)
    const double *s = P.sums + i * P.splits * 2;
    double d = lane < P.splits ? s[2 * lane] : 0.0;
    if (!(wave_sum_f64(d) > 0.0)) { // p nowhere above q: the target's own row
        d = lane < P.splits ? s[2 * lane + 1] : 0.0;
        r.q = nullptr;
        r.out = -1;
    }
    double c = d;
    for (int o = 1; o < 64; o *= 2) {
        const double up = __shfl_up(c, o);
        c += lane >= o ? up : 0.0;
    }
    const double total = __shfl(c, 63);
    const double at = fmax((double)P.u_sample[i] * total, 0.0); // NaN: 0
    int32_t *out = P.out + i * (P.k + 1);
    if (tid == 0)
        P.accepted[i] = acc;
    for (int j = tid; j <= (int)P.k; j += SMP_THREADS)
        if (j != acc)
            out[j] = j < acc ? P.tok[i * P.k + j] : -1;
    if (!(total > 0.0)) { // nothing to draw from
        if (tid == 0)
            out[acc] = -1;
        return;
    }
    // the split that holds the token: the first whose end passes `at`, else the last with anything in it
    const unsigned long long past = __ballot(c > at && d > 0.0), some = __ballot(d > 0.0);
    const int sp = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
    double run = __shfl(c, sp) - __shfl(d, sp); // what comes before the split
    if (sp > 0) // the same sum that the split before it ends with
        run = __shfl(c, sp - 1);
    else
        run = 0.0;
    const size_t v0 = sp * P.len, v1 = v0 + P.len < P.vocab ? v0 + P.len : P.vocab;
    int last = -1; // the last value so far with a probability, for a number that no sum passes
    for (size_t b = v0; b < v1; b += SMP_THREADS) {
        const size_t v = b + tid;
        const double e = v < v1 ? residual(r, v, as_prob(r.p[v])) : 0.0;
        double sum = e;
        for (int o = 1; o < 64; o *= 2) {
            const double up = __shfl_up(sum, o);
            sum += lane >= o ? up : 0.0;
        }
        if (lane == 63)
            sw[wave] = sum;
        __syncthreads();
        double before = run;
        for (int w = 0; w < W; w++) {
            if (w == wave)
                sum += before;
            before += sw[w];
        }
        run = before;
        const unsigned long long hit = __ballot(e > 0.0 && sum > at), any = __ballot(e > 0.0);
        if (lane == 0) {
            s_found[wave] = hit ? __builtin_ctzll(hit) : -1;
            s_last[wave] = any ? 63 - __builtin_clzll(any) : -1;
        }
        __syncthreads();
        int found = -1;
        for (int w = W - 1; w >= 0; w--)
            found = s_found[w] >= 0 ? w * 64 + s_found[w] : found;
        for (int w = 0; w < W; w++)
            last = s_last[w] >= 0 ? (int)(b + w * 64 + s_last[w]) : last;
        if (found >= 0) {
            if (tid == 0)
                out[acc] = (int32_t)(b + found);
            return;
        }
        __syncthreads();
    }
    if (tid == 0)
        out[acc] = last;
}

} // namespace lh

using namespace lh;

extern "C" {

size_t loomhip_token_probs_ws(size_t n, size_t vocab) {
    return n && vocab ? n * row_splits(n, vocab) * sizeof(ProbRec) : 0;
}

int loomhip_token_probs_dev(const float *logits, size_t n, size_t vocab, size_t stride, const float *temperature,
                            float *probs, size_t out_stride, void *ws, size_t ws_bytes, void *stream) {
    if (n == 0)
        return LOOMHIP_OK;
    if (!logits || !probs || vocab == 0)
        return fail(LOOMHIP_ERR_ARG, "token_probs: null argument or no vocabulary");
    if (vocab > 0x7fffffff || n > 65535)
        return fail(LOOMHIP_DECLINED, "token_probs: %zu rows of %zu not served", n, vocab);
    if (stride < vocab || out_stride < vocab)
        return fail(LOOMHIP_ERR_ARG, "token_probs: row stride %zu / %zu below %zu values", stride, out_stride, vocab);
    if (!ws || ws_bytes < loomhip_token_probs_ws(n, vocab) || (uintptr_t)ws % 16)
        return fail(LOOMHIP_ERR_ARG, "token_probs: the workspace takes %zu bytes at a multiple of 16, got %zu",
                    loomhip_token_probs_ws(n, vocab), ws_bytes);
    if (int rc = require_device())
        return rc;
    hipStream_t st = stream_of(stream);
    const int splits = row_splits(n, vocab);
    const size_t len = split_len(vocab, splits);
    ProbRec *rec = (ProbRec *)ws;
    hipLaunchKernelGGL(probs_reduce_kernel, dim3(splits, n), dim3(SMP_THREADS), 0, st, logits, vocab, stride,
                       temperature, len, rec);
    hipLaunchKernelGGL(probs_write_kernel, dim3(splits, n), dim3(SMP_THREADS), 0, st, logits, vocab, stride,
                       temperature, len, rec, probs, out_stride);
    note_launch();
    note_launch();
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? LOOMHIP_OK : hip_fail(e, "token_probs launch");
}

size_t loomhip_verify_drafts_ws(size_t n, size_t vocab) {
    return n && vocab ? n * row_splits(n, vocab) * 2 * sizeof(double) : 0;
}

int loomhip_verify_drafts_dev(const float *target_probs, const float *draft_probs, const int32_t *draft_tokens,
                              const int32_t *n_draft, const float *u_accept, const float *u_sample, size_t n, size_t k,
                              size_t vocab, int32_t *tokens_out, int32_t *n_accepted, void *ws, size_t ws_bytes,
                              void *stream) {
    if (n == 0)
        return LOOMHIP_OK;
    if (!target_probs || !u_sample || !tokens_out || !n_accepted || vocab == 0 ||
        (k && (!draft_tokens || !u_accept)))
        return fail(LOOMHIP_ERR_ARG, "verify_drafts: null argument or no vocabulary");
    if (vocab > 0x7fffffff || n > 65535 || k > 4096)
        return fail(LOOMHIP_DECLINED, "verify_drafts: %zu lanes of %zu drafts over %zu values not served", n, k, vocab);
    if (!ws || ws_bytes < loomhip_verify_drafts_ws(n, vocab) || (uintptr_t)ws % 16)
        return fail(LOOMHIP_ERR_ARG, "verify_drafts: the workspace takes %zu bytes at a multiple of 16, got %zu",
                    loomhip_verify_drafts_ws(n, vocab), ws_bytes);
    if (int rc = require_device())
        return rc;
    hipStream_t st = stream_of(stream);
    VerifyParams P;
    P.target = target_probs;
    P.draft = k ? draft_probs : nullptr;
    P.tok = draft_tokens;
    P.n_draft = n_draft;
    P.u_accept = u_accept;
    P.u_sample = u_sample;
    P.n = n;
    P.k = k;
    P.vocab = vocab;
    P.splits = row_splits(n, vocab);
    P.len = split_len(vocab, P.splits);
    P.sums = (double *)ws;
    P.out = tokens_out;
    P.accepted = n_accepted;
    hipLaunchKernelGGL(verify_sum_kernel, dim3(P.splits, n), dim3(SMP_THREADS), 0, st, P);
    hipLaunchKernelGGL(verify_pick_kernel, dim3(n), dim3(SMP_THREADS), 0, st, P);
    note_launch();
    note_launch();
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? LOOMHIP_OK : hip_fail(e, "verify_drafts launch");
}

} // extern "C"

// logprobs.hip -- log probabilities of given tokens, the rows' entropy and
// their likeliest alternatives.
//
//   m = max x,  S = sum e_v,  Z = sum e_v z_v,  z = (x - m) / T,  e = exp z
//   lp_v = z_v - log S,  entropy = log S - Z / S
//
// in one reading of the row.  The `top` largest are found in the registers that
// hold it: a wave's k-th largest of its lanes' maxima is a bound that k values
// reach, so no value below the largest such bound of the work group's waves is
// among the k; the few that reach it are collected in LDS and each counts
// those before it.  Where too many do (values arranged so that a few threads
// hold them all), the k are picked one after the other.
// A row that a work group can hold takes one launch; of a longer one each part
// leaves (m, S, Z) and its own k, which a second launch joins.
#include "sampling.hpp"

#include <type_traits>

namespace lh {

constexpr int LP_MAX_TOP = 32;
constexpr int LP_LIST = 1024;      // values collected at most
constexpr int LP_JOIN_N = 16;      // entries a thread joins
constexpr size_t LP_JOIN = SMP_THREADS * LP_JOIN_N; // a row's parts times top at most
constexpr size_t LP_ROW = 32768;   // one launch up to this row
constexpr size_t LP_MAX_VOCAB = LP_JOIN / LP_MAX_TOP * SMP_THREADS * 64;

struct LpRec {
    float m, s, z;
    int32_t at; // the first maximum
};
struct LpTop {
    float x;
    int32_t id; // -1: none
};
struct LogprobParams {
    const float *logits;
    size_t vocab, stride;
    const int32_t *tokens;
    const float *temperature;
    int top, splits;
    float *lp, *entropy;
    int32_t *top_ids;
    float *top_lp;
    LpRec *rec;  // [n][splits]
    LpTop *list; // [n][splits][top]
};

// Numbers in their order as unsigned ones (both zeros the same), none of them 0.
__device__ __forceinline__ uint32_t lp_order(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float lp_value(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
// A value's key: the larger one is the better, of equal values the one of the lower index; 0 is no value.
__device__ __forceinline__ uint64_t lp_key(float x, int id) { return (uint64_t)lp_order(x) << 32 | (uint32_t)~id; }

template <int THREADS>
struct LpShared {
    static constexpr int W = THREADS / 64;
    float m[W], s[W], z[W];
    int at[W];
    uint64_t key[W];
    int count;
    __attribute__((aligned(16))) uint64_t list[LP_LIST + 2];
    LpTop best[LP_MAX_TOP];
};

// The k best of the work group's values (x(j) with index id(j), j < N, of every thread; NaN and indices from `end` on
// are none) into sh.best, in order.
template <int THREADS, int N, class X, class Id>
__device__ __forceinline__ void lp_select(int k, X x, Id id, int end, LpShared<THREADS> &sh) {
    constexpr int W = THREADS / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const auto here = [&](int j) { return x(j) == x(j) && id(j) < end; };
    float mx = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < N; j++)
        mx = fmaxf(mx, x(j));
    bool any = mx > -__builtin_inff();
    if (!any) { // -inf is a value too
#pragma unroll
        for (int j = 0; j < N; j++)
            any |= here(j);
    }
    // the wave's k-th largest of its lanes' maxima: the largest number that k of them reach
    const uint32_t o = any ? lp_order(mx) : 0;
    uint32_t t = 0;
    for (int b = 31; b >= 0; b--)
        if (__popcll(__ballot(o >= (t | 1u << b))) >= k)
            t |= 1u << b;
    int last = end - 1; // of the values equal to it those up to this index
    if (t) {
        const uint64_t eq = __ballot(o == t);
        const int need = k - __popcll(__ballot(o > t));
        if (__popcll(eq) > need) { // the need-th lowest of the lanes' first indices
            int first = 0x7fffffff;
            if (o == t)
#pragma unroll
                for (int j = 0; j < N; j++)
                    if (x(j) == mx && id(j) < first)
                        first = id(j);
            uint32_t below = 0;
            for (int b = 30; b >= 0; b--)
                if (__popcll(__ballot((uint32_t)first < (below | 1u << b))) < need)
                    below |= 1u << b;
            last = (int)below;
        }
    }
    if (lane == 0)
        sh.key[wave] = t ? (uint64_t)t << 32 | (uint32_t)~last : 0;
    if (tid == 0)
        sh.count = 0;
    __syncthreads();
    uint64_t bound = sh.key[0];
#pragma unroll
    for (int w = 1; w < W; w++)
        bound = sh.key[w] > bound ? sh.key[w] : bound;
    const float from = bound ? lp_value((uint32_t)(bound >> 32)) : -__builtin_inff();
    const int upto = bound ? (int)~(uint32_t)bound : end - 1;
    const auto reaches = [&](int j) { return x(j) > from || (x(j) == from && id(j) <= upto); };
    int mine = 0;
#pragma unroll
    for (int j = 0; j < N; j++)
        mine += reaches(j);
    int at = mine ? atomicAdd(&sh.count, mine) : 0;
    if (mine) {
#pragma unroll
        for (int j = 0; j < N; j++)
            if (reaches(j)) {
                if (at < LP_LIST)
                    sh.list[at] = lp_key(x(j), id(j));
                at++;
            }
    }
    __syncthreads();
    const int count = sh.count;
    if (count <= LP_LIST) {
        if (tid == 0)
            sh.list[count] = 0; // read in pairs
        for (int r = count + tid; r < k; r += THREADS)
            sh.best[r] = {-__builtin_inff(), -1};
        __syncthreads();
        for (int c = tid; c < count; c += THREADS) {
            const uint64_t key = sh.list[c];
            int rank = 0;
            for (int j = 0; j < count; j += 2)
                rank += (sh.list[j] > key) + (sh.list[j + 1] > key);
            if (rank < k)
                sh.best[rank] = {lp_value((uint32_t)(key >> 32)), (int)~(uint32_t)key};
        }
    } else {
        uint64_t before = ~0ull;
        for (int r = 0; r < k; r++) { // count > k: there are k
            uint64_t best = 0;
#pragma unroll
            for (int j = 0; j < N; j++) {
                const uint64_t key = here(j) ? lp_key(x(j), id(j)) : 0;
                best = key < before && key > best ? key : best;
            }
            for (int s = 1; s < 64; s *= 2) {
                const uint64_t b2 = (uint64_t)__shfl_xor((long long)best, s);
                best = b2 > best ? b2 : best;
            }
            __syncthreads();
            if (lane == 0)
                sh.key[wave] = best;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < W; w++)
                best = sh.key[w] > best ? sh.key[w] : best;
            before = best;
            if (tid == 0)
                sh.best[r] = {lp_value((uint32_t)(best >> 32)), (int)~(uint32_t)best};
        }
    }
    __syncthreads();
}

// A row's results from its sums and its best: lp, entropy and the alternatives, by the work group's first lanes.
struct LpRow {
    float m;
    double s, z;
    int at;
};
__device__ __forceinline__ float lp_of(const LpRow &r, const ProbScale &sc, float t, float x, int id) {
    if (sc.greedy)
        return id == r.at && r.m > -__builtin_inff() ? 0.0f : -__builtin_inff();
    if (r.s != r.s)
        return __builtin_nanf("");
    if (x == -__builtin_inff())
        return x;
    return (float)(((double)x - (double)r.m) / (double)t - log(r.s));
}
__device__ __forceinline__ void lp_write(const LogprobParams &P, size_t row, const LpRow &r, const ProbScale &sc,
                                         const LpTop *best) {
    const int tid = threadIdx.x;
    const float t = P.temperature ? P.temperature[row] : 1.0f;
    if (tid == 0) {
        const int64_t id = P.tokens[row];
        P.lp[row] = id >= 0 && id < (int64_t)P.vocab ? lp_of(r, sc, t, P.logits[row * P.stride + id], (int)id)
                                                     : -__builtin_inff();
        // nothing above -inf: no token has a probability
        P.entropy[row] = sc.greedy || r.s == 0.0 ? 0.0f : (float)(log(r.s) - r.z / r.s);
    }
    if (tid < P.top) {
        const LpTop b = best[tid];
        P.top_ids[row * P.top + tid] = b.id;
        P.top_lp[row * P.top + tid] = b.id < 0 ? -__builtin_inff() : lp_of(r, sc, t, b.x, b.id);
    }
}

// (m, S, Z) of the values a work group holds; Z in z log2 e.
template <int THREADS, int NV>
__device__ __forceinline__ LpRec lp_sums(const smp_f4 (&v)[NV], size_t v0, const ProbScale &sc, LpShared<THREADS> &sh) {
    constexpr int W = THREADS / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float m = -__builtin_inff();
    int at = 0x7fffffff;
    if (sc.greedy) {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++)
                max_first(m, at, v[i][c], (int)(v0 + ((size_t)i * THREADS + tid) * 4 + c));
        for (int o = 1; o < 64; o *= 2)
            max_first(m, at, __shfl_xor(m, o), __shfl_xor(at, o));
    } else { // fmaxf passes a NaN over; its exponential is NaN, and with it the sums
#pragma unroll
        for (int i = 0; i < NV; i++)
            m = fmaxf(fmaxf(fmaxf(m, v[i][0]), v[i][1]), fmaxf(v[i][2], v[i][3]));
        m = wave_max(m);
    }
    if (lane == 0)
        sh.m[wave] = m, sh.at[wave] = at;
    __syncthreads();
    m = sh.m[0], at = sh.at[0];
#pragma unroll
    for (int w = 1; w < W; w++)
        max_first(m, at, sh.m[w], sh.at[w]);
    if (sc.greedy)
        return {m, 1.0f, 0.0f, at};
    const float from = m == -__builtin_inff() ? 0.0f : m;
    float s = 0.0f, z = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const float d = v[i][c] - from, e = exp_scaled(d, sc.hi, sc.lo);
            s += e;
            z = __builtin_fmaf(e, fmaxf(d * sc.hi, -200.0f), z); // e is 0 from -150 on, where d * hi may be -inf
        }
    for (int o = 1; o < 64; o *= 2) {
        s += __shfl_xor(s, o);
        z += __shfl_xor(z, o);
    }
    if (lane == 0)
        sh.s[wave] = s, sh.z[wave] = z;
    __syncthreads();
    s = sh.s[0], z = sh.z[0];
#pragma unroll
    for (int w = 1; w < W; w++)
        s += sh.s[w], z += sh.z[w];
    return {m, s, z, at};
}

template <int THREADS, int NV>
__global__ __launch_bounds__(THREADS) void logprobs_row_kernel(LogprobParams P) {
    __shared__ LpShared<THREADS> sh;
    const size_t row = blockIdx.x;
    const int tid = threadIdx.x;
    smp_f4 v[NV];
    row_part<NV, THREADS>(P.logits + row * P.stride, 0, P.vocab, -__builtin_inff(), v);
    const ProbScale sc = prob_scale(P.temperature, row);
    const LpRec r = lp_sums<THREADS, NV>(v, 0, sc, sh);
    if (P.top)
        lp_select<THREADS, NV * 4>(
            P.top, [&](int j) { return v[j / 4][j % 4]; },
            [&](int j) { return ((j / 4) * THREADS + tid) * 4 + j % 4; }, (int)P.vocab, sh);
    lp_write(P, row, {r.m, (double)r.s, (double)r.z * 0x1.62e42fefa39efp-1, r.at}, sc, sh.best);
}

template <int NV>
__global__ __launch_bounds__(SMP_THREADS) void logprobs_part_kernel(LogprobParams P) {
    __shared__ LpShared<SMP_THREADS> sh;
    const size_t row = blockIdx.x / P.splits, part = blockIdx.x;
    const int tid = threadIdx.x;
    const size_t v0 = (part - row * P.splits) * (NV * SMP_THREADS * 4);
    smp_f4 v[NV];
    row_part<NV>(P.logits + row * P.stride, v0, P.vocab, -__builtin_inff(), v);
    const ProbScale sc = prob_scale(P.temperature, row);
    const LpRec r = lp_sums<SMP_THREADS, NV>(v, v0, sc, sh);
    if (tid == 0)
        P.rec[part] = r;
    if (P.top) {
        lp_select<SMP_THREADS, NV * 4>(
            P.top, [&](int j) { return v[j / 4][j % 4]; },
            [&](int j) { return (int)v0 + ((j / 4) * SMP_THREADS + tid) * 4 + j % 4; }, (int)P.vocab, sh);
        if (tid < P.top)
            P.list[part * P.top + tid] = sh.best[tid];
    }
}

__global__ __launch_bounds__(SMP_THREADS) void logprobs_join_kernel(LogprobParams P) {
    __shared__ LpShared<SMP_THREADS> sh;
    __shared__ double ss[SMP_THREADS / 64], sz[SMP_THREADS / 64];
    const size_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const LpRec *rec = P.rec + row * P.splits;
    const ProbScale sc = prob_scale(P.temperature, row);
    float m = -__builtin_inff();
    int at = 0x7fffffff;
    for (int i = tid; i < P.splits; i += SMP_THREADS)
        max_first(m, at, rec[i].m, rec[i].at);
    for (int o = 1; o < 64; o *= 2)
        max_first(m, at, __shfl_xor(m, o), __shfl_xor(at, o));
    if (lane == 0)
        sh.m[wave] = m, sh.at[wave] = at;
    __syncthreads();
    m = sh.m[0], at = sh.at[0];
#pragma unroll
    for (int w = 1; w < SMP_THREADS / 64; w++)
        max_first(m, at, sh.m[w], sh.at[w]);
    // a part's sums are relative to its own maximum: z = z' + (m' - m)
    double s = 0.0, z = 0.0;
    for (int i = tid; i < P.splits; i += SMP_THREADS) {
        const LpRec r = rec[i];
        const float d = r.m - m;
        const double f = r.m == -__builtin_inff() ? 1.0 : (double)exp_scaled(d, sc.hi, sc.lo); // a part of -inf has 0 or NaN
        s += f * (double)r.s;
        z += f * ((double)r.z + (double)r.s * (double)fmaxf(d * sc.hi, -200.0f));
    }
    for (int o = 1; o < 64; o *= 2) {
        s += __shfl_xor(s, o);
        z += __shfl_xor(z, o);
    }
    if (lane == 0)
        ss[wave] = s, sz[wave] = z;
    __syncthreads();
    s = ss[0], z = sz[0];
#pragma unroll
    for (int w = 1; w < SMP_THREADS / 64; w++)
        s += ss[w], z += sz[w];
    if (P.top) {
        const LpTop *list = P.list + row * P.splits * P.top;
        const int all = P.splits * P.top;
        LpTop e[LP_JOIN_N];
#pragma unroll
        for (int j = 0; j < LP_JOIN_N; j++) {
            const int i = j * SMP_THREADS + tid;
            e[j] = {__builtin_nanf(""), 0};
            if (i < all) {
                e[j] = list[i];
                e[j].x = e[j].id < 0 ? __builtin_nanf("") : e[j].x;
            }
        }
        lp_select<SMP_THREADS, LP_JOIN_N>(
            P.top, [&](int j) { return e[j].x; }, [&](int j) { return e[j].id; }, (int)P.vocab, sh);
    }
    lp_write(P, row, {m, s, z * 0x1.62e42fefa39efp-1, at}, sc, sh.best);
}

static RowCut lp_cut(size_t n, size_t vocab, size_t top) {
    // as many parts as fill the chip, and no more than one work group joins
    size_t groups = 1024;
    const size_t most = top ? LP_JOIN / top : LP_JOIN;
    if ((groups + n - 1) / n > most)
        groups = most * n;
    return row_cut(n, vocab, groups);
}

} // namespace lh

using namespace lh;

extern "C" {

size_t loomhip_token_logprobs_ws(size_t n, size_t vocab, size_t top) {
    if (n == 0 || n > 65535 || vocab <= LP_ROW || vocab > LP_MAX_VOCAB || top > LP_MAX_TOP)
        return 0;
    return n * lp_cut(n, vocab, top).splits * (sizeof(LpRec) + top * sizeof(LpTop));
}

int loomhip_token_logprobs_dev(const float *logits, size_t n, size_t vocab, size_t stride, const int32_t *tokens,
                               const float *temperature, size_t top, float *logprobs, float *entropy, int32_t *top_ids,
                               float *top_logprobs, void *ws, size_t ws_bytes, void *stream) {
    const char *fn = "token_logprobs";
    if (n == 0)
        return LOOMHIP_OK;
    if (!logits || !tokens || !logprobs || !entropy || vocab == 0 || (top && (!top_ids || !top_logprobs)))
        return fail(LOOMHIP_ERR_ARG, "%s: null argument or no vocabulary", fn);
    if (n > 65535 || vocab > LP_MAX_VOCAB || top > LP_MAX_TOP)
        return fail(LOOMHIP_DECLINED, "%s: %zu rows of %zu, the best %zu not served", fn, n, vocab, top);
    if (((uintptr_t)logits | (uintptr_t)tokens | (uintptr_t)temperature | (uintptr_t)logprobs | (uintptr_t)entropy |
         (top ? (uintptr_t)top_ids | (uintptr_t)top_logprobs : 0)) % 4)
        return fail(LOOMHIP_ERR_ARG, "%s: a pointer is not aligned to its elements", fn);
    if (n > 1 && stride < vocab)
        return fail(LOOMHIP_ERR_ARG, "%s: row stride %zu below %zu values", fn, stride, vocab);
    const size_t need = loomhip_token_logprobs_ws(n, vocab, top);
    if (need && (!ws || ws_bytes < need || (uintptr_t)ws % 16))
        return fail(LOOMHIP_ERR_ARG, "%s: the workspace takes %zu bytes at a multiple of 16, got %zu", fn, need, ws_bytes);
    if (int rc = require_device())
        return rc;
    hipStream_t st = stream_of(stream);
    LogprobParams P = {logits, vocab, stride, tokens, temperature, (int)top, 1, logprobs, entropy, top_ids, top_logprobs,
                       nullptr, nullptr};
    if (vocab <= LP_ROW) {
        if (vocab <= 4096)
            hipLaunchKernelGGL((logprobs_row_kernel<256, 4>), dim3(n), dim3(256), 0, st, P);
        else if (vocab <= 16384)
            hipLaunchKernelGGL((logprobs_row_kernel<1024, 4>), dim3(n), dim3(1024), 0, st, P);
        else
            hipLaunchKernelGGL((logprobs_row_kernel<1024, 8>), dim3(n), dim3(1024), 0, st, P);
        note_launch();
    } else {
        const RowCut cut = lp_cut(n, vocab, top);
        P.splits = cut.splits;
        P.rec = (LpRec *)ws;
        P.list = (LpTop *)(P.rec + n * cut.splits);
        const dim3 g(n * cut.splits);
        if (cut.nv == 2)
            hipLaunchKernelGGL((logprobs_part_kernel<2>), g, dim3(SMP_THREADS), 0, st, P);
        else if (cut.nv == 4)
            hipLaunchKernelGGL((logprobs_part_kernel<4>), g, dim3(SMP_THREADS), 0, st, P);
        else if (cut.nv == 8)
            hipLaunchKernelGGL((logprobs_part_kernel<8>), g, dim3(SMP_THREADS), 0, st, P);
        else
            hipLaunchKernelGGL((logprobs_part_kernel<16>), g, dim3(SMP_THREADS), 0, st, P);
        hipLaunchKernelGGL(logprobs_join_kernel, dim3(n), dim3(SMP_THREADS), 0, st, P);
        note_launch();
        note_launch();
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? LOOMHIP_OK : hip_fail(e, "token_logprobs launch");
}

} // extern "C"

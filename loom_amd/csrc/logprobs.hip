// logprobs.hip -- log probabilities of given tokens, the rows' entropy and
// their likeliest alternatives.
//
//   m = max x,  S = sum e_v,  Z = sum e_v z_v,  z = (x - m) / T,  e = exp z
//   lp_v = z_v - log S,  entropy = log S - Z / S
//
// in one reading of the row.  The `top` largest are found in the registers that
// hold it: the k-th largest of the threads' maxima is a bound that k values
// reach, so no value below it is among the k; the few that reach it (a handful
// more than k) are collected in LDS, where each counts those before it.  Where
// too many do (values arranged so that a few threads hold them all), the k are
// picked one after the other.  A row of up to 32768 values takes one launch (a
// work group holds it, up to 128 values a thread; 9 us for 32000 with 5 best,
// where parts and their join take 10.7); of a longer one each part leaves (m, S,
// Z) and its own k, which a second launch joins.
//
// Bound by bytes without alternatives (509 rows of 151936 48 us, 6.4 TB/s, and 5
// for the join); with them by what a work group does one step after the other
// once it has its part: 64 rows with 20 best 14.8 us, without 9.2, and 6.6 for
// the join, 4.
#include "sampling.hpp"

#include <type_traits>

namespace lh {

constexpr int LP_MAX_TOP = 32;
constexpr int LP_WAVES = SMP_THREADS / 64;
constexpr int LP_LIST = 64;        // values collected of a wave at most
constexpr int LP_PAD = 8;          // they are read in pieces of this
// Threads whose maxima may reach the bound beside the k: fewer take more bits of the search, more leave more values to
// rank.  64 rows of 151936 with 20 best: 14.3 us with 4, 17.5 with 12.
constexpr int LP_SPARE = 4;
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

struct LpShared {
    float m[LP_WAVES], s[LP_WAVES], z[LP_WAVES];
    int at[LP_WAVES];
    uint32_t top[SMP_THREADS], bound;
    bool ties;
    uint64_t key[LP_WAVES];
    uint32_t count[LP_WAVES];
    __attribute__((aligned(16))) uint64_t list[LP_WAVES][LP_LIST];
    LpTop best[LP_MAX_TOP];
};

// The k best of the work group's values (x(j) with index id(j), j < N, of every thread; NaN and indices from `end` on
// are none) into sh.best, in order, for the first wave to read.
template <int N, class X, class Id>
__device__ __forceinline__ void lp_select(int k, X x, Id id, int end, LpShared &sh) {
    constexpr int W = LP_WAVES, LIST = LP_LIST, Q = N % 4 ? 1 : 4; // values are looked at by Q
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const auto here = [&](int j) { return x(j) == x(j) && id(j) < end; };
    float mq[N / Q], mx = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < N / Q; j++) {
        mq[j] = x(j * Q);
#pragma unroll
        for (int c = 1; c < Q; c++)
            mq[j] = fmaxf(mq[j], x(j * Q + c));
        mx = fmaxf(mx, mq[j]);
    }
    bool any = mx > -__builtin_inff();
    if (!any) { // -inf is a value too
#pragma unroll
        for (int j = 0; j < N; j++)
            any |= here(j);
    }
    // The bound: a number that k of the threads' maxima reach and not many more, or the k-th largest of them.  The first
    // wave looks for it, bit by bit.
    sh.top[tid] = any ? lp_order(mx) : 0;
    __syncthreads();
    constexpr uint32_t LEAST = 0x007fffffu; // the order of -inf
    if (wave == 0) {
        uint32_t o[W], t = 0;
#pragma unroll
        for (int w = 0; w < W; w++)
            o[w] = sh.top[w * 64 + lane];
        const auto reach = [&](uint32_t t) {
            int c = 0;
#pragma unroll
            for (int w = 0; w < W; w++)
                c += __popcll(__ballot(o[w] >= t));
            return c;
        };
        int b = 31, most = 0; // how many reach t
        // the largest's sign and most of its exponent are most often those of the k-th largest too
        float big = lp_value(o[0] > LEAST ? o[0] : LEAST);
#pragma unroll
        for (int w = 1; w < W; w++)
            big = fmaxf(big, lp_value(o[w] > LEAST ? o[w] : LEAST));
        const uint32_t head = lp_order(wave_max(big)) & 0xff000000u;
        if (head && reach(head) >= k) {
            t = head;
            most = reach(head);
            b = 23;
        }
        for (; b >= 0 && (most < k || most > k + LP_SPARE); b--) {
            const int c = reach(t | 1u << b);
            t |= c >= k ? 1u << b : 0;
            most = c >= k ? c : most;
        }
        if (lane == 0) {
            sh.bound = t && t < LEAST ? LEAST : t;
            sh.ties = t && most > k + LP_SPARE;
        }
    }
    __syncthreads();
    const uint32_t t = sh.bound;
    int upto = end - 1; // of the values equal to it those up to this index
    if (sh.ties) {      // many are equal to it: up to the index that makes up k of the threads' first ones
        int first = 0x7fffffff;
        if (sh.top[tid] == t)
#pragma unroll
            for (int j = 0; j < N; j++)
                if (x(j) == mx && id(j) < first)
                    first = id(j);
        const uint64_t over = __ballot(sh.top[tid] > t);
        if (lane == 0)
            sh.count[wave] = __popcll(over);
        __syncthreads();
        sh.top[tid] = (uint32_t)first;
        __syncthreads();
        uint32_t o[W], below = 0;
        int need = k;
#pragma unroll
        for (int w = 0; w < W; w++) {
            o[w] = sh.top[w * 64 + lane];
            need -= (int)sh.count[w];
        }
        for (int b = 30; b >= 0; b--) {
            int c = 0;
#pragma unroll
            for (int w = 0; w < W; w++)
                c += __popcll(__ballot(o[w] < (below | 1u << b)));
            below |= c < need ? 1u << b : 0;
        }
        upto = (int)below;
        __syncthreads(); // count is read
    }
    const float from = t ? lp_value(t) : -__builtin_inff();
    // what reaches the bound, into the wave's part of the list
    uint32_t mine = 0;
    const auto collect = [&](auto reaches) {
#pragma unroll
        for (int g = 0; g < N / Q; g++)
            if (__any(mq[g] >= from))
#pragma unroll
                for (int j = g * Q; j < g * Q + Q; j++) {
                    const uint64_t b = __ballot(reaches(j));
                    if (b) {
                        const uint32_t at = mine + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32),
                                                                             __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
                        if ((b >> lane & 1) && at < LIST)
                            sh.list[wave][at] = lp_key(x(j), id(j));
                        mine += __popcll(b);
                    }
                }
    };
    if (__any(mx >= from)) {
        if (from > -__builtin_inff() && upto == end - 1) // no tie to be told apart: the index says nothing
            collect([&](int j) { return x(j) >= from; });
        else
            collect([&](int j) { return x(j) > from || (x(j) == from && id(j) <= upto); });
    }
    if (lane == 0)
        sh.count[wave] = mine;
    if (mine + lane < LIST) // zeros, before no other, behind them
        sh.list[wave][mine + lane] = 0;
    __syncthreads();
    uint32_t most = 0, all = 0;
#pragma unroll
    for (int w = 0; w < W; w++) {
        all += sh.count[w];
        most = sh.count[w] > most ? sh.count[w] : most;
    }
    if (most <= LIST) {
        if (wave == 0) {
            if ((uint32_t)lane >= all && lane < k)
                sh.best[lane] = {-__builtin_inff(), -1};
            // sixteen of each wave's at a time, each counting those before it
            for (uint32_t i = lane & 15; i - (lane & 15) < most; i += 16) {
                const uint64_t key = sh.list[lane >> 4][i];
                int rank = 0;
                for (uint32_t j = 0; j < most; j += LP_PAD)
#pragma unroll
                    for (int w = 0; w < W; w++)
#pragma unroll
                        for (int e = 0; e < LP_PAD; e++)
                            rank += sh.list[w][j + e] > key;
                if (key && rank < k)
                    sh.best[rank] = {lp_value((uint32_t)(key >> 32)), (int)~(uint32_t)key};
            }
            wave_lds_sync();
        }
    } else {
        uint64_t before = ~0ull;
        for (int r = 0; r < k; r++) { // there are k
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
        __syncthreads();
    }
}

// A row's sums, and of them every thread's log S.
struct LpRow {
    float m;
    double s, z;
    int at;
};
// The given token and its logit, loaded by every thread before anything is waited for.
struct LpGiven {
    int id;
    float x;
};
__device__ __forceinline__ LpGiven lp_given(const LogprobParams &P, size_t row) {
    const int id = P.tokens[row];
    const bool in = id >= 0 && (uint32_t)id < (uint32_t)P.vocab;
    return {in ? id : -1, P.logits[row * P.stride + (in ? id : 0)]};
}
// A row's results: a thread of the first wave for each of the best, one of the second for the given token, of the third
// for the entropy.
__device__ __forceinline__ void lp_write(const LogprobParams &P, size_t row, const LpRow &r, const ProbScale &sc,
                                         const LpGiven &g, const LpTop *best) {
    const int tid = threadIdx.x;
    if (tid >= P.top && tid != 64 && tid != 128)
        return;
    const LpTop b = tid < P.top ? best[tid] : LpTop{g.x, g.id};
    const double log_s = log(r.s);
    float lp;
    if (b.id < 0)
        lp = -__builtin_inff();
    else if (sc.greedy)
        lp = b.id == r.at && r.m > -__builtin_inff() ? 0.0f : -__builtin_inff();
    else if (r.s != r.s)
        lp = __builtin_nanf("");
    else if (b.x == -__builtin_inff())
        lp = b.x;
    else
        lp = (float)(((double)b.x - (double)r.m) / (P.temperature ? (double)P.temperature[row] : 1.0) - log_s);
    if (tid < P.top) {
        P.top_ids[row * P.top + tid] = b.id;
        P.top_lp[row * P.top + tid] = lp;
    } else if (tid == 64) {
        P.lp[row] = lp;
    } else { // nothing above -inf: no token has a probability
        const double h = log_s - r.z / r.s;
        P.entropy[row] = sc.greedy || r.s == 0.0 || h < 0.0 ? 0.0f : (float)h; // below 0 by rounding alone
    }
}

// (m, S, Z) of the values a work group holds; Z in z log2 e.
template <int NV>
__device__ __forceinline__ LpRec lp_sums(const smp_f4 (&v)[NV], size_t v0, const ProbScale &sc, LpShared &sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float m = -__builtin_inff();
    int at = 0x7fffffff;
    bool nan = false;
    if (sc.greedy) {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++)
                max_first(m, at, v[i][c], (int)(v0 + ((size_t)i * SMP_THREADS + tid) * 4 + c));
        for (int o = 1; o < 64; o *= 2)
            max_first(m, at, __shfl_xor(m, o), __shfl_xor(at, o));
    } else { // fmaxf passes a NaN over
#pragma unroll
        for (int i = 0; i < NV; i++) {
            m = fmaxf(m, fmaxf(fmaxf(fmaxf(v[i][0], v[i][1]), v[i][2]), v[i][3]));
            nan |= __builtin_isunordered(v[i][0], v[i][1]) | __builtin_isunordered(v[i][2], v[i][3]);
        }
        m = wave_max(m);
    }
    if (lane == 0)
        sh.m[wave] = m, sh.at[wave] = at;
    __syncthreads();
    m = sh.m[0], at = sh.at[0];
#pragma unroll
    for (int w = 1; w < LP_WAVES; w++)
        max_first(m, at, sh.m[w], sh.at[w]);
    if (sc.greedy)
        return {m, 1.0f, 0.0f, at};
    // (x - m) / T log2 e = d hi + d lo; d no further below than where the exponential has long been 0, so that neither
    // product is infinite.  At a T past which d is of halves (1e30) that may be further than f32 reaches, and -inf is told
    // apart.
    const float from = m == -__builtin_inff() ? 0.0f : m, least = -300.0f / sc.hi;
    float s = 0.0f, z = 0.0f;
    const auto add = [&](float d) {
        const float h = __builtin_fmaf(d, sc.hi, d * sc.lo);
        const float e = __builtin_amdgcn_exp2f(h);
        s += e;
        z = __builtin_fmaf(e, h, z);
    };
    if (sc.part == 1.0f) {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++)
                add(fmaxf(v[i][c] - from, least));
    } else {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (v[i][c] != -__builtin_inff())
                    add(prob_diff(sc, v[i][c], from));
    }
    if (nan || m == __builtin_inff()) // lost on the way
        s = __builtin_nanf("");
    for (int o = 1; o < 64; o *= 2) {
        s += __shfl_xor(s, o);
        z += __shfl_xor(z, o);
    }
    if (lane == 0)
        sh.s[wave] = s, sh.z[wave] = z;
    __syncthreads();
    s = sh.s[0], z = sh.z[0];
#pragma unroll
    for (int w = 1; w < LP_WAVES; w++)
        s += sh.s[w], z += sh.z[w];
    return {m, s, z, at};
}

// The values of row part v0 .. that a thread holds, as lp_select takes them.
template <int NV>
__device__ __forceinline__ void lp_best(const LogprobParams &P, const smp_f4 (&v)[NV], size_t v0, LpShared &sh) {
    const int first = (int)v0 + (int)threadIdx.x * 4;
    lp_select<NV * 4>(
        P.top, [&](int j) { return v[j / 4][j % 4]; }, [&](int j) { return first + (j / 4) * SMP_THREADS * 4 + j % 4; },
        (int)P.vocab, sh);
}

template <int NV>
__global__ __launch_bounds__(SMP_THREADS, NV == 32 ? 1 : 2) void logprobs_row_kernel(LogprobParams P) {
    __shared__ LpShared sh;
    const size_t row = blockIdx.x;
    smp_f4 v[NV];
    row_part<NV>(P.logits + row * P.stride, 0, P.vocab, -__builtin_inff(), v);
    const LpGiven given = lp_given(P, row);
    const ProbScale sc = prob_scale(P.temperature, row);
    const LpRec r = lp_sums<NV>(v, 0, sc, sh);
    if (P.top)
        lp_best<NV>(P, v, 0, sh);
    lp_write(P, row, {r.m, (double)r.s, (double)r.z * 0x1.62e42fefa39efp-1, r.at}, sc, given, sh.best);
}

template <int NV>
__global__ __launch_bounds__(SMP_THREADS) void logprobs_part_kernel(LogprobParams P) {
    __shared__ LpShared sh;
    const size_t row = blockIdx.x / P.splits, part = blockIdx.x;
    const int tid = threadIdx.x;
    const size_t v0 = (part - row * P.splits) * (NV * SMP_THREADS * 4);
    smp_f4 v[NV];
    const float *x = P.logits + row * P.stride;
    if (v0 + NV * SMP_THREADS * 4 <= P.vocab) {
        // read once, past the caches: 509 rows of 151936 take 53.8 us, with plain loads 59.6
#pragma unroll
        for (int i = 0; i < NV; i++)
            v[i] = __builtin_nontemporal_load((const smp_f4u *)(x + v0 + ((size_t)i * SMP_THREADS + tid) * 4));
    } else {
        row_part<NV>(x, v0, P.vocab, -__builtin_inff(), v);
    }
    const ProbScale sc = prob_scale(P.temperature, row);
    const LpRec r = lp_sums<NV>(v, v0, sc, sh);
    if (tid == 0)
        P.rec[part] = r;
    if (P.top) {
        lp_best<NV>(P, v, v0, sh);
        if (tid < P.top)
            P.list[part * P.top + tid] = sh.best[tid];
    }
}

// N: entries of the parts' best that a thread takes
template <int N>
__global__ __launch_bounds__(SMP_THREADS) void logprobs_join_kernel(LogprobParams P) {
    __shared__ LpShared sh;
    __shared__ double ss[SMP_THREADS / 64], sz[SMP_THREADS / 64];
    const size_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const LpRec *rec = P.rec + row * P.splits;
    LpTop e[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
        // the parts' first ones into different threads, also where 256 is a multiple of top
        const int i = j * SMP_THREADS + (tid + j * 5) % SMP_THREADS;
        e[j] = {__builtin_nanf(""), -1};
        if (i < P.splits * P.top)
            e[j] = P.list[row * P.splits * P.top + i];
    }
    const LpGiven given = lp_given(P, row);
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
        const float d = prob_diff(sc, r.m, m);
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
#pragma unroll
        for (int j = 0; j < N; j++)
            e[j].x = e[j].id < 0 ? __builtin_nanf("") : e[j].x;
        lp_select<N>(
            P.top, [&](int j) { return e[j].x; }, [&](int j) { return e[j].id; }, (int)P.vocab, sh);
    }
    lp_write(P, row, {m, s, z * 0x1.62e42fefa39efp-1, at}, sc, given, sh.best);
}

static RowCut lp_cut(size_t n, size_t vocab, size_t top) {
    // as many parts as fill the chip twice over (64 rows of 151936: 9.2 us, with half as many 10.4; with 20 best 14.3 and
    // 15), and no more than one work group joins
    size_t groups = 2048;
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
        const auto run = [&](auto nv) {
            constexpr int NV = decltype(nv)::value;
            hipLaunchKernelGGL((logprobs_row_kernel<NV>), dim3(n), dim3(SMP_THREADS), 0, st, P);
        };
        if (vocab <= 4096)
            run(std::integral_constant<int, 4>{});
        else if (vocab <= 8192)
            run(std::integral_constant<int, 8>{});
        else if (vocab <= 16384)
            run(std::integral_constant<int, 16>{});
        else
            run(std::integral_constant<int, 32>{});
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
        const size_t entries = cut.splits * top;
        if (entries <= SMP_THREADS)
            hipLaunchKernelGGL(logprobs_join_kernel<1>, dim3(n), dim3(SMP_THREADS), 0, st, P);
        else if (entries <= SMP_THREADS * 4)
            hipLaunchKernelGGL(logprobs_join_kernel<4>, dim3(n), dim3(SMP_THREADS), 0, st, P);
        else
            hipLaunchKernelGGL(logprobs_join_kernel<LP_JOIN_N>, dim3(n), dim3(SMP_THREADS), 0, st, P);
        note_launch();
        note_launch();
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? LOOMHIP_OK : hip_fail(e, "token_logprobs launch");
}

} // extern "C"

// sampling.hip -- from logits to tokens for a batched serving step: token
// probabilities at a temperature, and the verification of drafted tokens
// against the target's probabilities from given random numbers.
#include "sampling.hpp"

#include <type_traits>

namespace lh {

// ---- token probabilities -------------------------------------------------------
// p_v = exp((x_v - m) / T) / sum_w exp((x_w - m) / T), m = max x.  A row that
// a work group can hold takes one launch; a longer one two: each (row, split)
// reduces its values to (max, sum of exponentials, first index of the max);
// then each (row, split) merges the row's records and writes its probabilities.
// T infinite: finite logits weigh alike, -inf still nothing.
// T not positive, NaN or so small that 1/T passes f32: 1 at the first maximum
// among the numbers (a NaN logit makes a row of any other T NaN).
// Bound by bytes: 160 rows of 151936 take 22.6 us for the sums (4.3 TB/s) and
// 31 for the second read, mostly from the last-level cache, and the write
// (medians of calls that follow each other).
struct ProbRec {
    float m, l;
    int32_t at;
    int32_t pad;
};

template <int NV>
__global__ __launch_bounds__(SMP_THREADS) void probs_reduce_kernel(const float *__restrict__ logits, size_t vocab,
                                                                   size_t stride, const float *__restrict__ temperature,
                                                                   int splits, ProbRec *__restrict__ rec) {
    __shared__ float sm[SMP_THREADS / 64], sl[SMP_THREADS / 64];
    __shared__ int sa[SMP_THREADS / 64];
    const size_t row = blockIdx.x / splits;
    const int split = blockIdx.x % splits;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t v0 = (size_t)split * (NV * SMP_THREADS * 4);
    smp_f4 v[NV];
    row_part<NV>(logits + row * stride, v0, vocab, -__builtin_inff(), v);
    const ProbScale sc = prob_scale(temperature, row);
    float m = -__builtin_inff();
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int c = 0; c < 4; c++)
            max_first(m, at, v[i][c], (int)(v0 + ((size_t)i * SMP_THREADS + tid) * 4 + c));
    for (int o = 1; o < 64; o *= 2)
        max_first(m, at, __shfl_xor(m, o), __shfl_xor(at, o));
    if (lane == 0)
        sm[wave] = m, sa[wave] = at;
    __syncthreads();
    m = sm[0], at = sa[0];
    for (int w = 1; w < SMP_THREADS / 64; w++)
        max_first(m, at, sm[w], sa[w]);
    const float from = m == -__builtin_inff() ? 0.0f : m; // nothing above -inf: zeros, or the NaN among them
    float l = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int c = 0; c < 4; c++)
            l += exp_scaled(prob_diff(sc, v[i][c], from), sc.hi, sc.lo);
    for (int o = 1; o < 64; o *= 2)
        l += __shfl_xor(l, o);
    if (lane == 0)
        sl[wave] = l;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < SMP_THREADS / 64; w++)
            l += sl[w];
        rec[blockIdx.x] = {m, l, at, 0};
    }
}

template <int NV>
__global__ __launch_bounds__(SMP_THREADS) void probs_write_kernel(const float *logits, size_t vocab, size_t stride,
                                                                  const float *__restrict__ temperature, int splits,
                                                                  const ProbRec *__restrict__ rec, float *probs,
                                                                  size_t out_stride) {
    // probs may be logits: a thread reads its values before it writes them
    // The parts in the reduction's order backwards, eight at a time: a part stays with its XCD, and those read last
    // may still be in its L2.
    const int item = (int)((gridDim.x - 1 - blockIdx.x) & ~7u) + (int)(blockIdx.x & 7);
    const int b = gridDim.x % 8 ? (int)(gridDim.x - 1 - blockIdx.x) : item;
    const size_t row = b / splits;
    const int split = b % splits, tid = threadIdx.x, lane = tid & 63;
    const size_t v0 = (size_t)split * (NV * SMP_THREADS * 4);
    smp_f4 v[NV];
    row_part<NV>(logits + row * stride, v0, vocab, -__builtin_inff(), v);
    float *p = probs + row * out_stride;
    const ProbScale sc = prob_scale(temperature, row);
    float m = -__builtin_inff();
    int at = 0x7fffffff;
    for (int s = lane; s < splits; s += 64)
        max_first(m, at, rec[row * splits + s].m, rec[row * splits + s].at);
    for (int o = 1; o < 64; o *= 2)
        max_first(m, at, __shfl_xor(m, o), __shfl_xor(at, o));
    float l = 0.0f;
    for (int s = lane; s < splits; s += 64) {
        const ProbRec r = rec[row * splits + s];
        l += r.m == -__builtin_inff() ? r.l : r.l * exp_scaled(prob_diff(sc, r.m, m), sc.hi, sc.lo);
    }
    for (int o = 1; o < 64; o *= 2)
        l += __shfl_xor(l, o);
    // nothing above -inf: no token has a probability, zeros (NaN by l where there is one among them)
    const float inv = l == 0.0f ? 1.0f : 1.0f / l;
    at = m == -__builtin_inff() ? -1 : at;
    m = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const size_t k = v0 + ((size_t)i * SMP_THREADS + tid) * 4;
        smp_f4 e;
#pragma unroll
        for (int c = 0; c < 4; c++)
            e[c] = sc.greedy ? ((int64_t)(k + c) == at ? 1.0f : 0.0f) : exp_scaled(prob_diff(sc, v[i][c], m), sc.hi, sc.lo) * inv;
        if (k + 4 <= vocab) {
            __builtin_nontemporal_store(e, (smp_f4u *)(p + k));
        } else {
#pragma unroll
            for (int c = 0; c < 3; c++)
                if (k + c < vocab)
                    p[k + c] = e[c];
        }
    }
}

// The same of a row that one work group holds in registers, in one launch.
template <int THREADS, int NV>
__global__ __launch_bounds__(THREADS) void probs_row_kernel(const float *logits, size_t vocab, size_t stride,
                                                            const float *__restrict__ temperature, float *probs,
                                                            size_t out_stride) {
    constexpr int W = THREADS / 64;
    __shared__ float sm[W], sl[W];
    __shared__ int sa[W];
    const size_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    smp_f4 v[NV];
    row_part<NV, THREADS>(logits + row * stride, 0, vocab, -__builtin_inff(), v);
    const ProbScale sc = prob_scale(temperature, row);
    float m = -__builtin_inff(), inv = 1.0f;
    if (sc.greedy) {
        int at = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++)
                max_first(m, at, v[i][c], (i * THREADS + tid) * 4 + c);
        for (int o = 1; o < 64; o *= 2)
            max_first(m, at, __shfl_xor(m, o), __shfl_xor(at, o));
        if (lane == 0)
            sm[wave] = m, sa[wave] = at;
        __syncthreads();
        m = sm[lane % W], at = sa[lane % W];
        for (int o = 1; o < W; o *= 2)
            max_first(m, at, __shfl_xor(m, o), __shfl_xor(at, o));
        at = m == -__builtin_inff() ? -1 : at; // nothing above -inf: no token has a probability
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++)
                v[i][c] = (i * THREADS + tid) * 4 + c == at ? 1.0f : 0.0f;
    } else {
        // fmaxf passes a NaN over; its exponential below is NaN, and with the sum the whole row
#pragma unroll
        for (int i = 0; i < NV; i++)
            m = fmaxf(fmaxf(fmaxf(m, v[i][0]), v[i][1]), fmaxf(v[i][2], v[i][3]));
        for (int o = 1; o < 64; o *= 2)
            m = fmaxf(m, __shfl_xor(m, o));
        if (lane == 0)
            sm[wave] = m;
        __syncthreads();
        m = sm[lane % W];
        for (int o = 1; o < W; o *= 2)
            m = fmaxf(m, __shfl_xor(m, o));
        m = m == -__builtin_inff() ? 0.0f : m; // every logit is -inf: a row of zeros
        float l = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                v[i][c] = exp_scaled(prob_diff(sc, v[i][c], m), sc.hi, sc.lo);
                l += v[i][c];
            }
        for (int o = 1; o < 64; o *= 2)
            l += __shfl_xor(l, o);
        if (lane == 0)
            sl[wave] = l;
        __syncthreads();
        l = sl[lane % W];
        for (int o = 1; o < W; o *= 2)
            l += __shfl_xor(l, o);
        inv = l == 0.0f ? 1.0f : 1.0f / l;
    }
    float *p = probs + row * out_stride;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const size_t k = ((size_t)i * THREADS + tid) * 4;
        const smp_f4 e = v[i] * inv;
        if (k + 4 <= vocab) {
            *(smp_f4u *)(p + k) = e;
        } else {
#pragma unroll
            for (int c = 0; c < 3; c++)
                if (k + c < vocab)
                    p[k + c] = e[c];
        }
    }
}
// Rows up to this many values take it, whatever their number: the logits are read once.  Measured, in a graph, against
// the two launches: one row of 4096 values 3.2 us for 7.3, of 32000 6.9 for 7.7; 1024 rows of 32000 53 us for 68.  A
// row of 65536, 64 values a thread, 12 for 7.6: past 32768 a single row waits for one work group's arithmetic.
constexpr size_t PROBS_ROW = 32768;

// ---- verification of drafted tokens ----------------------------------------------
// Lane i's drafted token j (x_j, drawn from q_j) is accepted while u_j * q_j(x_j) <
// p_j(x_j); after the first refusal, at row r, the next token comes from
// max(p_r - q_r, 0), after none from p_nd, by the inverse of the running sum
// at a given number u: the lowest v with c_v > u * c_last.  The products and
// the sums are in 64 bits: they decide a whole number.  A long row takes two
// launches: each (lane, part of the row) finds r and sums its values; then one
// work group per lane scans the parts' sums and the one part that holds the
// token.  One work group holds a shorter row, and does both.  Bound by bytes:
// 64 lanes of 151936 values take 13.6 us for two rows each (5.7 TB/s), then 6.
struct VerifyParams {
    const float *target, *draft; // [n][k+1][vocab], [n][k][vocab] or null
    const int32_t *tok, *n_draft;
    const float *u_accept, *u_sample;
    size_t n, k, vocab;
    int splits;   // parts of a row
    double *sums; // [n][splits][2]: of max(p - q, 0) and of p
    int32_t *out; // [n][k+1]
    int32_t *accepted;
};

// What counts as a probability: a positive finite number, anything else as 0.
__device__ __forceinline__ float as_prob(float p) {
    constexpr int POSITIVE = 0x080 | 0x100; // subnormal, normal
    return __builtin_amdgcn_classf(p, POSITIVE) ? p : 0.0f;
}

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
// What is left of p (as_prob) at v, q the drafter's value there.
__device__ __forceinline__ double residual(const VerifyRow &r, size_t v, float p, float q) {
    if (r.q)
        return fmax((double)p - (double)as_prob(q), 0.0);
    return (int64_t)v == r.out ? 0.0 : (double)p;
}

__device__ __forceinline__ double wave_sum_f64(double v) {
    for (int o = 1; o < 64; o *= 2)
        v += __shfl_xor(v, o);
    return v;
}

// Two rows are in registers here and the last step goes through one part alone: parts of 2048 or 4096 values.
static RowCut verify_cut(size_t n, size_t vocab) {
    const int nv = row_cut(n, vocab, 2048).nv == 2 ? 2 : 4;
    return {(int)((vocab + nv * 1024 - 1) / (nv * 1024)), nv};
}

template <int NV>
__global__ __launch_bounds__(SMP_THREADS) void verify_sum_kernel(VerifyParams P) {
    __shared__ double sd[SMP_THREADS / 64], sp[SMP_THREADS / 64];
    const size_t i = blockIdx.y;
    const int nd = verify_nd(P, i), acc = verify_accepted(P, i, nd);
    const VerifyRow r = verify_row(P, i, nd, acc);
    const size_t v0 = (size_t)blockIdx.x * (NV * SMP_THREADS * 4);
    smp_f4 p[NV], q[NV];
    row_part<NV>(r.p, v0, P.vocab, 0.0f, p);
    if (r.q)
        row_part<NV>(r.q, v0, P.vocab, 0.0f, q);
    double d = 0.0, all = 0.0;
#pragma unroll
    for (int x = 0; x < NV; x++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const float pv = as_prob(p[x][c]);
            d += residual(r, v0 + ((size_t)x * SMP_THREADS + threadIdx.x) * 4 + c, pv, r.q ? q[x][c] : 0.0f);
            all += (double)pv;
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
        if (blockIdx.x == 0)
            P.accepted[i] = acc;
    }
}

// A lane's running sums of d over the wave, and the wave's sum.
__device__ __forceinline__ double wave_scan_f64(double d, double *sum) {
    const int lane = threadIdx.x & 63;
    double c = d;
    for (int o = 1; o < 64; o *= 2) {
        const double up = __shfl_up(c, o);
        c += lane >= o ? up : 0.0;
    }
    *sum = __shfl(c, 63);
    return c;
}

// The part that holds the token, then of its 256 threads' runs of NV * 4 values (one after the other here) the one that
// does, then the value.  At each step the first whose running sum passes `at` and that has anything in it, else the last
// that has.
template <int NV>
__global__ __launch_bounds__(SMP_THREADS) void verify_pick_kernel(VerifyParams P) {
    constexpr int W = SMP_THREADS / 64, E = NV * 4;
    __shared__ double sw[W], before[SMP_THREADS];
    __shared__ int s_hit[W], s_last[W];
    const size_t i = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int nd = verify_nd(P, i), acc = P.accepted[i];
    VerifyRow r = verify_row(P, i, nd, acc);
    const double *s = P.sums + i * P.splits * 2;
    double left = 0.0, total = 0.0;
    for (int b = lane; b < P.splits; b += 64)
        left += s[2 * b], total += s[2 * b + 1];
    left = wave_sum_f64(left);
    int which = 0;
    if (left > 0.0) {
        total = left;
    } else { // p nowhere above q: the target's own row
        total = wave_sum_f64(total);
        which = 1;
        r.q = nullptr;
        r.out = -1;
    }
    const double at = fmax((double)P.u_sample[i] * total, 0.0); // NaN: 0
    int32_t *out = P.out + i * (P.k + 1);
    for (int j = tid; j <= (int)P.k; j += SMP_THREADS)
        if (j != acc)
            out[j] = j < acc ? P.tok[i * P.k + j] : -1;
    if (!(total > 0.0)) { // nothing to draw from
        if (tid == 0)
            out[acc] = -1;
        return;
    }
    int part = 0;
    double run = 0.0, base = 0.0; // the sums before the chunk of 64 parts, and before the part
    for (int b0 = 0; b0 < P.splits; b0 += 64) {
        const double d = b0 + lane < P.splits ? s[2 * (b0 + lane) + which] : 0.0;
        double sum;
        const double c = wave_scan_f64(d, &sum) + run;
        const unsigned long long some = __ballot(d > 0.0), past = __ballot(d > 0.0 && c > at);
        const int x = past ? __builtin_ctzll(past) : some ? 63 - __builtin_clzll(some) : -1;
        if (x >= 0) {
            part = b0 + x;
            base = x ? __shfl(c, x - 1) : run;
        }
        if (past)
            break;
        run += sum;
    }
    // the threads' runs
    const size_t v0 = (size_t)part * (NV * SMP_THREADS * 4) + (size_t)tid * E;
    double d = 0.0;
#pragma unroll
    for (int e = 0; e < E; e += 4) {
        const smp_f4 p = row_four(r.p, v0 + e, P.vocab, 0.0f);
        smp_f4 q = {0.0f, 0.0f, 0.0f, 0.0f};
        if (r.q)
            q = row_four(r.q, v0 + e, P.vocab, 0.0f);
#pragma unroll
        for (int c = 0; c < 4; c++)
            d += residual(r, v0 + e + c, as_prob(p[c]), q[c]);
    }
    double sum;
    double c = wave_scan_f64(d, &sum);
    if (lane == 63)
        sw[wave] = c;
    __syncthreads();
    double start = base;
    for (int w = 0; w < wave; w++)
        start += sw[w];
    const double up = __shfl_up(c, 1);
    before[tid] = lane ? start + up : start;
    c += start;
    const unsigned long long some = __ballot(d > 0.0), past = __ballot(d > 0.0 && c > at);
    if (lane == 0) {
        s_hit[wave] = past ? wave * 64 + __builtin_ctzll(past) : -1;
        s_last[wave] = some ? wave * 64 + 63 - __builtin_clzll(some) : -1;
    }
    __syncthreads();
    if (wave)
        return;
    int t = -1;
    for (int w = W - 1; w >= 0; w--)
        t = s_hit[w] >= 0 ? s_hit[w] : t;
    for (int w = W - 1; w >= 0 && t < 0; w--)
        t = s_last[w];
    if (t < 0) // the part held nothing after all: not with sums above zero
        t = 0;
    // the run's values, a lane each
    const size_t v = (size_t)part * (NV * SMP_THREADS * 4) + (size_t)t * E + lane;
    const double e = lane < E && v < P.vocab ? residual(r, v, as_prob(r.p[v]), r.q ? r.q[v] : 0.0f) : 0.0;
    const double ce = wave_scan_f64(e, &sum) + before[t];
    const unsigned long long any = __ballot(e > 0.0), hit = __ballot(e > 0.0 && ce > at);
    const int x = hit ? __builtin_ctzll(hit) : any ? 63 - __builtin_clzll(any) : 0;
    if (lane == x)
        out[acc] = any ? (int32_t)v : -1;
}

// Both steps in one launch of a row that 1024 threads hold in registers: a wave NV * 256 values one after the other, a
// thread four of every 256 of them.  The wave that holds the token, then its 256 that do, then the value, chosen as above.
constexpr int VERIFY_THREADS = 1024;
template <int NV>
__global__ __launch_bounds__(VERIFY_THREADS) void verify_row_kernel(VerifyParams P) {
    constexpr int W = VERIFY_THREADS / 64;
    __shared__ double sw[2][W];
    const size_t i = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int nd = verify_nd(P, i), acc = verify_accepted(P, i, nd);
    VerifyRow r = verify_row(P, i, nd, acc);
    const size_t v0 = (size_t)wave * NV * 256 + lane * 4;
    double total = 0.0, d, fours[NV]; // fours: what is left of a thread's four values together
    for (int pass = 0; pass < 2 && !(total > 0.0); pass++) {
        if (pass) // p nowhere above q: the target's own row
            r.q = nullptr, r.out = -1;
        smp_f4 p[NV], q[NV];
#pragma unroll
        for (int x = 0; x < NV; x++)
            p[x] = row_four(r.p, v0 + x * 256, P.vocab, 0.0f);
#pragma unroll
        for (int x = 0; x < NV; x++)
            q[x] = r.q ? row_four(r.q, v0 + x * 256, P.vocab, 0.0f) : smp_f4{0.0f, 0.0f, 0.0f, 0.0f};
        d = 0.0;
#pragma unroll
        for (int x = 0; x < NV; x++) {
            fours[x] = 0.0;
#pragma unroll
            for (int c = 0; c < 4; c++)
                fours[x] += residual(r, v0 + x * 256 + c, as_prob(p[x][c]), q[x][c]);
            d += fours[x];
        }
        d = wave_sum_f64(d);
        if (lane == 0)
            sw[pass][wave] = d;
        __syncthreads();
        d = lane < W ? sw[pass][lane] : 0.0;
        total = wave_sum_f64(d);
    }
    const double at = fmax((double)P.u_sample[i] * total, 0.0); // NaN: 0
    int32_t *out = P.out + i * (P.k + 1);
    if (tid == 0)
        P.accepted[i] = acc;
    for (int j = tid; j <= (int)P.k; j += VERIFY_THREADS)
        if (j != acc)
            out[j] = j < acc ? P.tok[i * P.k + j] : -1;
    if (!(total > 0.0)) { // nothing to draw from
        if (tid == 0)
            out[acc] = -1;
        return;
    }
    // the first that has anything and whose running sum passes `at`, else the last that has
    const auto pick = [&](double d, double c) {
        const unsigned long long some = __ballot(d > 0.0), past = __ballot(d > 0.0 && c > at);
        return past ? __builtin_ctzll(past) : some ? 63 - __builtin_clzll(some) : 0;
    };
    double sum;
    double c = wave_scan_f64(d, &sum);
    const int w = pick(d, c);
    if (wave != w)
        return;
    double before = w ? __shfl(c, w - 1) : 0.0;
    // the wave's NV sums at once: each step adds the other half's sums and keeps half of the NV, then lane x * 64 / NV
    // takes the x-th
    int o = 32;
#pragma unroll
    for (int half = NV / 2; half; half /= 2, o /= 2)
#pragma unroll
        for (int x = 0; x < half; x++) {
            const double lo = fours[x], hi = fours[x + half], got = __shfl_xor(lane & o ? lo : hi, o);
            fours[x] = (lane & o ? hi : lo) + got;
        }
    for (; o; o /= 2)
        fours[0] += __shfl_xor(fours[0], o);
    d = lane % (64 / NV) ? 0.0 : fours[0];
    c = wave_scan_f64(d, &sum) + before;
    const int part = pick(d, c);
    before = part ? __shfl(c, part - 1) : before;
    // a thread's four again: the registers of all of them would spill
    const size_t v = v0 + part / (64 / NV) * 256;
    const smp_f4 pv = row_four(r.p, v, P.vocab, 0.0f);
    const smp_f4 qv = r.q ? row_four(r.q, v, P.vocab, 0.0f) : smp_f4{0.0f, 0.0f, 0.0f, 0.0f};
    double e[4];
#pragma unroll
    for (int k = 0; k < 4; k++)
        e[k] = residual(r, v + k, as_prob(pv[k]), qv[k]);
    d = e[0] + e[1] + e[2] + e[3];
    c = wave_scan_f64(d, &sum) + before;
    const int t = pick(d, c);
    c = t ? __shfl(c, t - 1) : before;
    if (lane != t)
        return;
    size_t token = v;
    bool found = false;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        c += e[k];
        if (!found && e[k] > 0.0)
            token = v + k, found = c > at;
    }
    out[acc] = (int32_t)token;
}
// Rows up to this many values take it: the second launch costs the host 3.5 us, more than the one work group a lane
// costs the device.  Measured, in a graph, against the two launches: of 8192 values one lane 6.2 us for 8.0, 256 lanes
// 7.1 for 10.0; of 32000 one lane 8.2 for 7.9, 64 lanes 10.3 for 9.9, 256 lanes 16 for 20.
constexpr size_t VERIFY_ROW = 32768;

} // namespace lh

using namespace lh;

extern "C" {

size_t loomhip_token_probs_ws(size_t n, size_t vocab) {
    return n && vocab > PROBS_ROW ? n * row_cut(n, vocab).splits * sizeof(ProbRec) : 0;
}

int loomhip_token_probs_dev(const float *logits, size_t n, size_t vocab, size_t stride, const float *temperature,
                            float *probs, size_t out_stride, void *ws, size_t ws_bytes, void *stream) {
    if (n == 0)
        return LOOMHIP_OK;
    if (!logits || !probs || vocab == 0)
        return fail(LOOMHIP_ERR_ARG, "token_probs: null argument or no vocabulary");
    if (vocab > 0x7fffffff || n > 65535)
        return fail(LOOMHIP_DECLINED, "token_probs: %zu rows of %zu not served", n, vocab);
    if ((uintptr_t)logits % 4 || (uintptr_t)probs % 4 || (uintptr_t)temperature % 4)
        return fail(LOOMHIP_ERR_ARG, "token_probs: a pointer is not aligned to its elements");
    if (stride < vocab || out_stride < vocab)
        return fail(LOOMHIP_ERR_ARG, "token_probs: row stride %zu / %zu below %zu values", stride, out_stride, vocab);
    if (!(logits == probs && (stride == out_stride || n == 1)) && rows_overlap(probs, out_stride, vocab, logits, stride, vocab, n))
        return fail(LOOMHIP_ERR_ARG, "token_probs: probs overlaps logits without being them");
    const size_t need = loomhip_token_probs_ws(n, vocab);
    if (need && (!ws || ws_bytes < need || (uintptr_t)ws % 16))
        return fail(LOOMHIP_ERR_ARG, "token_probs: the workspace takes %zu bytes at a multiple of 16, got %zu", need,
                    ws_bytes);
    if (int rc = require_device())
        return rc;
    hipStream_t st = stream_of(stream);
    if (vocab <= PROBS_ROW) {
        const auto row = [&](auto threads, auto nv) {
            constexpr int THREADS = decltype(threads)::value, NV = decltype(nv)::value;
            hipLaunchKernelGGL((probs_row_kernel<THREADS, NV>), dim3(n), dim3(THREADS), 0, st, logits, vocab, stride,
                               temperature, probs, out_stride);
        };
        using std::integral_constant;
        constexpr integral_constant<int, 256> few{};
        constexpr integral_constant<int, 1024> many{};
        if (vocab <= 1024)
            row(few, integral_constant<int, 1>{});
        else if (vocab <= 4096)
            row(few, integral_constant<int, 4>{});
        else if (vocab <= 16384)
            row(many, integral_constant<int, 4>{});
        else
            row(many, integral_constant<int, 8>{});
        note_launch();
        const hipError_t e = hipGetLastError();
        return e == hipSuccess ? LOOMHIP_OK : hip_fail(e, "token_probs launch");
    }
    const RowCut cut = row_cut(n, vocab);
    if (n * cut.splits > 0xffffff)
        return fail(LOOMHIP_DECLINED, "token_probs: %zu rows of %zu not served", n, vocab);
    ProbRec *rec = (ProbRec *)ws;
    const dim3 g(n * cut.splits);
    const auto run = [&](auto nv) {
        constexpr int NV = decltype(nv)::value;
        hipLaunchKernelGGL((probs_reduce_kernel<NV>), g, dim3(SMP_THREADS), 0, st, logits, vocab, stride, temperature,
                           cut.splits, rec);
        hipLaunchKernelGGL((probs_write_kernel<NV>), g, dim3(SMP_THREADS), 0, st, logits, vocab, stride, temperature,
                           cut.splits, rec, probs, out_stride);
    };
    if (cut.nv == 2)
        run(std::integral_constant<int, 2>{});
    else if (cut.nv == 4)
        run(std::integral_constant<int, 4>{});
    else if (cut.nv == 8)
        run(std::integral_constant<int, 8>{});
    else
        run(std::integral_constant<int, 16>{});
    note_launch();
    note_launch();
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? LOOMHIP_OK : hip_fail(e, "token_probs launch");
}

size_t loomhip_verify_drafts_ws(size_t n, size_t vocab) {
    return n && vocab > VERIFY_ROW ? n * verify_cut(n, vocab).splits * 2 * sizeof(double) : 0;
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
    if (((uintptr_t)target_probs | (uintptr_t)draft_probs | (uintptr_t)draft_tokens | (uintptr_t)n_draft |
         (uintptr_t)u_accept | (uintptr_t)u_sample | (uintptr_t)tokens_out | (uintptr_t)n_accepted) % 4)
        return fail(LOOMHIP_ERR_ARG, "verify_drafts: a pointer is not aligned to its elements");
    const size_t need = loomhip_verify_drafts_ws(n, vocab);
    if (need && (!ws || ws_bytes < need || (uintptr_t)ws % 16))
        return fail(LOOMHIP_ERR_ARG, "verify_drafts: the workspace takes %zu bytes at a multiple of 16, got %zu", need,
                    ws_bytes);
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
    P.out = tokens_out;
    P.accepted = n_accepted;
    if (vocab <= VERIFY_ROW) {
        if (vocab <= 8192)
            hipLaunchKernelGGL((verify_row_kernel<2>), dim3(n), dim3(VERIFY_THREADS), 0, st, P);
        else
            hipLaunchKernelGGL((verify_row_kernel<8>), dim3(n), dim3(VERIFY_THREADS), 0, st, P);
        note_launch();
        const hipError_t e = hipGetLastError();
        return e == hipSuccess ? LOOMHIP_OK : hip_fail(e, "verify_drafts launch");
    }
    const RowCut cut = verify_cut(n, vocab);
    P.splits = cut.splits;
    P.sums = (double *)ws;
    const auto run = [&](auto nv) {
        constexpr int NV = decltype(nv)::value;
        hipLaunchKernelGGL((verify_sum_kernel<NV>), dim3(P.splits, n), dim3(SMP_THREADS), 0, st, P);
        hipLaunchKernelGGL((verify_pick_kernel<NV>), dim3(n), dim3(SMP_THREADS), 0, st, P);
    };
    if (cut.nv == 2)
        run(std::integral_constant<int, 2>{});
    else
        run(std::integral_constant<int, 4>{});
    note_launch();
    note_launch();
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? LOOMHIP_OK : hip_fail(e, "verify_drafts launch");
}

} // extern "C"

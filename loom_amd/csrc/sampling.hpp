// sampling.hpp -- rows of logits: how they are cut and loaded, and the scaled
// exponential, shared by the token probabilities (sampling.hip) and the log
// probabilities (logprobs.hip).
#pragma once

#include "runtime.hpp"

namespace lh {

constexpr int SMP_THREADS = 256;
typedef float smp_f4 __attribute__((ext_vector_type(4)));
typedef smp_f4 smp_f4u __attribute__((aligned(4))); // at any float: a row of an odd length starts anywhere

// How a row of `vocab` values is cut: work groups of NV * 1024 values, a thread NV times four, all of them loaded before
// the first is used.  Enough work groups to fill the chip four times over, none with fewer than 2048 values; up to
// 16384 (64 registers a thread).
struct RowCut {
    int splits, nv; // nv 2, 4, 8 or 16
};
static RowCut row_cut(size_t rows, size_t vocab, size_t groups = 1024) {
    const size_t want = (groups + rows - 1) / rows;
    int nv = 2;
    while (nv < 16 && (vocab + nv * 1024 - 1) / (nv * 1024) > want)
        nv *= 2;
    return {(int)((vocab + nv * 1024 - 1) / (nv * 1024)), nv};
}

// Values at .. at + 3 of a row, `fill` past its end.
__device__ __forceinline__ smp_f4 row_four(const float *x, size_t at, size_t vocab, float fill) {
    smp_f4 v = {fill, fill, fill, fill};
    if (at + 4 <= vocab) {
        v = *(const smp_f4u *)(x + at);
    } else {
#pragma unroll
        for (int c = 0; c < 3; c++)
            if (at + c < vocab)
                v[c] = x[at + c];
    }
    return v;
}
// The values of a work group's part of a row that its thread holds: four at (i * THREADS + tid) * 4 of the part.
template <int NV, int THREADS = SMP_THREADS>
__device__ __forceinline__ void row_part(const float *x, size_t v0, size_t vocab, float fill, smp_f4 (&v)[NV]) {
#pragma unroll
    for (int i = 0; i < NV; i++)
        v[i] = row_four(x, v0 + ((size_t)i * THREADS + threadIdx.x) * 4, vocab, fill);
}

// 2^(d c), d a difference of logits (prob_diff) and c its factor, split into a
// float and its remainder so that the exponent's rounding does not grow with d c.
__device__ __forceinline__ float exp_scaled(float d, float c_hi, float c_lo) {
    const float h = d * c_hi;
    const float r = __builtin_fmaf(d, c_lo, __builtin_fmaf(d, c_hi, -h));
    const float e = __builtin_amdgcn_exp2f(h);
    // d = -inf: h = -inf, r = NaN, e = 0
    return h > -150.0f || h != h ? __builtin_fmaf(e, r * 0.69314718f, e) : 0.0f;
}

// (x - m) / T log2 e = prob_diff(x, m) (hi + lo)
struct ProbScale {
    float hi, lo, part;
    bool greedy;
};
__device__ __forceinline__ ProbScale prob_scale(const float *temperature, size_t row) {
    const float t = temperature ? temperature[row] : 1.0f;
    double c = 0x1.71547652b82fep+0 / (double)t;
    // Past a T of 1e30 a difference of logits that f32 does not hold is no longer where the exponential is 0: the
    // difference of their halves is, with twice the factor.
    const float part = c < 1e-30 ? 0.5f : 1.0f;
    c = part == 0.5f ? 2.0 * c : c;
    // an infinite T weighs finite logits alike: the smallest factor there is, not 0, which times a masked -inf is NaN
    const float hi = (float)c == 0.0f ? 0x1p-149f : (float)c;
    return {hi, (float)(c - (double)hi), part, !(t > 0.0f) || !(hi < __builtin_inff())};
}
__device__ __forceinline__ float prob_diff(const ProbScale &sc, float x, float m) {
    return __builtin_fmaf(x, sc.part, -(m * sc.part));
}

__device__ __forceinline__ void max_first(float &m, int &at, float m2, int at2) {
    // the larger value; of equal ones the lower index; a NaN is never taken
    const bool take = m2 > m || (m2 == m && at2 < at);
    m = take ? m2 : m;
    at = take ? at2 : at;
}

} // namespace lh

// lora.hip -- the low-rank adapters of many requests beside one projection:
// out_t = base_t + s_e * B_e (A_e x_t), e the adapter of vector t (none: base_t).
// Everything is f32: the adapters' values widened exactly, products and sums
// in f32, as the projection's own activations and outputs are.
#include "runtime.hpp"

namespace lh {

constexpr int LORA_THREADS = 256;
constexpr int LORA_MAX_RANK = 256;

struct LoraParams {
    const void *a, *b; // [n_adapters][rank][cols], [n_adapters][rows][rank]
    const float *scale;
    size_t n_adapters, rows, cols;
    int rank;
    const float *x, *base;
    const int32_t *ids;
    float *out;
    size_t n, x_stride, base_stride, out_stride;
};

// Whether two device ranges [p, p + elements) share a byte.
static bool overlap(const void *p, size_t pn, const void *q, size_t qn) {
    const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
    return a < b + qn * 4 && b < a + pn * 4;
}

static int lora_check(const loomhip_lora *l, const float *x, size_t x_stride, const int32_t *ids, const float *base,
                      size_t base_stride, size_t n, float *out, size_t out_stride, LoraParams &P) {
    if (!l)
        return fail(LOOMHIP_ERR_ARG, "lora: no adapters");
    if (l->type != LH_F32 && l->type != LH_F16 && l->type != LOOMHIP_BF16)
        return fail(LOOMHIP_DECLINED, "lora: type %d not served", l->type);
    if (l->rank == 0 || l->rank > LORA_MAX_RANK)
        return fail(LOOMHIP_DECLINED, "lora: rank %zu not served (1 to %d)", l->rank, LORA_MAX_RANK);
    if (l->n_adapters == 0 || l->rows == 0 || l->cols == 0 || l->n_adapters > 0x7fffffff || l->rows > 0x7fffffff ||
        l->cols > 0x7fffffff || n > 0x7fffffff)
        return fail(LOOMHIP_ERR_ARG, "lora: %zu vectors, %zu adapters of %zu x %zu", n, l->n_adapters, l->rows, l->cols);
    if (n && (!l->a || !l->b || !l->scale || !x || !ids || !out))
        return fail(LOOMHIP_ERR_ARG, "lora: null argument");
    if (x_stride < l->cols || out_stride < l->rows || (base && base_stride < l->rows))
        return fail(LOOMHIP_ERR_ARG, "lora: a row stride below its row");
    const size_t es = l->type == LH_F32 ? 4 : 2;
    if ((uintptr_t)l->a % es || (uintptr_t)l->b % es || (uintptr_t)x % 4 || (uintptr_t)out % 4 || (uintptr_t)base % 4)
        return fail(LOOMHIP_ERR_ARG, "lora: a pointer is not aligned to its elements");
    // every vector's rows are read and written by different work groups
    const size_t on = n ? (n - 1) * out_stride + l->rows : 0;
    if (n && overlap(out, on, x, (n - 1) * x_stride + l->cols))
        return fail(LOOMHIP_ERR_ARG, "lora: out overlaps x");
    if (n && base && !(base == out && base_stride == out_stride) && overlap(out, on, base, (n - 1) * base_stride + l->rows))
        return fail(LOOMHIP_ERR_ARG, "lora: out overlaps base without being it");
    P = {l->a, l->b, l->scale, l->n_adapters, l->rows, l->cols, (int)l->rank, x, base, ids, out, n, x_stride,
         base_stride, out_stride};
    return LOOMHIP_OK;
}


template <typename T>
__device__ __forceinline__ float lora_widen(T v);
template <>
__device__ __forceinline__ float lora_widen(float v) { return v; }
template <>
__device__ __forceinline__ float lora_widen(_Float16 v) { return (float)v; }
template <>
__device__ __forceinline__ float lora_widen(uint16_t v) { return __uint_as_float((uint32_t)v << 16); } // bf16

// One work group per vector: its `rank` values A_e x, a wave each in turn, then its output rows.
template <typename T>
__global__ __launch_bounds__(LORA_THREADS) void lora_kernel(LoraParams P) {
    __shared__ float y[LORA_MAX_RANK];
    const size_t t = blockIdx.x;
    const int e = P.ids[t];
    const float *x = P.x + t * P.x_stride;
    const float *base = P.base ? P.base + t * P.base_stride : nullptr;
    float *out = P.out + t * P.out_stride;
    const int tid = threadIdx.x, lane = tid & 63;
    if (e < 0 || e >= (int)P.n_adapters) {
        for (size_t r = tid; r < P.rows; r += LORA_THREADS)
            out[r] = base ? base[r] : 0.0f;
        return;
    }
    const T *a = (const T *)P.a + (size_t)e * P.rank * P.cols;
    const T *b = (const T *)P.b + (size_t)e * P.rows * P.rank;
    for (int k = tid >> 6; k < P.rank; k += LORA_THREADS / 64) {
        float s = 0.0f;
        for (size_t c = lane; c < P.cols; c += 64)
            s = __builtin_fmaf(lora_widen(a[k * P.cols + c]), x[c], s);
        for (int o = 1; o < 64; o *= 2)
            s += __shfl_xor(s, o);
        if (lane == 0)
            y[k] = s * P.scale[e];
    }
    __syncthreads();
    for (size_t r = tid; r < P.rows; r += LORA_THREADS) {
        float s = 0.0f;
        for (int k = 0; k < P.rank; k++)
            s = __builtin_fmaf(lora_widen(b[r * P.rank + k]), y[k], s);
        out[r] = base ? base[r] + s : s;
    }
}

} // namespace lh

using namespace lh;

extern "C" {

size_t loomhip_lora_ws(const loomhip_lora *l, size_t n) { return 0; }

int loomhip_lora_dev(const loomhip_lora *l, const float *x, size_t x_stride, const int32_t *ids, const float *base,
                     size_t base_stride, size_t n, float *out, size_t out_stride, void *ws, size_t ws_bytes,
                     void *stream) {
    LoraParams P;
    if (int rc = lora_check(l, x, x_stride, ids, base, base_stride, n, out, out_stride, P))
        return rc;
    if (n == 0)
        return LOOMHIP_OK;
    if (int rc = require_device())
        return rc;
    hipStream_t st = stream_of(stream);
    if (l->type == LH_F32)
        hipLaunchKernelGGL(lora_kernel<float>, dim3(n), dim3(LORA_THREADS), 0, st, P);
    else if (l->type == LH_F16)
        hipLaunchKernelGGL(lora_kernel<_Float16>, dim3(n), dim3(LORA_THREADS), 0, st, P);
    else
        hipLaunchKernelGGL(lora_kernel<uint16_t>, dim3(n), dim3(LORA_THREADS), 0, st, P);
    note_launch();
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? LOOMHIP_OK : hip_fail(e, "lora launch");
}

} // extern "C"

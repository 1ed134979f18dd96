// lora.hip -- the low-rank adapters of many requests beside one projection:
// out_t = base_t + s_e * B_e (A_e x_t), e the adapter of vector t (none: base_t).
// Everything is f32: the adapters' values widened exactly, products and sums
// in f32, as the projection's own activations and outputs are.
//
// Two launches: y = A_e x for every vector into the workspace, then out.  In
// decode (most vectors name adapters of their own, so the adapters' bytes are
// the work) a wave takes a few rows of A_e or B_e for one vector with plain
// multiply-adds; small adapters take both steps in one launch.  In prefill (a
// request's tokens share an adapter) 16 vectors of one adapter are the columns
// of f32 matrix-core tiles (v_mfma_f32_16x16x4_f32), found among 128 vectors
// at a time.  What an adapter holds reaches its own vectors only.
#include "runtime.hpp"

#include <type_traits>

namespace lh {

typedef float lora_f4 __attribute__((ext_vector_type(4)));
// The same at any element: rows of odd lengths start anywhere.
typedef lora_f4 lora_f4u __attribute__((aligned(4)));
typedef uint32_t lora_u2u __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t lora_u4 __attribute__((ext_vector_type(4)));
typedef lora_u4 lora_u4u __attribute__((aligned(2)));

constexpr int LORA_THREADS = 256;
constexpr int LORA_MAX_RANK = 256;
constexpr double LORA_FEW = 160e6;    // bytes
constexpr size_t LORA_SMALL = 131072; // bytes of one A_e

struct LoraParams {
    const void *a, *b; // [n_adapters][rank][cols], [n_adapters][rows][rank]
    const float *scale;
    size_t n_adapters, rows, cols;
    int rank;
    const float *x, *base;
    const int32_t *ids;
    float *out;
    size_t n, x_stride, base_stride, out_stride;
    float *y;   // [ks][n][rp]: scale * A_e x over each split
    int rp, ks; // rank rounded up to 16, splits of the columns
};

constexpr size_t LORA_MAX_N = 65535 * 64; // vectors, and rows: the launches' work groups

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
    if (n > LORA_MAX_N || l->rows > LORA_MAX_N)
        return fail(LOOMHIP_DECLINED, "lora: %zu vectors, %zu rows not served", n, l->rows);
    if (n && (!l->a || !l->b || !l->scale || !x || !ids || !out))
        return fail(LOOMHIP_ERR_ARG, "lora: null argument");
    if (x_stride < l->cols || out_stride < l->rows || (base && base_stride < l->rows))
        return fail(LOOMHIP_ERR_ARG, "lora: a row stride below its row");
    const size_t es = l->type == LH_F32 ? 4 : 2;
    if ((uintptr_t)l->a % es || (uintptr_t)l->b % es ||
        ((uintptr_t)l->scale | (uintptr_t)x | (uintptr_t)ids | (uintptr_t)out | (uintptr_t)base) % 4)
        return fail(LOOMHIP_ERR_ARG, "lora: a pointer is not aligned to its elements");
    // every vector's rows are read and written by different work groups
    if (rows_overlap(out, out_stride, l->rows, x, x_stride, l->cols, n))
        return fail(LOOMHIP_ERR_ARG, "lora: out overlaps x");
    if (base && !(base == out && (base_stride == out_stride || n == 1)) &&
        rows_overlap(out, out_stride, l->rows, base, base_stride, l->rows, n))
        return fail(LOOMHIP_ERR_ARG, "lora: out overlaps base without being it");
    P = {l->a, l->b, l->scale, l->n_adapters, l->rows, l->cols, (int)l->rank, x, base, ids, out, n, x_stride,
         base_stride, out_stride, nullptr, 0, 1};
    return LOOMHIP_OK;
}


// Four consecutive elements as f32, and one.
template <typename T>
__device__ __forceinline__ float lora_one(const T *p) {
    if constexpr (std::is_same_v<T, uint16_t>) // bf16
        return __uint_as_float((uint32_t)*p << 16);
    else
        return (float)*p;
}
template <typename T>
__device__ __forceinline__ lora_f4 lora_four(const T *p) {
    if constexpr (std::is_same_v<T, float>) {
        return *(const lora_f4u *)p;
    } else {
        const lora_u2u v = *(const lora_u2u *)p;
        if constexpr (std::is_same_v<T, uint16_t>)
            return lora_f4{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
                           __uint_as_float(v.y & 0xffff0000u)};
        else
            return lora_f4{half_bits_to_float(v.x), half_bits_to_float(v.x >> 16), half_bits_to_float(v.y),
                           half_bits_to_float(v.y >> 16)};
    }
}
// Elements k .. k + 3 of a row of `len`, zero past its end.
template <typename T>
__device__ __forceinline__ lora_f4 lora_at(const T *row, size_t k, size_t len) {
    lora_f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (k + 4 <= len) {
        v = lora_four(row + k);
    } else {
#pragma unroll
        for (int i = 0; i < 3; i++)
            if (k + i < len)
                v[i] = lora_one(row + k + i);
    }
    return v;
}
// 16 bytes of elements as f32: eight, or four of f32.
template <typename T>
__device__ __forceinline__ void lora_wide(lora_u4 u, float *v) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (std::is_same_v<T, float>) {
            v[i] = __uint_as_float(u[i]);
        } else {
            v[2 * i] = std::is_same_v<T, uint16_t> ? __uint_as_float(u[i] << 16) : half_bits_to_float(u[i]);
            v[2 * i + 1] = std::is_same_v<T, uint16_t> ? __uint_as_float(u[i] & 0xffff0000u) : half_bits_to_float(u[i] >> 16);
        }
    }
}
// 16 bytes from element k of a row of `len` on, zero past its end.
template <typename T>
__device__ __forceinline__ lora_u4 lora_raw(const T *row, size_t k, size_t len) {
    constexpr int E = 16 / sizeof(T);
    lora_u4 u = {0, 0, 0, 0};
    if (k + E <= len) {
        u = *(const lora_u4u *)(row + k);
    } else {
#pragma unroll
        for (int i = 0; i < E - 1; i++)
            if (k + i < len) {
                if constexpr (sizeof(T) == 4)
                    u[i] = __float_as_uint(row[k + i]);
                else
                    u[i / 2] |= (uint32_t)((const uint16_t *)row)[k + i] << i % 2 * 16;
            }
    }
    return u;
}
// Eight.
template <typename T>
__device__ __forceinline__ void lora_eight(const T *p, float *v) {
    lora_wide<T>(*(const lora_u4u *)p, v);
    if constexpr (std::is_same_v<T, float>)
        lora_wide<T>(*(const lora_u4u *)(p + 4), v + 4);
}
// The eight from k on of a row of `len`, zero past its end.
template <typename T>
__device__ __forceinline__ void lora_eight_at(const T *row, int k, int len, float (&v)[8]) {
    if (k + 8 <= len) {
        lora_eight(row + k, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            v[i] = k + i < len ? lora_one(row + k + i) : 0.0f;
    }
}
// The sum over aligned groups of L lanes, in all of them.
template <int L>
__device__ __forceinline__ float lora_sum(float v) {
    if constexpr (L >= 2)
        v += dpp_f<0xB1>(v, v);
    if constexpr (L >= 4)
        v += dpp_f<0x4E>(v, v);
    if constexpr (L >= 8)
        v += dpp_f<0x141>(v, v);
    if constexpr (L >= 16)
        v += dpp_f<0x140>(v, v);
    if constexpr (L >= 32)
        v += __shfl_xor(v, 16);
    if constexpr (L >= 64)
        v += __shfl_xor(v, 32);
    return v;
}
__device__ __forceinline__ bool lora_names(const LoraParams &P, int e) { return e >= 0 && (size_t)e < P.n_adapters; }

// ---- few vectors ------------------------------------------------------------------
// y[t][r .. r + RPW): a wave per RPW rows of A_e, a lane every 64th group of eight columns.
template <typename T, int RPW>
__global__ __launch_bounds__(LORA_THREADS) void lora_few_y_kernel(LoraParams P) {
    const size_t t = blockIdx.y;
    const int e = P.ids[t], lane = threadIdx.x & 63;
    const int r0 = (blockIdx.x * (LORA_THREADS / 64) + (threadIdx.x >> 6)) * RPW;
    if (!lora_names(P, e) || r0 >= P.rank)
        return;
    const float *x = P.x + t * P.x_stride;
    const T *a[RPW];
#pragma unroll
    for (int i = 0; i < RPW; i++)
        a[i] = (const T *)P.a + ((size_t)e * P.rank + (r0 + i < P.rank ? r0 + i : P.rank - 1)) * P.cols;
    float s[RPW];
#pragma unroll
    for (int i = 0; i < RPW; i++)
        s[i] = 0.0f;
    const size_t eights = P.cols / 8 * 8;
#pragma unroll 2
    for (size_t k = lane * 8; k < eights; k += 512) {
        float xv[8], av[RPW][8];
        lora_eight(x + k, xv);
#pragma unroll
        for (int i = 0; i < RPW; i++)
            lora_eight(a[i] + k, av[i]);
#pragma unroll
        for (int i = 0; i < RPW; i++)
#pragma unroll
            for (int c = 0; c < 8; c++)
                s[i] = __builtin_fmaf(av[i][c], xv[c], s[i]);
    }
    const size_t k = eights + lane;
    if (k < P.cols)
#pragma unroll
        for (int i = 0; i < RPW; i++)
            s[i] = __builtin_fmaf(lora_one(a[i] + k), x[k], s[i]);
#pragma unroll
    for (int i = 0; i < RPW; i++) {
        s[i] = lora_sum<64>(s[i]);
        if (lane == 0 && r0 + i < P.rank)
            P.y[t * P.rp + r0 + i] = s[i] * P.scale[e];
    }
}

// out[t][..]: LPR lanes per row of B_e, each with the same ranks of every row (its part of y stays in registers): Q times
// eight in a row.  LORA_PASSES passes of 64 / LPR rows a wave.
constexpr int LORA_PASSES = 4;
template <typename T, int LPR, int Q>
__global__ __launch_bounds__(LORA_THREADS) void lora_few_out_kernel(LoraParams P) {
    constexpr int RPI = 64 / LPR, W = LORA_THREADS / 64;
    const size_t t = blockIdx.y;
    const int e = P.ids[t], lane = threadIdx.x & 63, sub = lane % LPR;
    const size_t w0 = ((size_t)blockIdx.x * W + (threadIdx.x >> 6)) * (LORA_PASSES * RPI);
    const float *base = P.base ? P.base + t * P.base_stride : nullptr;
    float *out = P.out + t * P.out_stride;
    const bool named = lora_names(P, e);
    const T *b = (const T *)P.b + (named ? (size_t)e * P.rows * P.rank : 0);
    const int rank = P.rank;
    float y[Q][8], v[LORA_PASSES][Q][8], o[LORA_PASSES];
    const auto k_of = [&](int q, int c) { return (q * LPR + sub) * 8 + c; };
    const auto row = [&](int p) { return w0 + p * RPI + lane / LPR; };
    const auto load = [&](auto eight) {
#pragma unroll
        for (int p = 0; p < LORA_PASSES; p++) {
            const size_t at = row(p) < P.rows ? row(p) : P.rows - 1;
            o[p] = base ? base[at] : 0.0f;
#pragma unroll
            for (int q = 0; q < Q; q++)
                eight(b + at * rank, k_of(q, 0), v[p][q]);
        }
    };
    if (rank % 8 == 0) // ranks past the last are the first ones again, and left out of the sum
        load([&](const T *r, int k, float (&v)[8]) { lora_eight(r + (k < rank ? k : 0), v); });
    else
        load([&](const T *r, int k, float (&v)[8]) { lora_eight_at(r, k, rank, v); });
#pragma unroll
    for (int q = 0; q < Q; q++)
#pragma unroll
        for (int c = 0; c < 8; c++)
            y[q][c] = k_of(q, c) < rank ? P.y[t * P.rp + k_of(q, c)] : 0.0f;
#pragma unroll
    for (int p = 0; p < LORA_PASSES; p++) {
        const size_t r = row(p);
        float s = 0.0f;
#pragma unroll
        for (int q = 0; q < Q; q++)
#pragma unroll
            for (int c = 0; c < 8; c++)
                s = k_of(q, 0) < rank ? __builtin_fmaf(v[p][q][c], y[q][c], s) : s;
        s = lora_sum<LPR>(s);
        if (sub == 0 && r < P.rows)
            out[r] = named ? o[p] + s : o[p];
    }
}

// Both steps in one launch, where A_e is small: a work group forms the vector's whole y for itself, LPR * 8 / 16 rows of
// A_e a wave, then its rows of B_e; the first of those are loaded before y is formed.
constexpr int LORA_ONE = 1024;
template <typename T, int LPR>
__global__ __launch_bounds__(LORA_ONE) void lora_one_kernel(LoraParams P) {
    constexpr int W = LORA_ONE / 64, RPI = 64 / LPR, R = LPR > 2 ? LPR / 2 : 1;
    __shared__ float ys[W * R];
    const size_t t = blockIdx.y, step = (size_t)gridDim.x * W * RPI;
    const int e = P.ids[t], lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane % LPR, rank = P.rank;
    const float *x = P.x + t * P.x_stride, *base = P.base ? P.base + t * P.base_stride : nullptr;
    float *out = P.out + t * P.out_stride;
    const bool named = lora_names(P, e);
    const T *a = (const T *)P.a + (named ? (size_t)e * rank * P.cols : 0);
    const T *b = (const T *)P.b + (named ? (size_t)e * P.rows * rank : 0);
    float v[8], o;
    const auto load = [&](size_t r0) {
        const size_t r = r0 + lane / LPR, at = r < P.rows ? r : P.rows - 1;
        o = base ? base[at] : 0.0f;
        lora_eight_at(b + at * rank, sub * 8, rank, v);
    };
    size_t r0 = ((size_t)blockIdx.x * W + wave) * RPI;
    load(r0);
    if (named && wave * R < rank) {
        const T *ar[R];
        float s[R] = {};
#pragma unroll
        for (int i = 0; i < R; i++)
            ar[i] = a + (size_t)(wave * R + i < rank ? wave * R + i : 0) * P.cols;
        const size_t eights = P.cols / 8 * 8;
#pragma unroll 4
        for (size_t c = lane * 8; c < eights; c += 512) {
            float xv[8], av[8];
            lora_eight(x + c, xv);
#pragma unroll
            for (int i = 0; i < R; i++) {
                lora_eight(ar[i] + c, av);
#pragma unroll
                for (int j = 0; j < 8; j++)
                    s[i] = __builtin_fmaf(av[j], xv[j], s[i]);
            }
        }
        const size_t c = eights + lane;
        if (c < P.cols)
#pragma unroll
            for (int i = 0; i < R; i++)
                s[i] = __builtin_fmaf(lora_one(ar[i] + c), x[c], s[i]);
#pragma unroll
        for (int i = 0; i < R; i++) {
            const float y = lora_sum<64>(s[i]) * P.scale[e];
            if (lane == 0)
                ys[wave * R + i] = y;
        }
    }
    __syncthreads();
    float y[8];
#pragma unroll
    for (int c = 0; c < 8; c++)
        y[c] = named && sub * 8 + c < rank ? ys[sub * 8 + c] : 0.0f;
    while (r0 < P.rows) {
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < 8; c++)
            s = __builtin_fmaf(v[c], y[c], s);
        s = lora_sum<LPR>(s);
        const size_t r = r0 + lane / LPR;
        const float sum = named ? o + s : o;
        r0 += step;
        if (r0 < P.rows)
            load(r0);
        if (sub == 0 && r < P.rows)
            out[r] = sum;
    }
}

// ---- many vectors -----------------------------------------------------------------
// Tiles of v_mfma_f32_16x16x4_f32 with 16 vectors as columns: lane l has column l % 16 and one of four contracted
// indices, l / 16.  Which four a product takes is free as long as both operands agree: lane group g has those of its 16
// bytes.  The result: column l % 16, rows 4 (l / 16) + i.

// The vectors of a block of LORA_BLOCK that name an adapter, put together by it: tiles of up to 16 vectors that name one.
// Which vectors share an adapter follows from a ballot for each bit of its number, where its tiles begin from a scan.
constexpr int LORA_BLOCK = 128;
struct LoraTiles {
    int key[LORA_BLOCK], first[LORA_BLOCK]; // of each vector its adapter (-1: none); of an adapter's first one its first tile
    int adapter[LORA_BLOCK];                // of each tile
    short vec[LORA_BLOCK][16];              // of each tile its vectors, -1 past the last
    int total[2];                           // tiles whose adapter's first vector is in each half
};
__device__ __forceinline__ int lora_tiles(const LoraParams &P, size_t t0, LoraTiles &L) {
    static_assert(LORA_BLOCK == 128, "two waves");
    const int i = threadIdx.x, wave = i >> 6, lane = i & 63;
    const int here = P.n - t0 < LORA_BLOCK ? (int)(P.n - t0) : LORA_BLOCK;
    if (i < LORA_BLOCK) {
        const int id = i < here ? P.ids[t0 + i] : -1;
        L.key[i] = lora_names(P, id) ? id : -1;
    }
    for (int c = i; c < LORA_BLOCK * 8; c += blockDim.x)
        ((int *)&L.vec[0][0])[c] = -1;
    __syncthreads();
    int key = -1, before = 0, lead = 0;
    if (wave < 2) {
        const int k0 = L.key[lane], k1 = L.key[64 + lane];
        key = wave ? k1 : k0;
        // the vectors of each half that name the same adapter, bit by bit of its number
        unsigned long long m0 = __ballot(k0 >= 0), m1 = __ballot(k1 >= 0);
        for (int bit = 0; (P.n_adapters - 1) >> bit; bit++) {
            const unsigned long long b0 = __ballot(k0 >> bit & 1), b1 = __ballot(k1 >> bit & 1);
            const unsigned long long flip = key >> bit & 1 ? 0 : ~0ull;
            m0 &= b0 ^ flip;
            m1 &= b1 ^ flip;
        }
        const unsigned long long under = (1ull << lane) - 1;
        before = wave ? __popcll(m0) + __popcll(m1 & under) : __popcll(m0 & under);
        lead = m0 ? __builtin_ctzll(m0) : m1 ? 64 + __builtin_ctzll(m1) : 0;
        const int mine = key >= 0 && before == 0 ? (__popcll(m0) + __popcll(m1) + 15) / 16 : 0;
        int sum = mine; // up to and with this vector's
        for (int o = 1; o < 64; o *= 2) {
            const int up = __shfl_up(sum, o);
            sum += lane >= o ? up : 0;
        }
        L.first[i] = sum - mine;
        if (lane == 63)
            L.total[wave] = sum;
    }
    __syncthreads();
    if (wave < 2 && key >= 0) {
        const int tile = L.first[lead] + (lead < 64 ? 0 : L.total[0]) + before / 16;
        L.vec[tile][before % 16] = (short)i;
        L.adapter[tile] = key;
    }
    __syncthreads();
    return L.total[0] + L.total[1];
}

// y for every LORA_Z-th tile of a block and one of ks splits of the columns: W waves take an equal part each, their sums
// meet in LDS.  The second launch adds the splits, once a work group, so there are as few as fill the chip.  RT: tiles
// of 16 ranks.  A wave reads 128 bytes of every row of A_e and the same columns of x at a time, whole cache lines in one
// instruction, and gives them their places through a piece of LDS of its own: loaded as the products want them, 16 rows a
// quarter line each, rows a power of two apart throw each other's lines out of the cache (4096 columns, rank 64, 1408
// vectors: 41 us for 27 this way).
constexpr int LORA_Z = LORA_BLOCK / 16;
__host__ __device__ constexpr int lora_y_waves(int rt) { return rt <= 8 ? 8 : 4; }
template <typename T, int RT>
__global__ __launch_bounds__(64 * lora_y_waves(RT)) void lora_many_y_kernel(LoraParams P) {
    constexpr int W = lora_y_waves(RT), E = 16 / sizeof(T), KC = 8 * E; // elements of 16 and of 128 bytes of A_e
    constexpr int XC = KC / 4, XL = KC / 16;                            // 16-byte pieces of a row of x, loads of 16 rows
    constexpr int RB = RT < 4 ? RT : 4;                                 // tiles of A_e in LDS at a time
    constexpr int XS = KC * 4 + 16, AS = 128 + 16, STAGE = 16 * XS + RB * 16 * AS;
    constexpr int PARTS = W * RT * 64 * 16;
    __shared__ char smem[W * STAGE > PARTS ? W * STAGE : PARTS] __attribute__((aligned(16)));
    __shared__ LoraTiles L;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
    lora_f4 *const part = (lora_f4 *)smem; // [W][RT][64], once the columns are done
    char *const xs = smem + wave * STAGE, *const as = xs + 16 * XS;
    const size_t t0 = (size_t)blockIdx.x * LORA_BLOCK;
    const int tiles = lora_tiles(P, t0, L);
    const size_t share = (P.cols + KC * W * P.ks - 1) / (KC * W * P.ks) * KC; // columns a wave
    const size_t k0 = (blockIdx.z * W + wave) * share, k1 = k0 + share < P.cols ? k0 + share : P.cols;
    for (int tile = blockIdx.y; tile < tiles; tile += LORA_Z) {
        const int e = L.adapter[tile];
        const T *a = (const T *)P.a + (size_t)e * P.rank * P.cols;
        const float *x[XL];
        const T *ar[RT][2];
#pragma unroll
        for (int i = 0; i < XL; i++) {
            const int v = L.vec[tile][i * (64 / XC) + lane / XC];
            x[i] = P.x + (t0 + (v < 0 ? L.vec[tile][0] : v)) * P.x_stride;
        }
#pragma unroll
        for (int r = 0; r < RT; r++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                // ranks past the last: the last one's, dropped with the rows of y
                const int row = r * 16 + h * 8 + lane / 8;
                ar[r][h] = a + (size_t)(row < P.rank ? row : P.rank - 1) * P.cols;
            }
        lora_f4 xv[XL];
        lora_u4 av[RT][2];
        const auto load = [&](size_t k) {
#pragma unroll
            for (int i = 0; i < XL; i++)
                xv[i] = lora_at(x[i], k + lane % XC * 4, k1);
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                    av[r][h] = lora_raw(ar[r][h], k + lane % 8 * E, k1);
        };
        lora_f4 acc[RT];
#pragma unroll
        for (int r = 0; r < RT; r++)
            acc[r] = lora_f4{0.0f, 0.0f, 0.0f, 0.0f};
        load(k0);
        for (size_t k = k0; k < k1; k += KC) {
            lora_f4 xf[2][E / 4];
#pragma unroll
            for (int i = 0; i < XL; i++)
                *(lora_f4 *)(xs + (i * (64 / XC) + lane / XC) * XS + lane % XC * 16) = xv[i];
#pragma unroll
            for (int r0 = 0; r0 < RT; r0 += RB) {
#pragma unroll
                for (int r = 0; r < RB; r++)
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        *(lora_u4 *)(as + (r * 16 + h * 8 + lane / 8) * AS + lane % 8 * 16) = av[r0 + r][h];
                wave_lds_sync();
                if (r0 == 0)
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int c = 0; c < E / 4; c++)
                            xf[h][c] = *(const lora_f4 *)(xs + col * XS + (h * 4 + g) * E * 4 + c * 16);
                if (r0 + RB == RT)
                    load(k + KC); // while the products run
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int r = 0; r < RB; r++) {
                        float v[E];
                        lora_wide<T>(*(const lora_u4 *)(as + (r * 16 + col) * AS + (h * 4 + g) * 16), v);
#pragma unroll
                        for (int c = 0; c < E; c++)
                            acc[r0 + r] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[c], xf[h][c / 4][c % 4], acc[r0 + r], 0, 0, 0);
                    }
                wave_lds_sync(); // read before the next stores
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RT; r++)
            part[(wave * RT + r) * 64 + lane] = acc[r];
        __syncthreads();
        const int v = L.vec[tile][col];
        for (int r = wave; r < RT; r += W) {
            lora_f4 y = part[r * 64 + lane];
#pragma unroll
            for (int w = 1; w < W; w++)
                y += part[(w * RT + r) * 64 + lane];
            if (v >= 0 && r * 16 < P.rp)
                *(lora_f4 *)(P.y + ((size_t)blockIdx.z * P.n + t0 + v) * P.rp + r * 16 + g * 4) = y * P.scale[e];
        }
        __syncthreads();
    }
}

// out for a block's vectors and 64 rows: a wave every LORA_OW-th tile, M-tile m the rows 16 m + .. of B_e.  The products
// leave a lane 16 bytes of 16 vectors' rows; they meet in LDS, and a wave takes 16 of the block's vectors as they lie, 256
// bytes of a row at a time: base is on its way before the tiles are known, and so is y, whose splits are added on the way
// into LDS (added one after the other where the products want them, rank 64 took 28 us for 22, 1000 vectors x 3001).
// Waves hide each other's loads: held to 128 registers a thread, 136 took 31.
constexpr int LORA_OW = 8, LORA_OUT = 64, LORA_OUT_PAD = LORA_OUT + 4;
template <typename T>
__global__ __launch_bounds__(64 * LORA_OW, 4) void lora_many_out_kernel(LoraParams P) {
    static_assert(LORA_OW * 16 == LORA_BLOCK, "sixteen vectors a wave");
    constexpr int MT = LORA_OUT / 16, E = 16 / sizeof(T); // elements of 16 bytes of B_e
    __shared__ LoraTiles L;
    // [vector][row] and [vector][rank], padded against bank conflicts
    __shared__ float sums[LORA_BLOCK * LORA_OUT_PAD] __attribute__((aligned(16)));
    __shared__ float ys[LORA_BLOCK * LORA_OUT_PAD] __attribute__((aligned(16)));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
    const size_t t0 = (size_t)blockIdx.y * LORA_BLOCK, step = (size_t)gridDim.x * LORA_OUT;
    size_t r0 = (size_t)blockIdx.x * LORA_OUT;
    lora_f4 o[4];
    const auto load = [&](lora_f4 (&o)[4], size_t row) {
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const size_t t = t0 + wave * 16 + p * 4 + g;
            o[p] = lora_f4{0.0f, 0.0f, 0.0f, 0.0f};
            if (P.base && t < P.n)
                o[p] = lora_at(P.base + t * P.base_stride, row, P.rows);
        }
    };
    load(o, r0 + col * 4);
    const int tiles = lora_tiles(P, t0, L);
    // y of the block's vectors, 64 ranks of it, the splits added and zero past the last rank
    const auto stage = [&](int k0) {
        for (int i = threadIdx.x; i < LORA_BLOCK * 16; i += 64 * LORA_OW) {
            const int v = i / 16, k = k0 + i % 16 * 4;
            lora_f4 y = {0.0f, 0.0f, 0.0f, 0.0f};
            if (t0 + v < P.n && k < P.rp)
                for (int s = 0; s < P.ks; s++)
                    y += *(const lora_f4 *)(P.y + ((size_t)s * P.n + t0 + v) * P.rp + k);
#pragma unroll
            for (int c = 0; c < 4; c++)
                y[c] = k + c < P.rank ? y[c] : 0.0f;
            *(lora_f4 *)(ys + v * LORA_OUT_PAD + i % 16 * 4) = y;
        }
    };
    stage(0);
    __syncthreads();
    for (; r0 < P.rows; r0 += step) {
        for (int k0 = 0; k0 < P.rank; k0 += 64) {
            if (P.rank > 64 && (k0 || r0 >= step)) {
                __syncthreads();
                stage(k0);
                __syncthreads();
            }
            for (int tile = wave; tile < tiles; tile += LORA_OW) {
                const int e = L.adapter[tile], v = L.vec[tile][col];
                const T *b = (const T *)P.b + (size_t)e * P.rows * P.rank;
                const float *y = ys + (v < 0 ? L.vec[tile][0] : v) * LORA_OUT_PAD;
                lora_f4 acc[MT];
#pragma unroll
                for (int m = 0; m < MT; m++)
                    acc[m] = k0 && v >= 0 ? *(const lora_f4 *)(sums + v * LORA_OUT_PAD + m * 16 + g * 4)
                                          : lora_f4{0.0f, 0.0f, 0.0f, 0.0f};
                for (int k = k0; k < k0 + 64 && k < P.rank; k += 4 * E) {
                    lora_u4 bv[MT];
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        const size_t r = r0 + m * 16 + col;
                        bv[m] = lora_raw(b + (r < P.rows ? r : P.rows - 1) * P.rank, k + g * E, P.rank);
                    }
                    lora_f4 ye[E / 4];
#pragma unroll
                    for (int c = 0; c < E / 4; c++)
                        ye[c] = *(const lora_f4 *)(y + k - k0 + g * E + c * 4);
#pragma unroll
                    for (int m = 0; m < MT; m++) {
                        float be[E];
                        lora_wide<T>(bv[m], be);
#pragma unroll
                        for (int c = 0; c < E; c++)
                            acc[m] = __builtin_amdgcn_mfma_f32_16x16x4f32(be[c], ye[c / 4][c % 4], acc[m], 0, 0, 0);
                    }
                }
                if (v >= 0)
#pragma unroll
                    for (int m = 0; m < MT; m++)
                        *(lora_f4 *)(sums + v * LORA_OUT_PAD + m * 16 + g * 4) = acc[m];
            }
        }
        __syncthreads();
        const size_t row = r0 + col * 4;
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const int v = wave * 16 + p * 4 + g;
            const size_t t = t0 + v;
            if (t < P.n && L.key[v] >= 0)
                o[p] += *(const lora_f4 *)(sums + v * LORA_OUT_PAD + col * 4);
            float *out = P.out + t * P.out_stride + row;
            if (t < P.n) {
                if (row + 4 <= P.rows) {
                    *(lora_f4u *)out = o[p];
                } else {
#pragma unroll
                    for (int c = 0; c < 3; c++)
                        if (row + c < P.rows)
                            out[c] = o[p][c];
                }
            }
        }
        __syncthreads();
        if (r0 + step < P.rows)
            load(o, r0 + step + col * 4);
    }
}

template <typename T, int LPR, int Q>
static void lora_few_out(const LoraParams &P, hipStream_t st) {
    const size_t rows = (LORA_THREADS / 64) * LORA_PASSES * (64 / LPR);
    hipLaunchKernelGGL((lora_few_out_kernel<T, LPR, Q>), dim3((P.rows + rows - 1) / rows, P.n), dim3(LORA_THREADS), 0, st,
                       P);
}
template <typename T>
static void lora_both(const LoraParams &P, hipStream_t st) {
    // work groups for half the chip, no more: each reads A_e again
    const int lpr = P.rank <= 8 ? 1 : P.rank <= 16 ? 2 : P.rank <= 32 ? 4 : 8;
    const size_t most = (P.rows * lpr + LORA_ONE - 1) / LORA_ONE, want = (128 + P.n - 1) / P.n;
    const dim3 g(want < most ? want : most, P.n);
    if (lpr == 1)
        hipLaunchKernelGGL((lora_one_kernel<T, 1>), g, dim3(LORA_ONE), 0, st, P);
    else if (lpr == 2)
        hipLaunchKernelGGL((lora_one_kernel<T, 2>), g, dim3(LORA_ONE), 0, st, P);
    else if (lpr == 4)
        hipLaunchKernelGGL((lora_one_kernel<T, 4>), g, dim3(LORA_ONE), 0, st, P);
    else
        hipLaunchKernelGGL((lora_one_kernel<T, 8>), g, dim3(LORA_ONE), 0, st, P);
}
template <typename T>
static void lora_few(const LoraParams &P, hipStream_t st) {
    constexpr int W = LORA_THREADS / 64;
    // rows of A_e a wave: one while that leaves the chip few waves, else two (a vector is read once for both)
    const int rpw = P.n * P.rank <= 2048 ? 1 : 2;
    const dim3 gy((P.rank + W * rpw - 1) / (W * rpw), P.n);
    if (rpw == 1)
        hipLaunchKernelGGL((lora_few_y_kernel<T, 1>), gy, dim3(LORA_THREADS), 0, st, P);
    else
        hipLaunchKernelGGL((lora_few_y_kernel<T, 2>), gy, dim3(LORA_THREADS), 0, st, P);
    if (P.rank <= 8)
        lora_few_out<T, 1, 1>(P, st);
    else if (P.rank <= 16)
        lora_few_out<T, 2, 1>(P, st);
    else if (P.rank <= 32)
        lora_few_out<T, 4, 1>(P, st);
    else if (P.rank <= 64)
        lora_few_out<T, 8, 1>(P, st);
    else if (P.rank <= 128)
        lora_few_out<T, 16, 1>(P, st);
    else
        lora_few_out<T, 16, 2>(P, st);
}

template <typename T, int RT>
static void lora_many_y(const LoraParams &P, hipStream_t st) {
    hipLaunchKernelGGL((lora_many_y_kernel<T, RT>), dim3((P.n + LORA_BLOCK - 1) / LORA_BLOCK, LORA_Z, P.ks),
                       dim3(64 * lora_y_waves(RT)), 0, st, P);
}
template <typename T>
static void lora_many(const LoraParams &P, hipStream_t st) {
    if (P.rp <= 16)
        lora_many_y<T, 1>(P, st);
    else if (P.rp <= 32)
        lora_many_y<T, 2>(P, st);
    else if (P.rp <= 64)
        lora_many_y<T, 4>(P, st);
    else if (P.rp <= 128)
        lora_many_y<T, 8>(P, st);
    else
        lora_many_y<T, 16>(P, st);
    const size_t blocks = (P.n + LORA_BLOCK - 1) / LORA_BLOCK, parts = (P.rows + LORA_OUT - 1) / LORA_OUT;
    // work groups that the chip holds at once, each on through the rows: 2048 x 4096 x rank 32 20.4 us, one a part 24.4
    const size_t want = (512 + blocks - 1) / blocks;
    const dim3 g(want < parts ? want : parts, blocks);
    hipLaunchKernelGGL((lora_many_out_kernel<T>), g, dim3(64 * LORA_OW), 0, st, P);
}

// Whether the vectors are taken one by one: while all their reads of A_e and B_e, mostly from L2, stay under LORA_FEW
// bytes.  Measured at 4096 x 2048, rank 64, fp16 (bf16 the same): 101 MB (128 vectors) 18 us one by one, 21 as tiles, 28
// as tiles of mixed requests; 201 MB 30, 21, 29; 403 MB 54, 23, 33.  f32: 101 MB (64 vectors) 13, 19; 201 MB 20, 21, 30;
// 403 MB 36, 22, 30.  Rank 16, fp16: 101 MB 15, 18, 23; 201 MB 24, 23, 28.  At rank 256 the line lies too low (201 MB, 64
// vectors, 41 for 55).
template <class L>
static bool lora_is_few(const L &l, size_t n, size_t es) {
    return n <= 65535 && (double)n * l.rank * (l.rows + l.cols) * es <= LORA_FEW;
}
// Of those, whether one launch does both steps: the second costs the host 3.5 us, and each work group reads A_e again.
// Measured, in a graph, against two launches, fp16: A_e of 64 KB, rank 8, 1 vector 4.2 us for 5.1, 256 6.2 for 7.2; of
// 128 KB, rank 16, 1 vector 5.5 for 5.3, 32 6.2 for 5.5, 256 9.3 for 10.1; rank 64, 1 vector 5.0 for 5.1, 32 8.1 for 7.3.
// f32: 64 KB, rank 8, 1 vector 4.3 for 5.6, 32 4.5 for 5.9, 256 6.3 for 8.1; 128 KB, rank 16, 5.2 for 5.7, 5.9 for 5.9,
// 10.1 for 11.2; 256 KB, rank 64, 1 vector 6.4 for 5.8.
template <class L>
static bool lora_is_one(const L &l, size_t n, size_t es) {
    return lora_is_few(l, n, es) && l.rank <= 64 && l.rank * l.cols * es <= LORA_SMALL;
}
// Returns the launches.
template <typename T>
static int lora_run(const LoraParams &P, hipStream_t st) {
    if (lora_is_one(P, P.n, sizeof(T))) {
        lora_both<T>(P, st);
        return 1;
    }
    if (lora_is_few(P, P.n, sizeof(T)))
        lora_few<T>(P, st);
    else
        lora_many<T>(P, st);
    return 2;
}

// Splits of the columns: a work group for every CU, none under 512 columns.
static int lora_splits(size_t cols, size_t n) {
    const size_t tiles = (n + 15) / 16, s = (256 + tiles - 1) / tiles, most = (cols + 511) / 512;
    return (int)(s > most ? most : s > 4 ? 4 : s);
}
static size_t lora_ws_bytes(const loomhip_lora *l, size_t n) {
    if (lora_is_one(*l, n, l->type == LH_F32 ? 4 : 2))
        return 0;
    return lora_splits(l->cols, n) * n * ((l->rank + 15) / 16 * 16) * 4;
}

} // namespace lh

using namespace lh;

extern "C" {

size_t loomhip_lora_ws(const loomhip_lora *l, size_t n) {
    return l && n && n <= LORA_MAX_N && l->rank && l->rank <= LORA_MAX_RANK && l->cols && l->rows ? lora_ws_bytes(l, n) : 0;
}

int loomhip_lora_dev(const loomhip_lora *l, const float *x, size_t x_stride, const int32_t *ids, const float *base,
                     size_t base_stride, size_t n, float *out, size_t out_stride, void *ws, size_t ws_bytes,
                     void *stream) {
    LoraParams P;
    if (int rc = lora_check(l, x, x_stride, ids, base, base_stride, n, out, out_stride, P))
        return rc;
    if (n == 0)
        return LOOMHIP_OK;
    const size_t need = lora_ws_bytes(l, n);
    if (need && (!ws || ws_bytes < need || (uintptr_t)ws % 16))
        return fail(LOOMHIP_ERR_ARG, "lora: the workspace takes %zu bytes at a multiple of 16, got %zu", need, ws_bytes);
    if (int rc = require_device())
        return rc;
    P.y = (float *)ws;
    P.rp = (int)((l->rank + 15) / 16 * 16);
    P.ks = lora_splits(l->cols, n);
    hipStream_t st = stream_of(stream);
    const int launches = l->type == LH_F32   ? lora_run<float>(P, st)
                         : l->type == LH_F16 ? lora_run<_Float16>(P, st)
                                             : lora_run<uint16_t>(P, st);
    for (int i = 0; i < launches; i++)
        note_launch();
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? LOOMHIP_OK : hip_fail(e, "lora launch");
}

} // extern "C"

// paged_attn.hip -- attention of one new token of every lane over its pages.
//
//   out = sum_t p_t v_t,  p = softmax of scale * (q . k_t) over the rows t seen
//
// The query heads of a key head (up to 16) are the columns of the matrix
// products.  A work group's four waves take a lane's rows in turn, a tile
// of rows each: no wave waits for another before the end, where their running
// maxima, sums and products are joined.
//
// Products on the matrix cores, in the cache's own type (mfma 16x16x32), exact
// in the cached values and near f32 in the others: an f16 cache takes the query
// (scaled by a power of two of its own) and the weights in two f16 parts (22
// bits; what is far below the largest of them to within 2^-38 of that), a bf16
// cache in three bf16 parts (24).  The sums are f32.
//
// S^T = K Q^T: a lane holds one query head (column lane % 16) and, of each 32
// rows, the rows 4 (lane / 16) + i and 16 + 4 (lane / 16) + i, i < 4.  These
// eight weights are the B operand of O^T = V^T P^T as they stand, if its 8
// contracted indices mean those rows; the A operand's lane then needs the same
// rows of one value column, which two LDS transpose reads (ds_read_b64_tr_b16)
// give from row-major values.
//
// Bound by the bytes of the rows: a wave's tile is loaded into registers (a
// page's rows wherever they lie, 16 bytes a thread), put into LDS when the wave
// is through with the one before, and the next tile's loads go out; two work
// groups a CU keep up to 128 KB in flight, and the products (512 cycles of a
// tile's 7500) hide behind them.  Measured, 32 heads of 128 over 4 key heads: 8
// lanes of up to 65536 rows, bf16, 103 us (604 MB, 5.9 TB/s, where a plain read
// of that many bytes runs at 7.0: work groups start and end together, and
// pieces are up to a twentieth longer than the share), 32 lanes of up to 4096,
// f16, 29 us (139 MB, 4.8 TB/s: lengths, plan and pages one after the other stand
// before the first tiles) and 5 for the records; one lane of 256 rows 6.9.
#include "runtime.hpp"

#include <type_traits>

namespace lh {

typedef _Float16 pg_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 pg_b8 __attribute__((ext_vector_type(8)));
typedef short pg_s4 __attribute__((ext_vector_type(4)));
typedef float pg_f4 __attribute__((ext_vector_type(4)));
typedef uint32_t pg_u4 __attribute__((ext_vector_type(4)));

int pages_check(const loomhip_pages *c, size_t n_kv, size_t hd, const char *fn);

constexpr int PG_THREADS = 256, PG_WAVES = PG_THREADS / 64;
constexpr int PG_MAX_HD = 256;
constexpr int PG_COLS = 16; // query heads of an item
// Rows up to which no lane is cut (a launch less, but an item's rows one tile of a wave after the other); half as many at
// head sizes over 128.  Measured, in a graph, 1, 8 and 64 lanes of 32 heads of 128 over 4, whole against cut: 256 rows
// 6.7, 7.3, 8.3 us for 10.3, 10.9, 14.6; 512 rows 9.5, 11.2, 12.9 for 10.5, 11.3, 18; 1024 rows 17, 20, 23 for 11, 12,
// 24.  Of 8 heads of 256 over 2: 256 rows 11.5, 12.8, 13.9 for 14.1, 15.1, 16.1; 512 rows 21, 22, 23 for 14.8, 16, 21.
constexpr size_t PG_WHOLE = 512;

// f16: two parts of a value, of a size that the second is normal; bf16: three, of f32's own range.
struct PgF16 {
    typedef pg_h8 v8;
    typedef _Float16 elem;
    static constexpr int PARTS = 2;
    // weights are 2^(s - m + shift), at most 2^14: their second parts stay normal
    static __device__ __forceinline__ float shift(uint32_t) { return 14.0f; }
    static __device__ __forceinline__ pg_f4 mfma(v8 a, v8 b, pg_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
struct PgBf16 {
    typedef pg_b8 v8;
    typedef __bf16 elem;
    static constexpr int PARTS = 3;
    // Values reach as far as f32: all weights of a lane's rows together are less than 1/2, so that no sum of products is
    // larger than the largest value.  No smaller than that takes, for the weights themselves end at 2^-126.
    static __device__ __forceinline__ float shift(uint32_t rows) { return (float)(__clz((int)rows) - 33); }
    static __device__ __forceinline__ pg_f4 mfma(v8 a, v8 b, pg_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <class T>
__device__ __forceinline__ void pg_split(float x, int e, typename T::v8 (&p)[T::PARTS]) {
#pragma unroll
    for (int i = 0; i < T::PARTS; i++) {
        const typename T::elem h = (typename T::elem)x;
        p[i][e] = h;
        x -= (float)h;
    }
}

// A record's item (lane, key head, block, numbered in this order; -1 but for an item's first record) and how many it has.
struct PgDesc {
    int32_t item, pieces;
};

struct PagedAttnParams {
    loomhip_pages c;
    const float *q;
    const int32_t *len;
    int n, n_heads, n_kv, hd, group, blocks; // group: query heads of a key head, in `blocks` blocks of PG_COLS
    uint32_t window;                         // 0: none
    uint32_t page_mul, page_shift;           // pg_page
    uint32_t page_units, row_units;          // from page to page and row to row, in 16 bytes
    float scale;
    float *out;
    int cols;          // query heads of a record
    uint32_t *records; // how many were left
    PgDesc *desc;      // [records]
    float2 *ml;        // [records][cols]
    float *part;       // [records][cols][hd]
};

// r / page_size for r < 2^31: with 2^(l - 1) < page_size <= 2^l and m = floor(2^(31 + l) / page_size) + 1, which has 32
// bits, m page_size is past 2^(31 + l) by at most 2^l, so r m / 2^(31 + l) is past r / page_size by less than 1 / page_size.
__device__ __forceinline__ uint32_t pg_page(const PagedAttnParams &P, uint32_t r) {
    return P.page_mul ? __umulhi(r, P.page_mul) >> P.page_shift : r;
}
// Rows [first, end) that lane i sees.
__device__ __forceinline__ void pg_span(const PagedAttnParams &P, int i, uint32_t &first, uint32_t &end) {
    const uint32_t most = (uint32_t)(P.c.page_size * P.c.table_width);
    const int len = P.len[i];
    end = len < 0 ? 0 : (uint32_t)len < most ? (uint32_t)len : most;
    first = P.window && P.window < end ? end - P.window : 0;
}

// A value and its row's partners in the other three rows of 16 lanes.
__device__ __forceinline__ float pg_max4(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float pg_sum4(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Tile rows are padded in LDS so that fragment reads spread over the banks: keys
// are read as 16 bytes of sixteen rows, values as 32 bytes of four rows.
template <int HDP>
struct PgCfg {
    static constexpr int KT = HDP == 64 ? 64 : 32;   // rows of a wave's tile
    static constexpr int CH = HDP / 8, RPI = 64 / CH; // 16-byte chunks of a row, rows a load instruction takes
    static constexpr int NL = KT / RPI;              // loads of a tile's keys, and of its values
    static constexpr int KS = HDP * 2 + 16, VS = HDP * 2 + 32, VO = KT * KS;
    static constexpr int WAVE = KT * (KS + VS); // bytes of a wave's tile
    static constexpr int OS = HDP + 4;          // floats from a head's joined sums to the next
    static constexpr int JOIN = PG_COLS * OS * 4;
    static constexpr int BYTES = PG_WAVES * (WAVE > JOIN ? WAVE : JOIN);
};

// Query heads [h0, h0 + heads) of lane i, which sees `rows` rows and reads key
// head kvh, against its rows [r0, r1): the four waves' (m, l, o), in LDS.
template <class T, int HDP, bool ONCE, bool EARLY>
__device__ __forceinline__ void pg_rows(const PagedAttnParams &P, int i, int kvh, int h0, int heads, uint32_t rows,
                                        uint32_t r0, uint32_t r1, char *smem, float (*sm)[PG_COLS],
                                        float (*sl)[PG_COLS]) {
    using C = PgCfg<HDP>;
    constexpr int STEPS = HDP / 32, DB = HDP / 16, NB = C::KT / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, quad = lane >> 4, col = lane & 15;
    const int hd = P.hd;
    const float shift = T::shift(rows);
    char *tile = smem + wave * C::WAVE;

    // the page of the lane's row (lane % KT) of the tile that starts at row `at`; the first two tiles' are on their way
    // while the query is split
    const int32_t *table = P.c.table + (size_t)i * P.c.table_stride;
    const auto page_of = [&](uint32_t at) {
        const uint32_t r = at + lane % C::KT;
        return r < r1 ? table[pg_page(P, r)] : -1;
    };
    uint32_t at = r0 + wave * C::KT, unit;
    const int32_t page = page_of(at);
    int32_t next = page_of(at + PG_WAVES * C::KT);

    // the query's parts: 8 (lane / 16) + j of every 32 values
    pg_f4 qv[STEPS][2];
    {
        const float *q = P.q + ((size_t)i * P.n_heads + h0 + (col < heads ? col : 0)) * hd;
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int d = s * 32 + quad * 8;
            qv[s][0] = *(const pg_f4 *)(q + (d < hd ? d : 0));
            qv[s][1] = *(const pg_f4 *)(q + (d < hd ? d : 0) + 4);
        }
    }
    typename T::v8 qp[STEPS][T::PARTS];
    float cs = P.scale * 0x1.715476p+0f; // scores in log2 units
    const auto split = [&] {
        float amax = 0.0f, f = 1.0f;
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const bool in = col < heads && s * 32 + quad * 8 < hd;
                qv[s][e / 4][e % 4] = in ? qv[s][e / 4][e % 4] : 0.0f;
                amax = fmaxf(amax, fabsf(qv[s][e / 4][e % 4]));
            }
        if (T::PARTS == 2) { // the largest element brought to 2^13 .. 2^14
            amax = pg_max4(amax);
            const int e = (int)(__float_as_uint(amax) >> 23);
            const int k = e > 0 && e < 255 ? (140 - e > 120 ? 120 : 140 - e < -120 ? -120 : 140 - e) : 0;
            f = __uint_as_float((uint32_t)(127 + k) << 23);
            cs *= __uint_as_float((uint32_t)(127 - k) << 23);
        }
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int e = 0; e < 8; e++)
                pg_split<T>(qv[s][e / 4][e % 4] * f, e, qp[s]);
    };
    // The first tile's loads go out before the query is split (EARLY) or after.  Measured, before and after: 100 lanes of up
    // to 4096 rows, heads of 128, 98.8 us and 104.7, 8 of up to 65536 110 and 113; one lane of 256 rows 7.0 and 6.8, 8 of up
    // to 30000, heads of 256, 64.9 and 63.2.
    if (EARLY)
        __builtin_amdgcn_sched_barrier(0);
    else
        split();

    // staging: the lane's chunk of a row, the first of its rows
    const int chunk = (lane % C::CH) * 8 < hd ? lane % C::CH : hd / 8 - 1; // past the head's end: the last one again
    const uint16_t *kb = (const uint16_t *)P.c.k + (size_t)kvh * P.c.head_stride + chunk * 8;
    const uint16_t *vb = (const uint16_t *)P.c.v + (size_t)kvh * P.c.head_stride + chunk * 8;
    pg_u4 rk[C::NL], rv[C::NL];
    // The tile that starts at row `at`: where the lane's row begins, in 16-byte units, and which rows are there.  A row
    // that is not (past the end, on no page) is loaded as the pool's first.
    const auto place = [&](uint32_t at, int32_t page, uint32_t &unit) {
        const uint32_t r = at + lane % C::KT;
        const bool in = r < r1 && page >= 0 && (uint32_t)page < (uint32_t)P.c.n_pages;
        unit = in ? (uint32_t)page * P.page_units + (r - pg_page(P, r) * (uint32_t)P.c.page_size) * P.row_units : 0u;
        return __ballot(in);
    };
    // The rows' chunks, their places from the lanes that have them.  Rows that one item alone reads (ONCE) pass the caches
    // by: 604 MB and the records take 111 us, with plain loads 121; 139 MB 34.4 and 37.3.  Where four blocks of heads share
    // them, 307 MB in all, 70 us and 65 (41 with the blocks on one XCD, pg_turn).
    const auto load = [&](uint32_t unit) {
        uint32_t from[C::NL];
#pragma unroll
        for (int c = 0; c < C::NL; c++)
            from[c] = (uint32_t)__shfl((int)unit, c * C::RPI + lane / C::CH);
        if constexpr (ONCE) {
#pragma unroll
            for (int c = 0; c < C::NL; c++) {
                rk[c] = __builtin_nontemporal_load((const pg_u4 *)(kb + (size_t)from[c] * 8));
                rv[c] = __builtin_nontemporal_load((const pg_u4 *)(vb + (size_t)from[c] * 8));
            }
        } else {
#pragma unroll
            for (int c = 0; c < C::NL; c++) {
                rk[c] = *(const pg_u4 *)(kb + (size_t)from[c] * 8);
                rv[c] = *(const pg_u4 *)(vb + (size_t)from[c] * 8);
            }
        }
    };

    constexpr uint64_t ALL = C::KT == 64 ? ~0ull : (1ull << 32) - 1;
    uint64_t live = place(at, page, unit) & ALL;
    if (at < r1)
        load(unit);
    if (EARLY) {
        __builtin_amdgcn_sched_barrier(0);
        split();
    }

    pg_f4 o[DB];
#pragma unroll
    for (int b = 0; b < DB; b++)
        o[b] = pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -__builtin_inff(), l = 0.0f;

    const int st = (lane / C::CH) * C::KS + (lane % C::CH) * 16, vt = C::VO + (lane / C::CH) * C::VS + (lane % C::CH) * 16;
    const int k_at = col * C::KS + quad * 16, v_at = C::VO + (4 * quad + (col >> 2)) * C::VS + 8 * (col & 3);
    const auto value_frag = [&](int b, int db) {
        const auto at = (__attribute__((address_space(3))) char *)(tile + v_at) + b * 32 * C::VS + db * 32;
        const pg_s4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pg_s4 *)at);
        const pg_s4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pg_s4 *)(at + 16 * C::VS));
        return __builtin_bit_cast(typename T::v8, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
    };

    for (; at < r1; at += PG_WAVES * C::KT) {
        const uint64_t here = live;
        live = place(at + PG_WAVES * C::KT, next, unit) & ALL;
        next = page_of(at + 2 * PG_WAVES * C::KT);
        wave_lds_sync(); // the reads of the tile before
#pragma unroll
        for (int c = 0; c < C::NL; c++) {
            *(pg_u4 *)(tile + st + c * C::RPI * C::KS) = rk[c];
            if (here != ALL && !(here >> (c * C::RPI + lane / C::CH) & 1))
                rv[c] = pg_u4{0, 0, 0, 0}; // a weight of zero times what lies there
            *(pg_u4 *)(tile + vt + c * C::RPI * C::VS) = rv[c];
        }
        if (at + PG_WAVES * C::KT < r1)
            load(unit);
        wave_lds_sync();
        if (here == 0)
            continue;
        float s[NB][8], mx = -__builtin_inff();
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                pg_f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int x = 0; x < STEPS; x++) {
                    const auto kf = *(const typename T::v8 *)(tile + k_at + (b * 32 + h * 16) * C::KS + x * 64);
#pragma unroll
                    for (int p = T::PARTS - 1; p >= 0; p--)
                        acc = T::mfma(kf, qp[x][p], acc);
                }
#pragma unroll
                for (int e = 0; e < 4; e++)
                    s[b][h * 4 + e] = acc[e] * cs;
            }
        if (here != ALL) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (!(here >> (b * 32 + (e / 4) * 16 + quad * 4 + e % 4) & 1))
                        s[b][e] = -__builtin_inff();
        }
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 8; e++)
                mx = fmaxf(mx, s[b][e]);
        if (__any(mx > m)) {
            const float m2 = fmaxf(m, pg_max4(mx));
            const float f = m == m2 ? 1.0f : __builtin_amdgcn_exp2f(m - m2); // 0 at the first
            m = m2;
            l *= f;
#pragma unroll
            for (int b = 0; b < DB; b++)
                o[b] *= f;
        }
        const float top = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            typename T::v8 pp[T::PARTS];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float w = __builtin_amdgcn_exp2f(s[b][e] - top + shift); // in this order: the shift is lost in a large m
                l += w;
                pg_split<T>(w, e, pp);
            }
#pragma unroll
            for (int d = 0; d < DB; d++) {
                const auto vf = value_frag(b, d);
#pragma unroll
                for (int p = T::PARTS - 1; p >= 0; p--)
                    o[d] = T::mfma(vf, pp[p], o[d]);
            }
        }
    }
    l = pg_sum4(l);
    m = pg_max4(m); // equal already
    __syncthreads(); // all tiles are read: their room is the join's
    float *so = (float *)smem + wave * PG_COLS * C::OS + col * C::OS + quad * 4;
#pragma unroll
    for (int b = 0; b < DB; b++)
        *(pg_f4 *)(so + b * 16) = o[b];
    if (quad == 0)
        sm[wave][col] = m, sl[wave][col] = l;
    __syncthreads();
}

// What the waves left joined, for the thread's head and four columns: 2^(m - M) o summed, and M and l.
template <int HDP>
__device__ __forceinline__ pg_f4 pg_join(const char *smem, float (*sm)[PG_COLS], float (*sl)[PG_COLS], int h, int d,
                                         float &M, float &L) {
    using C = PgCfg<HDP>;
    const float *so = (const float *)smem;
    M = sm[0][h];
#pragma unroll
    for (int w = 1; w < PG_WAVES; w++)
        M = fmaxf(M, sm[w][h]);
    L = 0.0f;
    pg_f4 a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < PG_WAVES; w++) {
        const float f = sm[w][h] == M ? 1.0f : __builtin_amdgcn_exp2f(sm[w][h] - M);
        L += sl[w][h] * f;
        a += *(const pg_f4 *)(so + (w * PG_COLS + h) * C::OS + d) * f;
    }
    return a;
}
// The result of sums a and L: zero where nothing was seen.  An infinity here comes from a cached one (sums of finite values
// stay finite), which the weights' second parts turn into NaN for some heads and not for others: NaN for all.
__device__ __forceinline__ pg_f4 pg_result(pg_f4 a, float L) {
    a *= L == 0.0f ? 0.0f : 1.0f / L;
    return a + a * 0.0f;
}

// Which of `all` pieces work group x takes: those of the blocks of heads that read the same rows (side by side in the
// pieces' order) on one of the eight XCDs, to which work groups go in turn.
__device__ __forceinline__ uint32_t pg_turn(const PagedAttnParams &P, uint32_t x, uint32_t all) {
    const uint32_t blocks = (uint32_t)P.blocks, span = 8 * blocks, g = x / span, r = x - g * span;
    return blocks == 1 || (g + 1) * span > all ? x : g * span + r % 8 * blocks + r / 8;
}

template <int HDP>
constexpr int pg_groups = HDP == 256 ? 1 : 2;                        // work groups of a CU (LDS and registers)
constexpr int pg_room(size_t hd) { return hd > 128 ? 256 : 512; } // work groups that run at a time

// One item (lane, key head, block of its query heads) a work group: all of the lane's rows.
template <class T, int HDP, bool ONCE>
__global__ __launch_bounds__(PG_THREADS, pg_groups<HDP>) void paged_attn_kernel(PagedAttnParams P) {
    using C = PgCfg<HDP>;
    __shared__ __attribute__((aligned(16))) char smem[C::BYTES];
    __shared__ float sm[PG_WAVES][PG_COLS], sl[PG_WAVES][PG_COLS];
    const int w = (int)pg_turn(P, blockIdx.x, gridDim.x);
    const int block = w % P.blocks, ik = w / P.blocks, i = ik / P.n_kv, kvh = ik - i * P.n_kv;
    const int h0 = kvh * P.group + block * PG_COLS;
    const int heads = P.group - block * PG_COLS < PG_COLS ? P.group - block * PG_COLS : PG_COLS;
    uint32_t r0, r1;
    pg_span(P, i, r0, r1);
    pg_rows<T, HDP, ONCE, false>(P, i, kvh, h0, heads, r1 - r0, r0, r1, smem, sm, sl);
    for (int x = threadIdx.x; x < heads * (HDP / 4); x += PG_THREADS) {
        const int h = x / (HDP / 4), d = x % (HDP / 4) * 4;
        float M, L;
        const pg_f4 a = pg_join<HDP>(smem, sm, sl, h, d, M, L);
        if (d < P.hd)
            *(pg_f4 *)(P.out + ((size_t)i * P.n_heads + h0 + h) * P.hd + d) = pg_result(a, L);
    }
}

// The sum of a value over the wave's lanes up to this one: shifts by 1, 2, 4 and 8 in the rows of 16 lanes, then the rows'
// totals carried on.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t pg_dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ uint32_t pg_scan(uint32_t v) {
    v += pg_dpp<0x111, 0xF>(v);
    v += pg_dpp<0x112, 0xF>(v);
    v += pg_dpp<0x114, 0xF>(v);
    v += pg_dpp<0x118, 0xF>(v);
    v += pg_dpp<0x142, 0xA>(v);
    v += pg_dpp<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ uint32_t pg_last(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, 63); }
// a / b for a <= 2^24, which has f32's digits: a reciprocal of a unit in the last place and the product's rounding take the
// quotient at most 3 * 2^-24 of itself off, 1 at b = 3, and nothing where b is a power of two; so it is one off at most.
// A lane has at most 2^31 / 128 units, a call at most 2^23 items and 4 records for each work group that runs at a time.
// Every a with every b up to 70000 was compared with the division of whole numbers.
__device__ __forceinline__ uint32_t pg_div(uint32_t a, uint32_t b) {
    const uint32_t q = (uint32_t)((float)a * __builtin_amdgcn_rcpf((float)b));
    const uint32_t r = a - q * b;
    return (int32_t)r < 0 ? q - 1 : r >= b ? q + 1 : q;
}

// The same with long items cut into pieces, a work group a piece.  How, every
// wave works out by itself from the lengths: a lane of u units (a tile for each
// wave) is cut into p = ceil(u / L) pieces of equal length, L the smallest of
// some lengths from the chip's share (all units over the work groups that run
// at a time) to twice that at which the pieces run in one round of the chip;
// half the share where there are too many items for that (the work groups then
// take pieces in turn).  Pieces are numbered lane by lane, [piece][item], so that
// the blocks of query heads that read the same rows run side by side.  A piece
// of a lane that is cut leaves a record (m, l, o).
template <class T, int HDP, bool ONCE>
__global__ __launch_bounds__(PG_THREADS, pg_groups<HDP>) void paged_attn_cut_kernel(PagedAttnParams P) {
    using C = PgCfg<HDP>;
    constexpr uint32_t UNIT = PG_WAVES * C::KT, ROOM = pg_room(HDP);
    // L in sixteenths of the share.  Every quarter alone cut eight long lanes of 18 units a work group at 23 (126 us), these
    // at 19 (114).
    constexpr int CUTS = 6, SIXTEENTHS[CUTS] = {16, 17, 18, 20, 24, 32};
    __shared__ __attribute__((aligned(16))) char smem[C::BYTES];
    __shared__ float sm[PG_WAVES][PG_COLS], sl[PG_WAVES][PG_COLS];
    __shared__ uint32_t before[2][65], firsts[2][64]; // pieces and records before a thread's lanes, its first lane's rows
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t items = (uint32_t)P.n_kv * P.blocks; // of a lane
    // every thread's lanes, a run of them
    const int per = (P.n + 63) / 64, i0 = lane * per, i1 = i0 + per < P.n ? i0 + per : P.n;
    const auto units = [&](int i) {
        uint32_t first, end;
        pg_span(P, i, first, end);
        return (end - first + UNIT - 1) / UNIT;
    };
    uint32_t first0 = 0, end0 = 0; // of the first one, which is most often the only one
    if (i0 < i1)
        pg_span(P, i0, first0, end0);
    const uint32_t u0 = (end0 - first0 + UNIT - 1) / UNIT;
    const auto each = [&](auto f) {
        if (i0 < i1)
            f(u0, i0);
        for (int i = i0 + 1; i < i1; i++)
            f(units(i), i);
    };
    uint32_t total = 0;
    each([&](uint32_t u, int) { total += u; });
    total = pg_last(pg_scan(total));
    constexpr uint32_t MOST = 1 << 26; // longer than any lane
    const uint64_t exact = ((uint64_t)total * items + ROOM - 1) / ROOM;
    const uint32_t share = exact < 1 ? 1 : exact > MOST ? MOST : (uint32_t)exact;
    // ceil(u / L), at least 1; within a rounding of whole numbers it may be one off, which unsettles nothing: whoever counts
    // pieces counts them so
    const auto pieces = [](uint32_t u, uint32_t L) {
        return u ? (uint32_t)((float)u * __builtin_amdgcn_rcpf((float)L) * 0x1.fffffp-1f) + 1 : 1;
    };
    uint32_t cut[CUTS], count[CUTS];
#pragma unroll
    for (int x = 0; x < CUTS; x++) {
        cut[x] = (share * SIXTEENTHS[x] + 15) / 16;
        count[x] = 0;
    }
    each([&](uint32_t u, int) {
#pragma unroll
        for (int x = 0; x < CUTS; x++)
            count[x] += pieces(u, cut[x]);
    });
#pragma unroll
    for (int x = 0; x < CUTS; x++)
        count[x] = pg_scan(count[x]);
    uint32_t L = (share + 1) / 2;
#pragma unroll
    for (int x = CUTS - 1; x >= 0; x--)
        if (pg_last(count[x]) * items <= ROOM)
            L = cut[x];
    // pieces and records of the lanes up to this thread's last
    uint32_t np = 0, nr = 0;
    each([&](uint32_t u, int) {
        const uint32_t p = pieces(u, L);
        np += p;
        nr += p > 1 ? p : 0;
    });
    const uint32_t to_p = pg_scan(np), to_r = pg_scan(nr), all = pg_last(to_p) * items;
    if (blockIdx.x == 0 && tid == 63)
        *P.records = to_r * items;
    if (tid < 64) { // out of the registers
        before[0][lane] = to_p - np, before[1][lane] = to_r - nr;
        if (lane == 63)
            before[0][64] = to_p;
        firsts[0][lane] = first0, firsts[1][lane] = end0;
    }
    __syncthreads();
    for (uint32_t x = blockIdx.x; x < all; x += gridDim.x) {
        const uint32_t w = ONCE ? x : pg_turn(P, x, all);
        // its lane, by the thread that has it: the lane's pieces, those before it and the records before them
        uint32_t sum = before[0][lane], rec = before[1][lane], p = 1, first = firsts[0][lane], end = firsts[1][lane];
        const bool has = sum * items <= w && w < before[0][lane + 1] * items;
        int i = lane * per;
        if (has)
            for (;; pg_span(P, ++i, first, end)) {
                p = pieces((end - first + UNIT - 1) / UNIT, L);
                if (w < (sum + p) * items)
                    break;
                sum += p;
                rec += p > 1 ? p : 0;
            }
        const int src = __builtin_ctzll(__ballot(has));
        const auto from = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, src); };
        i = (int)from((uint32_t)i), p = from(p), sum = from(sum), rec = from(rec), first = from(first), end = from(end);
        const uint32_t turn = pg_div(w, items), piece = turn - sum, item = w - turn * items; // sum * items are before it
        const uint32_t u = (end - first + UNIT - 1) / UNIT, base = pg_div(u, p), more = u - base * p;
        const uint32_t a = base * piece + (piece < more ? piece : more), b = a + base + (piece < more);
        const int kvh = ONCE ? item : item / P.blocks, block = ONCE ? 0 : item - kvh * P.blocks;
        const int h0 = kvh * P.group + block * PG_COLS;
        const int heads = P.group - block * PG_COLS < PG_COLS ? P.group - block * PG_COLS : PG_COLS;
        pg_rows<T, HDP, ONCE, HDP <= 128>(P, i, kvh, h0, heads, end - first, first + a * UNIT, b == u ? end : first + b * UNIT, smem,
                                             sm, sl);
        rec = rec * items + item * p + piece;
        for (int x = tid; x < heads * (HDP / 4); x += PG_THREADS) {
            const int h = x / (HDP / 4), d = x % (HDP / 4) * 4;
            float M, S;
            const pg_f4 v = pg_join<HDP>(smem, sm, sl, h, d, M, S);
            if (d < P.hd) {
                if (p == 1)
                    *(pg_f4 *)(P.out + ((size_t)i * P.n_heads + h0 + h) * P.hd + d) = pg_result(v, S);
                else
                    *(pg_f4 *)(P.part + ((size_t)rec * P.cols + h) * P.hd + d) = v;
            }
            if (p > 1 && d == 0)
                P.ml[(size_t)rec * P.cols + h] = make_float2(M, S);
        }
        if (p > 1 && tid == 0)
            P.desc[rec] = {piece == 0 ? (int32_t)(i * (int)items + (int)item) : -1, (int32_t)p};
        __syncthreads(); // the join is read: its room is the next tiles'
    }
}

// The records of the item whose first one is blockIdx.x joined, WPH waves for
// a query head: M = max m, out = sum 2^(m - M) o / sum 2^(m - M) l.
template <int HDP, int WPH>
__global__ __launch_bounds__(PG_THREADS) void paged_attn_join_kernel(PagedAttnParams P) {
    constexpr int LPR = HDP / 4, PAR = 64 / LPR; // threads of a record, a wave's records side by side
    __shared__ pg_f4 so[PG_WAVES][64];
    __shared__ float sl[PG_WAVES][64];
    const uint32_t rec = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t records = *P.records;
    const PgDesc desc = P.desc[rec]; // undefined past the records
    if (rec >= records || desc.item < 0)
        return;
    const int items = P.n_kv * P.blocks, i = desc.item / items, item = desc.item - i * items, kvh = item / P.blocks;
    const int block = item - kvh * P.blocks, n = desc.pieces, h = blockIdx.y * (PG_WAVES / WPH) + wave / WPH;
    const int heads = P.group - block * PG_COLS < PG_COLS ? P.group - block * PG_COLS : PG_COLS;
    const int g = lane / LPR, d = lane % LPR * 4;
    float M = -__builtin_inff(), l = 0.0f;
    pg_f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    if (h < heads) {
        const size_t at = (size_t)rec * P.cols + h; // of a piece's next: P.cols further
        for (int r = lane; r < n; r += 64)
            M = fmaxf(M, P.ml[at + (size_t)r * P.cols].x);
        M = wave_max(M);
#pragma unroll 8
        for (int r = wave % WPH * PAR + g; r < n; r += WPH * PAR) {
            const size_t s = at + (size_t)r * P.cols;
            const float2 ml = P.ml[s];
            const pg_f4 v = d < P.hd ? *(const pg_f4 *)(P.part + s * P.hd + d) : pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
            const float f = ml.x == M ? 1.0f : __builtin_amdgcn_exp2f(ml.x - M);
            l += ml.y * f;
            o += v * f;
        }
#pragma unroll
        for (int x = LPR; x < 64; x *= 2) {
            l += __shfl_xor(l, x);
#pragma unroll
            for (int e = 0; e < 4; e++)
                o[e] += __shfl_xor(o[e], x);
        }
    }
    if constexpr (WPH > 1) {
        so[wave][lane] = o;
        sl[wave][lane] = l;
        __syncthreads();
        if (wave % WPH)
            return;
#pragma unroll
        for (int x = 1; x < WPH; x++)
            o += so[wave + x][lane], l += sl[wave + x][lane];
    }
    if (h < heads && g == 0 && d < P.hd)
        *(pg_f4 *)(P.out + ((size_t)i * P.n_heads + kvh * P.group + block * PG_COLS + h) * P.hd + d) = pg_result(o, l);
}

// How a call runs.
struct PgPlan {
    int room;
    size_t records; // at most; 0: no lane is cut, one launch
};
static PgPlan pg_plan(size_t max_rows, size_t items, size_t hd) {
    PgPlan p;
    p.room = pg_room(hd);
    // Pieces at twice the share: an item's rounding up and half of the chip's work groups.  Otherwise a piece of a cut lane
    // has more than half of L, and L is at least half of the share.
    p.records = items <= (size_t)p.room / 2 ? p.room : 4 * (size_t)p.room;
    if (max_rows <= (hd > 128 ? PG_WHOLE / 2 : PG_WHOLE))
        p.records = 0;
    return p;
}
static size_t pg_ws_bytes(const PgPlan &p, size_t hd, size_t cols) {
    return p.records ? 16 + p.records * (sizeof(PgDesc) + cols * (hd * 4 + sizeof(float2))) : 0;
}
static size_t pg_cols(size_t n_heads, size_t n_kv) { return n_heads / n_kv < PG_COLS ? n_heads / n_kv : PG_COLS; }
static size_t pg_items(size_t n, size_t n_heads, size_t n_kv) {
    return n * n_kv * ((n_heads / n_kv + PG_COLS - 1) / PG_COLS);
}

} // namespace lh

using namespace lh;

constexpr size_t PG_MAX_ROWS = (size_t)1 << 38; // positions of all lanes: their units are counted in 32 bits
// The sizes the kernels index in 32 bits.
static bool pg_served(size_t n, size_t n_heads, size_t n_kv, size_t hd) {
    return n && n <= 65535 && n_heads && n_kv && n_heads % n_kv == 0 && hd && hd % 8 == 0 && hd <= PG_MAX_HD &&
           n_heads <= 65535 && n * n_heads <= (size_t)1 << 23;
}

extern "C" {

size_t loomhip_paged_attn_ws(size_t max_rows, size_t n, size_t n_heads, size_t n_kv_heads, size_t head_dim) {
    if (!pg_served(n, n_heads, n_kv_heads, head_dim))
        return 0;
    return pg_ws_bytes(pg_plan(max_rows, pg_items(n, n_heads, n_kv_heads), head_dim), head_dim, pg_cols(n_heads, n_kv_heads));
}

int loomhip_paged_attn_dev(const loomhip_pages *c, const float *q, const int32_t *len, size_t n, size_t n_heads,
                           size_t n_kv_heads, size_t head_dim, float scale, size_t window, float *out, void *ws,
                           size_t ws_bytes, void *stream) {
    const char *fn = "paged_attn";
    if (n == 0)
        return LOOMHIP_OK;
    if (!q || !out || !len || n_heads == 0 || n_kv_heads == 0 || n_heads % n_kv_heads)
        return fail(LOOMHIP_ERR_ARG, "%s: null argument, or %zu heads over %zu key heads", fn, n_heads, n_kv_heads);
    if (!pg_served(n, n_heads, n_kv_heads, head_dim))
        return fail(LOOMHIP_DECLINED, "%s: %zu lanes of %zu heads of %zu not served", fn, n, n_heads, head_dim);
    if (int rc = pages_check(c, n_kv_heads, head_dim, fn))
        return rc;
    if (n * (c->page_size * c->table_width) > PG_MAX_ROWS)
        return fail(LOOMHIP_DECLINED, "%s: %zu lanes of %zu positions not served", fn, n, c->page_size * c->table_width);
    if (n > c->n_lanes)
        return fail(LOOMHIP_ERR_ARG, "%s: %zu lanes, a table of %zu", fn, n, c->n_lanes);
    if ((uintptr_t)len % 4)
        return fail(LOOMHIP_ERR_ARG, "%s: lengths not aligned to their elements", fn);
    if ((uintptr_t)q % 16 || (uintptr_t)out % 16)
        return fail(LOOMHIP_DECLINED, "%s: q or out not at a multiple of 16 bytes", fn);
    const size_t max_rows = c->page_size * c->table_width, items = pg_items(n, n_heads, n_kv_heads);
    const PgPlan plan = pg_plan(max_rows, items, head_dim);
    const size_t need = pg_ws_bytes(plan, head_dim, pg_cols(n_heads, n_kv_heads));
    if (need && (!ws || ws_bytes < need || (uintptr_t)ws % 16))
        return fail(LOOMHIP_ERR_ARG, "%s: the workspace takes %zu bytes at a multiple of 16, got %zu", fn, need, ws_bytes);
    if (int rc = require_device())
        return rc;
    PagedAttnParams P = {};
    P.c = *c;
    P.q = q;
    P.len = len;
    P.n = (int)n;
    P.n_heads = (int)n_heads;
    P.n_kv = (int)n_kv_heads;
    P.hd = (int)head_dim;
    P.group = (int)(n_heads / n_kv_heads);
    P.blocks = (P.group + PG_COLS - 1) / PG_COLS;
    const int bits = c->page_size > 1 ? 64 - __builtin_clzll(c->page_size - 1) : 0; // 2^bits >= page_size
    P.page_mul = bits ? (uint32_t)(((uint64_t)1 << (31 + bits)) / c->page_size + 1) : 0;
    P.page_shift = bits ? bits - 1 : 0;
    P.page_units = (uint32_t)(c->page_stride / 8);
    P.row_units = (uint32_t)(c->row_stride / 8);
    P.window = window > 0x7fffffff ? 0 : (uint32_t)window; // longer than any lane: none
    P.scale = scale;
    P.out = out;
    hipStream_t st = stream_of(stream);
    P.cols = (int)pg_cols(n_heads, n_kv_heads);
    if (need) {
        P.records = (uint32_t *)ws;
        P.part = (float *)((char *)ws + 16);
        P.ml = (float2 *)(P.part + plan.records * P.cols * head_dim);
        P.desc = (PgDesc *)(P.ml + plan.records * P.cols);
    }
    const auto run = [&](auto type, auto size, auto once) {
        using T = decltype(type);
        constexpr int HDP = decltype(size)::value;
        constexpr bool ONCE = decltype(once)::value;
        if (!need) {
            hipLaunchKernelGGL((paged_attn_kernel<T, HDP, ONCE>), dim3(items), dim3(PG_THREADS), 0, st, P);
            note_launch();
            return;
        }
        // as many work groups as run at a time, or as there can be pieces
        const size_t unit = PG_WAVES * PgCfg<HDP>::KT, most = items * ((max_rows + unit - 1) / unit);
        hipLaunchKernelGGL((paged_attn_cut_kernel<T, HDP, ONCE>), dim3(most < (size_t)plan.room ? most : plan.room),
                           dim3(PG_THREADS), 0, st, P);
        // with few items there may be hundreds of an item's records: two waves for a head.  Measured, 64 records of heads of
        // 128 and 256, and about four of 112 items: one wave 10.3 us, 29 and 5.0, two 7.1, 6.2 and 4.6, four 5.6, 10 and 5.9.
        const auto join = [&](auto waves) {
            constexpr int WPH = decltype(waves)::value, EACH = PG_WAVES / WPH;
            hipLaunchKernelGGL((paged_attn_join_kernel<HDP, WPH>), dim3(plan.records, (P.cols + EACH - 1) / EACH),
                               dim3(PG_THREADS), 0, st, P);
        };
        if (plan.records > (size_t)plan.room)
            join(std::integral_constant<int, 1>{});
        else
            join(std::integral_constant<int, 2>{});
        note_launch();
        note_launch();
    };
    const auto sized = [&](auto type, auto once) {
        if (head_dim <= 64)
            run(type, std::integral_constant<int, 64>{}, once);
        else if (head_dim <= 128)
            run(type, std::integral_constant<int, 128>{}, once);
        else
            run(type, std::integral_constant<int, 256>{}, once);
    };
    const auto typed = [&](auto once) { c->type == LH_F16 ? sized(PgF16{}, once) : sized(PgBf16{}, once); };
    if (P.blocks == 1)
        typed(std::true_type{});
    else
        typed(std::false_type{});
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? LOOMHIP_OK : hip_fail(e, "paged_attn launch");
}

} // extern "C"

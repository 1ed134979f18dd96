// prefix_attn.hip -- attention of a batch that shares a long prefix: every
// lane's query rows over one prefix cache, joined with the lane's own rows.
//
//   out = sum_t p_t v_t,  p = softmax of scale * (q . k_t) over the rows t seen
//
// The rows of all lanes that read one key head are the columns of a matrix
// product against the prefix, so each prefix tile is read once per 128 rows
// and not once per lane.  A work item is (key head, row block, a range of
// prefix rows) or (lane, key head, row block, a range of own rows); items
// leave (m, l, o) records, the running maximum and sum of a softmax over their
// range, and prefix_attn_merge_kernel joins a row's records.
//
// Products on the f16 matrix cores (v_mfma_f32_32x32x16_f16), two bits short
// of f32: the f32 query is scaled by a power of two of its own and split into
// two f16 parts (22 significant bits where f32 has 24; elements below 2^-16 of
// the row's largest are off by up to 2^-38 of it) against the exact fp16 keys,
// the weights p into two f16 parts against the exact fp16 values, f32 sums.
// One f16 part alone (11 bits) would leave 2e-4.  A third part each would be
// half as many products again; against 64 bits the error is 2e-7 to 5e-7 of the
// output's size (elementary operations in f32: 3e-7 to 17e-7).
//
// S^T = K Q^T: a lane holds one query (column lane % 32) and, of each 32 keys,
// the rows 8 (i / 4) + 4 (lane / 32) + i % 4, i < 16.  These registers are the
// B operand of O^T = V^T P^T as they stand, if its 16 contracted indices
// (lane / 32, j < 8) mean the keys 8 (j / 4) + 4 (lane / 32) + j % 4; the A
// operand's lane then needs 4 + 4 consecutive keys of one value column, which
// the LDS transpose read (ds_read_b64_tr_b16) gives from row-major values.
// The softmax of a query needs one exchange between the two half waves.
//
// Measured, heads of 128, 32 over 4 key heads, at the median of calls that
// follow each other: 190 query tokens of 64 lanes against 16384 shared and up
// to 640 own rows 130 us (121 at best: the clock falls under sustained matrix
// work), bound by the matrix cores (104 GFLOP in two-part products, 800
// TFLOP/s of the 1001 a large library product reaches), the merge 11; 32 lanes
// of one token against 4096 and 512 rows 20.6 us (27 MB), one round of short
// ranges, the merge 4.6.
#include "runtime.hpp"
#include <cmath>
#include <type_traits>
#include <utility>

namespace lh {

typedef _Float16 pa_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 pa_h2 __attribute__((ext_vector_type(2)));
typedef __fp16 pa_f2 __attribute__((ext_vector_type(2)));
typedef short pa_s4 __attribute__((ext_vector_type(4)));
typedef float pa_f16 __attribute__((ext_vector_type(16)));
typedef float pa_f4 __attribute__((ext_vector_type(4)));

constexpr int PA_THREADS = 256;
constexpr int PA_MAX_HD = 256;
// p = 2^(s - m + PA_SHIFT): the running maximum m moves only where eight
// weights sum to more than PA_MOST, so most tiles rescale nothing; p stays
// below 2^14 (f16 ends at 2^16) and its low part stays normal down to 2^-9 of
// the maximum, below that off by at most 2^-31 of it.
constexpr float PA_SHIFT = 6.0f, PA_MOST = 16384.0f;

struct PrefixAttnParams {
    loomhip_kv_rows pre, own;
    const float *q;
    const int32_t *own_len, *q_len;
    int n, n_q, n_heads, n_kv, hd;
    float scale;
    float *out;
    bool zero_rest; // rows past q_len
    // Items: prefix [kv][split][row block], then own [lane][kv][split][row block].  The prefix's split count depends on
    // how many rows the lanes have (q_len is on the device): pa_pre_cut's, at most pre_splits, left in *cut.
    int pre_splits, pre_items, xcd_slots;
    int own_blocks, own_splits, own_len_split;
    int slots;   // own_splits + pre_splits, in that order
    int *cut;
    float *part; // [row][slot][hd], row = (lane * n_q + token) * n_heads + head
    float2 *ml;  // [row][slot]
};

__device__ __forceinline__ int pa_clamp(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
__device__ __forceinline__ int pa_q_len(const PrefixAttnParams &P, int i) {
    return P.q_len ? pa_clamp(P.q_len[i], 0, P.n_q) : P.n_q;
}
__device__ __forceinline__ int pa_own_len(const PrefixAttnParams &P, int i) {
    return P.own.rows ? pa_clamp(P.own_len[i], 0, (int)P.own.rows) : 0;
}
// own rows that query j of L sees
__device__ __forceinline__ int pa_seen(int len, int L, int j) { return len - L + 1 + j < 0 ? 0 : len - L + 1 + j; }

// The largest of a value and the other half wave's.
__device__ __forceinline__ float pa_half_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pa_half_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// f(0), f(1), .. f(N - 1) with the number a constant.
template <class F, int... I>
__device__ __forceinline__ void pa_for(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void pa_for(F f) {
    pa_for(f, std::make_integer_sequence<int, N>{});
}

// A work group's four waves as RW row groups of 32 queries by 4 / RW key
// groups: a tile of TK cache rows, KPW of them for each wave, in blocks of 32.
// RW = 4 shares a tile among 128 queries; RW = 1 takes up to 32 queries (a
// lane's own rows, a small batch) with its waves side by side along the keys.
// PIPE: the tiles alternate between two LDS buffers, the loads of the one after
// next in registers, and the next block's scores are multiplied while this
// block's weights are formed; without it (short ranges, or a head whose query
// and sums leave no registers) a tile is loaded as it comes.
// LDS rows are padded so that fragment reads spread over the banks with every
// address a constant from one register: keys are read as 16 bytes of eight
// rows at a time, which 16 bytes more a row put 4 banks apart; values by 16
// lanes as 32 bytes of four rows, which 32 bytes more put 8 banks apart.
template <int HDP, int RW>
struct PaCfg {
    static constexpr int KW = 4 / RW, KPW = RW == 4 && HDP < 256 ? 64 : 32, TK = KW * KPW, NB = KPW / 32;
    static constexpr bool PIPE = RW > 1 && HDP < 256;
    static constexpr int CH = HDP / 8;               // 16-byte chunks of a row
    static constexpr int NCH = TK * CH / PA_THREADS; // chunks a thread stages, of keys and of values each
    static constexpr int KS = HDP * 2 + 16, VS = HDP * 2 + 32; // bytes from an LDS row to the next
    static constexpr int VO = TK * KS, TILE = VO + TK * VS;    // where a tile's values start, its bytes
    static constexpr int TILES = (PIPE ? 2 : 1) * TILE;
    static constexpr int ROWS = 4 * 32 * HDP * 4; // queries on their way in (RW * 32 rows), records on their way out
    static constexpr int BYTES = TILES > ROWS ? TILES : ROWS;
};

// Query rows [row0, row0 + RW * 32) of the item (map: their global row, -1 past the end; lim: the first key each
// does not see) against cache rows [k0, k1) at k / v (one head's rows, `stride` elements apart): records into slot
// `slot`.  border: rows from here on are not seen by every query.
template <int HDP, int RW>
__device__ __forceinline__ void pa_item(const PrefixAttnParams &P, const uint16_t *__restrict__ kp,
                                        const uint16_t *__restrict__ vp, size_t stride, int k0, int k1, int border,
                                        int slot, const int *map, const int *lim, char *smem, int *flag) {
    using C = PaCfg<HDP, RW>;
    constexpr int STEPS = HDP / 16, DB = HDP / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int half = lane >> 5, col = lane & 31;
    const int rw = wave % RW, kw = wave / RW;
    const int row = map[rw * 32 + col], limit = lim[rw * 32 + col] < k1 ? lim[rw * 32 + col] : k1;
    const int hd = P.hd;

    // staging: thread t's chunks are t, t + 256, ..
    uint4 rk[C::NCH], rv[C::NCH];
    constexpr int RSTEP = PA_THREADS / C::CH;        // rows from a thread's chunk to its next
    const int sch = tid % C::CH, srow = tid / C::CH; // its column of chunks, its first row
    // Rows past the last and chunks past the head's end are the last one again: their scores are masked, their weights
    // zero, their columns not written.
    const int ssrc = (sch * 8 < hd ? sch : hd / 8 - 1) * 16;
    uint32_t soff[C::NCH]; // byte offsets from the tile's first row
    const auto place = [&](int last) { // rows up to `last` of the tile
#pragma unroll
        for (int c = 0; c < C::NCH; c++) {
            const int r = srow + c * RSTEP;
            soff[c] = (uint32_t)(r < last ? r : last) * ((uint32_t)stride * 2) + ssrc;
        }
    };
    const auto load = [&](const uint16_t *__restrict__ p, int kt, int c) {
        return *(const uint4 *)((const char *)(p + (size_t)kt * stride) + soff[c]);
    };
    const auto load_tile = [&](const uint16_t *__restrict__ p, uint4 *to, int kt) {
#pragma unroll
        for (int c = 0; c < C::NCH; c++)
            to[c] = load(p, kt, c);
    };
    const int k_st = srow * C::KS + sch * 16, v_st = C::VO + srow * C::VS + sch * 16;
    const auto store_keys = [&](char *to, int c) { *(uint4 *)(to + k_st + c * RSTEP * C::KS) = rk[c]; };
    const auto store_values = [&](char *to, int c) { *(uint4 *)(to + v_st + c * RSTEP * C::VS) = rv[c]; };
    const auto store_tile = [&](char *to) {
#pragma unroll
        for (int c = 0; c < C::NCH; c++) {
            store_keys(to, c);
            store_values(to, c);
        }
    };
    // Values that some query does not see are left out of the product where they are not finite: they would reach it
    // as 0 * v.  strange: there was one.
    bool strange = false;
    const auto clean = [&](int kt) {
        if (kt + C::TK > border) {
#pragma unroll
            for (int c = 0; c < C::NCH; c++)
                if (kt + srow + c * RSTEP >= border) {
                    uint32_t *w = (uint32_t *)&rv[c];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const bool lo = (w[e] & 0x7c00u) == 0x7c00u, hi = (w[e] & 0x7c000000u) == 0x7c000000u;
                        strange |= lo | hi;
                        w[e] &= (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0x0000ffffu : 0xffffffffu);
                    }
                }
        }
    };
    if (tid == 0)
        *flag = 0;
    place(k1 - 1 - k0);
    if (HDP < 256) { // the first tile, in flight while the queries are split
        load_tile(kp, rk, k0);
        load_tile(vp, rv, k0);
    }

    // The queries through LDS (a lane's loads of its own row would touch 32 rows each), then each its largest element
    // brought to 2^13 .. 2^14 by a power of two and split into two f16 parts.
    constexpr int QC = HDP / 4, QN = RW * 32 * QC / PA_THREADS; // 16-byte columns of a row, shifted by the row against
                                                                // bank conflicts; columns a thread takes
    constexpr int QB = QN < 8 ? QN : 8;                         // loads in flight
    const int qc = tid % QC, qr = tid / QC;
    const size_t qat = qc * 4 < hd ? qc * 4 : 0;
#pragma unroll
    for (int n0 = 0; n0 < QN; n0 += QB) {
        pa_f4 v[QB];
        int R[QB];
#pragma unroll
        for (int x = 0; x < QB; x++) {
            R[x] = map[qr + (n0 + x) * (PA_THREADS / QC)];
            v[x] = *(const pa_f4 *)(P.q + (size_t)(R[x] < 0 ? 0 : R[x]) * hd + qat);
        }
#pragma unroll
        for (int x = 0; x < QB; x++) {
            const int r = qr + (n0 + x) * (PA_THREADS / QC);
            *(pa_f4 *)(smem + (r * QC + (qc + r) % QC) * 16) =
                R[x] >= 0 && qc * 4 < hd ? v[x] : pa_f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    __syncthreads();
    pa_h8 qh[STEPS], ql[STEPS];
    float cs; // scores in log2 units per unit of the split query's
    {
        const int r = rw * 32 + col;
        float v[STEPS][8], amax = 0.0f;
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const pa_f4 a = *(const pa_f4 *)(smem + (r * QC + (s * 4 + half * 2 + x + r) % QC) * 16);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    v[s][x * 4 + e] = a[e];
                    amax = fmaxf(amax, fabsf(a[e]));
                }
            }
        amax = pa_half_max(amax);
        // the power of two from amax's exponent (126 for the smallest: the query stays as small as it is)
        const int e = (int)(__float_as_uint(amax) >> 23);
        const int k = e > 0 && e < 255 ? pa_clamp(13 + 127 - e, -120, 120) : 0;
        const float f = __uint_as_float((uint32_t)(127 + k) << 23) * (P.scale < 0.0f ? -1.0f : 1.0f);
        cs = fabsf(P.scale) * 0x1.715476p+0f * __uint_as_float((uint32_t)(127 - k) << 23);
        cs = cs < 0x1p-126f ? 0x1p-126f : cs; // not 0: it multiplies a masked key's -inf (scores stay far below 1)
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float x = v[s][e] * f;
                const _Float16 h = (_Float16)x;
                qh[s][e] = h;
                ql[s][e] = (_Float16)(x - (float)h);
            }
    }

    const int kb = kw * C::KPW; // the wave's keys of a tile
    const int k_at = (kb + col) * C::KS + half * 16;
    const int v_at = C::VO + (kb + 4 * half + ((lane & 15) >> 2)) * C::VS + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
    pa_f16 o[DB];
#pragma unroll
    for (int b = 0; b < DB; b++)
#pragma unroll
        for (int i = 0; i < 16; i++)
            o[b][i] = 0.0f;
    float m = -__builtin_inff(), l = 0.0f;

    // Fragments: keys of block b and 16 columns of the head, values of 16 keys and 32 columns.
    const auto key_frag = [&](const char *tile, int b, int st) {
        return *(const pa_h8 *)(tile + k_at + b * 32 * C::KS + st * 32);
    };
    const auto value_frag = [&](char *tile, int b, int st, int db) {
        const auto at = (__attribute__((address_space(3))) char *)(tile + v_at) + (b * 32 + st * 16) * C::VS + db * 64;
        const pa_s4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s4 *)at);
        const pa_s4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s4 *)(at + 8 * C::VS));
        return __builtin_bit_cast(pa_h8, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    // -inf for the keys of block b of the tile at kt that the lane's query does not see
    const auto mask = [&](pa_f16 &s, int kt, int b) {
        if (kt + C::TK > border || kt + C::TK > k1) {
            const int seen = limit - kt - kb - b * 32 - 4 * half; // of the lane's keys, counted from its first
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float v = 8 * (i / 4) + i % 4 < seen ? s[i] : -__builtin_inff();
                asm volatile("" : "+v"(v)); // kept inside the branch: the selects would run in every block
                s[i] = v;
            }
        }
    };
    // Weights are taken against m, the running maximum of the scores of some block before: p = 2^(s - m + PA_SHIFT).
    // No block's own maximum is formed: the sum of eight weights, which is wanted anyway, tells whether one of them is
    // past what m allows (or no number); then m moves to this block's and the eight are formed again.
    float sub = 0.0f; // PA_SHIFT - m
    const auto largest = [](const pa_f16 &s) {
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; i++)
            mx = fmaxf(mx, s[i]);
        return mx;
    };
    const auto grow = [&](const pa_f16 &s) {
        const float m2 = fmaxf(m, pa_half_max(largest(s)) * cs);
        const float f = m == m2 ? 1.0f : __builtin_amdgcn_exp2f(m - m2); // -inf before the first seen key: 0
        m = m2;
        sub = PA_SHIFT - (m == -__builtin_inff() ? 0.0f : m);
        l *= f;
#pragma unroll
        for (int b = 0; b < DB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++)
                o[b][i] *= f;
        // a query that has seen nothing yet has no m: its first finite score has to come back here
        if (m == -__builtin_inff())
            sub = __builtin_inff();
    };
    // A block's weights, in two f16 parts: piece by piece, of each pair of values first the weights and their sum, then
    // the parts.  Pieces 2 j and 2 j + 1 do the values 2 j; eight values make a half.
    pa_h8 ph[2], pl[2];
    float w0, w1, sum;
    const auto piece = [&](const pa_f16 &s, int j) {
        const int i = j & ~1;
        if (j % 2 == 0) {
            w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], cs, sub));
            w1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i + 1], cs, sub));
            sum = i % 8 == 0 ? w0 + w1 : sum + (w0 + w1);
        } else {
            const pa_h2 h = {(_Float16)w0, (_Float16)w1};
            const float r0 = w0 - (float)h[0], r1 = w1 - (float)h[1];
            const pa_h2 g = {(_Float16)r0, (_Float16)r1};
            ph[i / 8][i % 8] = h[0], ph[i / 8][i % 8 + 1] = h[1];
            pl[i / 8][i % 8] = g[0], pl[i / 8][i % 8 + 1] = g[1];
        }
    };
    // After the eight of a half: taken again where m was too small for them.
    const auto settle = [&](const pa_f16 &s, int x) {
        if (__any(!(sum <= PA_MOST))) {
            grow(s);
            if (sub == __builtin_inff())
                sub = 0.0f; // nothing seen: every weight is 2^-inf
#pragma unroll
            for (int j = 0; j < 8; j++)
                piece(s, x * 8 + j);
            if (m == -__builtin_inff())
                sub = __builtin_inff();
        }
        l += sum;
    };
    // Scores of a block (S^T = K Q^T) and in their shadow the first half of the weights of the block before, and
    // whatever `other` does at each step.  Products issue in order and each waits for the one before it, 32 cycles: the
    // other work goes between them, about five vector instructions each (4.6 cycles).  Fragments are read AHEAD before
    // their products: the first of them before the call, and here the first of the values of the products that follow.
    constexpr int AHEAD = HDP == 128 ? 3 : 4, FRAGS = 2 * DB;
    pa_h8 kf[STEPS], vf[FRAGS];
    const auto keys_ahead = [&](const char *tile, int b) {
#pragma unroll
        for (int st = 0; st < AHEAD; st++)
            kf[st] = key_frag(tile, b, st);
    };
    const auto values_ahead = [&](char *tile, int b) {
#pragma unroll
        for (int x = 0; x < AHEAD; x++)
            vf[x] = value_frag(tile, b, x / DB, x % DB);
    };
    const auto scores = [&](const char *tile, int b, const pa_f16 &before, auto weigh, char *then_tile, int then_b,
                            auto other) __attribute__((always_inline)) {
        constexpr bool W = decltype(weigh)::value;
        pa_f16 s;
#pragma unroll
        for (int i = 0; i < 16; i++)
            s[i] = 0.0f;
        __builtin_amdgcn_sched_barrier(0);
        pa_for<STEPS>([&](auto step) {
            constexpr int st = decltype(step)::value, PIECES = 8; // 8 of 16 values
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[st], qh[st], s, 0, 0, 0);
            if constexpr (st + AHEAD < STEPS)
                kf[st + AHEAD] = key_frag(tile, b, st + AHEAD);
            else if constexpr (W) {
                constexpr int x = st + AHEAD - STEPS;
                vf[x] = value_frag(then_tile, then_b, x / DB, x % DB);
            }
            if constexpr (W)
#pragma unroll
                for (int j = st * PIECES / STEPS; j < (st + 1) * PIECES / STEPS; j++)
                    piece(before, j);
            __builtin_amdgcn_sched_barrier(0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[st], ql[st], s, 0, 0, 0);
            other(step);
            __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (W) {
            asm volatile("" : "+v"(ph[0]), "+v"(pl[0])); // formed here, not past the next branch
            settle(before, 0);
        }
        return s;
    };
    // O^T += V^T P^T of a block, in whose shadow the second half of its weights, `other`, and the first reads of the keys
    // that come after.
    const auto products = [&](char *tile, int b, const pa_f16 &now, const char *then_tile, int then_b, auto read_keys,
                              auto other) __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        pa_for<FRAGS>([&](auto frag) {
            constexpr int x = decltype(frag)::value, st = x / DB, db = x % DB;
            if constexpr (x == DB) {
                asm volatile("" : "+v"(ph[1]), "+v"(pl[1]));
                if constexpr (C::PIPE)
                    settle(now, 1);
                else
                    l += sum;
                __builtin_amdgcn_sched_barrier(0);
            }
            const auto shadow = [&](int y) { // y of 0, 1
                if (st == 0)
#pragma unroll
                    for (int j = 8 + (2 * db + y) * 4 / DB; j < 8 + (2 * db + y + 1) * 4 / DB; j++)
                        piece(now, j);
            };
            o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[x], ph[st], o[db], 0, 0, 0);
            if constexpr (x + AHEAD < FRAGS)
                vf[x + AHEAD] = value_frag(tile, b, (x + AHEAD) / DB, (x + AHEAD) % DB);
            else if constexpr (decltype(read_keys)::value)
                kf[x + AHEAD - FRAGS] = key_frag(then_tile, then_b, x + AHEAD - FRAGS);
            shadow(0);
            __builtin_amdgcn_sched_barrier(0);
            o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[x], pl[st], o[db], 0, 0, 0);
            shadow(1);
            other(frag);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    const auto nothing = [](auto) {};
    constexpr std::true_type yes;
    constexpr std::false_type no;
    __syncthreads(); // the queries are out of LDS
    if constexpr (C::PIPE) {
        char *cur = smem, *nxt = smem + C::TILE;
        clean(k0);
        store_tile(cur);
        __syncthreads();
        const int kl = k0 + (k1 - k0 - 1) / C::TK * C::TK; // the last tile
        int kn = k0 + C::TK < kl ? k0 + C::TK : kl;         // the next one
        place(k1 - 1 - kn);
        load_tile(kp, rk, kn);
        load_tile(vp, rv, kn);
        keys_ahead(cur, 0);
        pa_f16 s = scores(cur, 0, pa_f16{}, no, nullptr, 0, nothing);
        mask(s, k0, 0);
        grow(s);
        if (C::NB == 2)
            keys_ahead(cur, 1);
        // Past the last tile the next one's stores, loads and scores are the last one's again, used by nobody.
        for (int kt = k0; kt < k1; kt += C::TK) {
            clean(kn);
            const int k2 = kn + C::TK < kl ? kn + C::TK : kl;
            const auto store_next = [&](auto at) { // the next tile's buffer was last read before the barrier below
                constexpr int i = decltype(at)::value;
                if constexpr (i < C::NCH)
                    store_keys(nxt, i);
                else
                    store_values(nxt, i - C::NCH);
            };
            const auto load_next = [&](auto at) {
                constexpr int i = decltype(at)::value;
                if constexpr (i < C::NCH)
                    rk[i] = load(kp, k2, i);
                else
                    rv[i - C::NCH] = load(vp, k2, i - C::NCH);
            };
            static_assert(2 * C::NCH == STEPS && FRAGS == STEPS, "a store each step, a load each fragment");
            const bool more = kt + C::TK < k1;
            if (k2 + C::TK > k1)
                place(k1 - 1 - k2);
            if constexpr (C::NB == 2) {
                pa_f16 s1 = scores(cur, 1, s, yes, cur, 0, store_next);
                mask(s1, kt, 1);
                __syncthreads(); // the next tile is there
                products(cur, 0, s, nxt, 0, yes, load_next);
                s = scores(nxt, 0, s1, yes, cur, 1, nothing);
                if (more)
                    mask(s, kn, 0);
                products(cur, 1, s1, nxt, 1, yes, nothing);
            } else {
                store_tile(nxt);
                __syncthreads();
                keys_ahead(nxt, 0);
                pa_f16 s1 = scores(nxt, 0, s, yes, cur, 0, nothing);
                if (more)
                    mask(s1, kn, 0);
                products(cur, 0, s, nullptr, 0, no, load_next);
                s = s1;
            }
            __syncthreads(); // this tile is read
            kn = k2;
            char *const t = cur;
            cur = nxt;
            nxt = t;
        }
    } else {
        for (int kt = k0; kt < k1; kt += C::TK) {
            __syncthreads();
            if (HDP == 256 || kt > k0) {
                place(k1 - 1 - kt);
                load_tile(kp, rk, kt);
                if (HDP == 256)
#pragma unroll
                    for (int c = 0; c < C::NCH; c++)
                        store_keys(smem, c);
                load_tile(vp, rv, kt);
            }
            clean(kt);
            if (HDP == 256)
#pragma unroll
                for (int c = 0; c < C::NCH; c++)
                    store_values(smem, c);
            else
                store_tile(smem);
            __syncthreads();
            keys_ahead(smem, 0);
            pa_f16 s = scores(smem, 0, pa_f16{}, no, nullptr, 0, nothing);
            values_ahead(smem, 0);
            mask(s, kt, 0);
            if (__any(largest(s) * cs > m + (14.0f - PA_SHIFT))) // a block a tile: as cheap as the check of the sum
                grow(s);
            if (m == -__builtin_inff())
                sub = 0.0f; // nothing seen: every weight is 2^-inf
#pragma unroll
            for (int j = 0; j < 8; j++)
                piece(s, j);
            l += sum;
            products(smem, 0, s, nullptr, 0, no, nothing);
        }
    }
    l = pa_half_sum(l);
    if (strange)
        *flag = 1;

    // Records: o as it stands relative to m (both carry PA_SHIFT), through LDS, where the key groups of a row group are
    // joined and from where whole rows are written (a lane holds 16 bytes here and there of its row).
    {
        __shared__ float sm[4][32], sl[4][32];
        __syncthreads();
        if (half == 0)
            sm[wave][col] = m, sl[wave][col] = l;
        __syncthreads();
        float M = sm[rw][col];
#pragma unroll
        for (int w = 1; w < C::KW; w++)
            M = fmaxf(M, sm[rw + w * RW][col]);
        const float f = m == M ? 1.0f : __builtin_amdgcn_exp2f(m - M);
        float *so = (float *)smem + (size_t)wave * 32 * HDP;
#pragma unroll
        for (int db = 0; db < DB; db++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int d = db * 32 + 2 * i + 4 * half;
                // 16-byte columns shifted by the query, so the lanes' rows spread over the banks
                *(pa_f4 *)(so + col * HDP + ((d / 4 + col) % (HDP / 4)) * 4) =
                    pa_f4{o[db][i] * f, o[db][i + 1] * f, o[db][i + 2] * f, o[db][i + 3] * f};
            }
        __syncthreads();
#pragma unroll
        for (int n0 = 0; n0 < QN; n0++) {
            const int rr = qr + n0 * (PA_THREADS / QC), R = map[rr], g = rr / 32, c = rr % 32;
            pa_f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < C::KW; w++)
                v += *(const pa_f4 *)((const float *)smem + (size_t)(g + w * RW) * 32 * HDP + c * HDP + (qc + c) % QC * 4);
            if (R >= 0 && qc * 4 < hd)
                *(pa_f4 *)(P.part + ((size_t)R * P.slots + slot) * hd + qc * 4) = v;
        }
        if (tid < RW * 32 && map[tid] >= 0) {
            const int g = tid / 32, c = tid % 32;
            float mm = sm[g][c], ll = 0.0f;
#pragma unroll
            for (int w = 1; w < C::KW; w++)
                mm = fmaxf(mm, sm[g + w * RW][c]);
#pragma unroll
            for (int w = 0; w < C::KW; w++)
                ll += sl[g + w * RW][c] * (sm[g + w * RW][c] == mm ? 1.0f : __builtin_amdgcn_exp2f(sm[g + w * RW][c] - mm));
            P.ml[(size_t)map[tid] * P.slots + slot] = make_float2(mm, ll);
        }
    }
    // The values taken out of the tiles, for the queries that see them: a weight of any size times them is no number.
    __syncthreads();
    if (*flag)
        for (int at = tid; at < RW * 32 * hd; at += PA_THREADS) {
            const int rr = at / hd, d = at % hd, R = map[rr];
            const int end = lim[rr] < k1 ? lim[rr] : k1;
            for (int t = border > k0 ? border : k0; R >= 0 && t < end; t++) {
                const uint32_t v = vp[(size_t)t * stride + d];
                if ((v & 0x7c00u) == 0x7c00u)
                    P.part[((size_t)R * P.slots + slot) * hd + d] += half_bits_to_float(v);
            }
        }
}

// All lanes' live query rows in order: lane, token < q_len, head of the group.  Every thread takes lanes tid, tid + 256,
// ..; the running sum of their token counts tells where a lane's rows are.
struct PaTokens {
    int L, end, all; // of the chunk of 256 lanes scanned last: the thread's lane's tokens, their end, all of them
};
__device__ __forceinline__ PaTokens pa_scan(const PrefixAttnParams &P, int i0, int *scan) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int i = i0 + tid, L = i < P.n ? pa_q_len(P, i) : 0;
    int c = L;
    for (int o = 1; o < 64; o *= 2) {
        const int up = __shfl_up(c, o);
        c += lane >= o ? up : 0;
    }
    if (lane == 63)
        scan[wave] = c;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < PA_THREADS / 64; w++) {
        c += w < wave ? scan[w] : 0;
        all += scan[w];
    }
    __syncthreads();
    return {L, c, all};
}
__device__ __forceinline__ int pa_count(const PrefixAttnParams &P, int *scan, PaTokens &last) {
    if (!P.q_len)
        return P.n * P.n_q;
    int all = 0;
    for (int i0 = 0; i0 < P.n; i0 += PA_THREADS) {
        last = pa_scan(P, i0, scan);
        all += last.all;
    }
    return all;
}
// The block's rows [r0, r0 + R), -1 past the last, by way of its tokens (tok: lane * n_q + token).
template <int R>
__device__ __forceinline__ void pa_map(const PrefixAttnParams &P, int kvh, int r0, int tokens, PaTokens t, int *map,
                                       int *tok, int *scan) {
    const int G = P.n_heads / P.n_kv, tid = threadIdx.x;
    const int t0 = r0 / G, t1 = t0 + R < tokens ? t0 + R : tokens; // at least the block's tokens
    if (P.q_len) {
        int before = 0;
        for (int i0 = 0; i0 < P.n && before < t1; i0 += PA_THREADS) {
            if (P.n > PA_THREADS)
                t = pa_scan(P, i0, scan);
            const int first = before + t.end - t.L; // the lane's first token
            for (int j = first < t0 ? t0 - first : 0; j < t.L && first + j < t1; j++)
                tok[first + j - t0] = (i0 + tid) * P.n_q + j;
            before += t.all;
        }
        __syncthreads();
    }
    for (int r = tid; r < R; r += PA_THREADS) {
        const int at = (r0 + r) / G, h = r0 + r - at * G;
        map[r] = at < tokens ? (P.q_len ? tok[at - t0] : at) * P.n_heads + kvh * G + h : -1;
    }
    __syncthreads();
}

// The prefix's splits for `blocks` row blocks of every key head: a lane per candidate, the cheapest of
//   rounds of the chip's work groups * (an item's start and end + its tiles) + records to be joined,
// in the time of a 64-row tile, two work groups to a CU (3 us: measured start and end 8 us, 1024 records 0.3 us; at heads
// of 128, and taken for the other sizes too).
constexpr float PA_ITEM = 3.0f, PA_RECORD = 0.09f / 1024.0f;
__host__ __device__ inline int pa_split_len(int rows, int splits) {
    return ((rows + splits - 1) / splits + 127) / 128 * 128;
}
// rows of the cache, splits s, items a split (x), work groups at a time, query rows of a split's records; infinite for a
// count that leaves a split empty
__host__ __device__ inline float pa_cost(int rows, int s, int x, int room, float records) {
    const int len = pa_split_len(rows, s);
    if ((int64_t)(s - 1) * len >= rows)
        return __builtin_inff();
    return (float)(((uint32_t)x * s + room - 1) / room) * (PA_ITEM + (float)(len / 64)) + PA_RECORD * (float)s * records;
}
__device__ __forceinline__ int pa_pre_cut(const PrefixAttnParams &P, int blocks, int block_rows) {
    const int s = (threadIdx.x & 63) + 1, x = P.n_kv * blocks;
    float cost = pa_cost((int)P.pre.rows, s, x, P.xcd_slots * 8, (float)(x * block_rows));
    if (s > 1 && (s > P.pre_splits || x * s > P.pre_items))
        cost = __builtin_inff();
    int best = s;
    for (int o = 1; o < 64; o *= 2) {
        const float c2 = __shfl_xor(cost, o);
        const int b2 = __shfl_xor(best, o);
        const bool take = c2 < cost || (c2 == cost && b2 < best);
        cost = take ? c2 : cost;
        best = take ? b2 : best;
    }
    return __builtin_amdgcn_readfirstlane(best);
}

template <int HDP, int RWP, int RWO>
__global__ __launch_bounds__(PA_THREADS, HDP == 256 ? 1 : 2) void prefix_attn_kernel(PrefixAttnParams P) {
    constexpr int BP = PaCfg<HDP, RWP>::BYTES, BO = PaCfg<HDP, RWO>::BYTES;
    __shared__ __attribute__((aligned(16))) char smem[BP > BO ? BP : BO];
    constexpr int RM = (RWP > RWO ? RWP : RWO) * 32;
    __shared__ int map[RM], lim[RM], scan[PA_THREADS / 64], flag;
    const int G = P.n_heads / P.n_kv, tid = threadIdx.x;
    if ((int)blockIdx.x < P.pre_items) {
        PaTokens last = {0, 0, 0};
        const int tokens = pa_count(P, scan, last);
        const int blocks = (tokens * G + RWP * 32 - 1) / (RWP * 32);
        const int splits = P.q_len ? pa_pre_cut(P, blocks, RWP * 32) : P.pre_splits;
        // Work groups go to the eight XCDs in turn: each XCD takes a run of items, so the row blocks of one (key head,
        // split) find its rows in one L2.
        const int all = P.n_kv * splits * blocks, per = (all + 7) / 8, at = blockIdx.x >> 3;
        const int item = (blockIdx.x & 7) * per + at;
        if (blockIdx.x == 0 && tid == 0)
            *P.cut = splits;
        if (at >= per || item >= all)
            return;
        const int ks = item / blocks, rb = item - ks * blocks, kvh = ks / splits, sp = ks - kvh * splits;
        pa_map<RWP * 32>(P, kvh, rb * RWP * 32, tokens, last, map, lim, scan);
        const int rows = (int)P.pre.rows, len = pa_split_len(rows, splits);
        const int k0 = sp * len, k1 = k0 + len < rows ? k0 + len : rows;
        for (int r = tid; r < RWP * 32; r += PA_THREADS)
            lim[r] = k1;
        __syncthreads();
        pa_item<HDP, RWP>(P, P.pre.k + (size_t)kvh * P.pre.head_stride, P.pre.v + (size_t)kvh * P.pre.head_stride,
                          P.pre.row_stride, k0, k1, k1, P.own_splits + sp, map, lim, smem, &flag);
    } else {
        int b = blockIdx.x - P.pre_items;
        const int rb = b % P.own_blocks;
        b /= P.own_blocks;
        const int sp = b % P.own_splits;
        b /= P.own_splits;
        const int kvh = b % P.n_kv, i = b / P.n_kv;
        const int L = pa_q_len(P, i), len = pa_own_len(P, i), r0 = rb * RWO * 32;
        const int k0 = sp * P.own_len_split, k1 = k0 + P.own_len_split < len ? k0 + P.own_len_split : len;
        if (k0 >= len || r0 >= L * G)
            return;
        for (int r = tid; r < RWO * 32; r += PA_THREADS) {
            const bool in = r0 + r < L * G;
            const int j = (r0 + r) / G;
            map[r] = in ? (i * P.n_q + j) * P.n_heads + kvh * G + (r0 + r) % G : -1;
            lim[r] = in ? pa_seen(len, L, j) : k1; // no query: nothing to take out, its scores are zero
        }
        __syncthreads();
        const size_t base = (size_t)i * P.own.lane_stride + (size_t)kvh * P.own.head_stride;
        pa_item<HDP, RWO>(P, P.own.k + base, P.own.v + base, P.own.row_stride, k0, k1, pa_seen(len, L, 0), sp, map, lim,
                          smem, &flag);
    }
}

// A row's records joined: M = max m, out = sum 2^(m - M) o / sum 2^(m - M) l, a wave per row.
constexpr int PA_MERGE_ROWS = PA_THREADS / 64;
template <int LPR>
__global__ __launch_bounds__(PA_THREADS) void prefix_attn_merge_kernel(PrefixAttnParams P, int rows) {
    const int row = blockIdx.x * PA_MERGE_ROWS + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= rows)
        return;
    const int token = row / P.n_heads, i = token / P.n_q, j = token % P.n_q;
    if (j >= pa_q_len(P, i)) {
        if (P.zero_rest && lane * 4 < P.hd)
            *(pa_f4 *)(P.out + (size_t)row * P.hd + lane * 4) = pa_f4{0.0f, 0.0f, 0.0f, 0.0f};
        return;
    }
    const int len = pa_own_len(P, i);
    // the slots that were written: the own splits that start below the lane's length, and the prefix's
    const int own = P.own_splits ? (len + P.own_len_split - 1) / P.own_len_split : 0;
    const int slots = own + (P.pre_splits ? *P.cut : 0), skip = P.own_splits - own;
    const float2 *ml = P.ml + (size_t)row * P.slots;
    const float *part = P.part + (size_t)row * P.slots * P.hd;
    float M = -__builtin_inff();
    for (int s = lane; s < slots; s += 64)
        M = fmaxf(M, ml[s < own ? s : s + skip].x);
    M = wave_max(M);
    // the wave's lanes as groups of LPR along the row, each with every GRP-th record
    constexpr int GRP = 64 / LPR;
    const int g = lane / LPR, d = lane % LPR * 4;
    float l = 0.0f;
    pa_f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int x = g; x < slots; x += GRP) {
        const int s = x < own ? x : x + skip;
        const float2 r = ml[s];
        const pa_f4 v = d < P.hd ? *(const pa_f4 *)(part + (size_t)s * P.hd + d) : pa_f4{0.0f, 0.0f, 0.0f, 0.0f};
        const float w = r.x == M ? 1.0f : __builtin_amdgcn_exp2f(r.x - M);
        l += r.y * w;
        o += v * w;
    }
#pragma unroll
    for (int x = LPR; x < 64; x *= 2) {
        l += __shfl_xor(l, x);
#pragma unroll
        for (int e = 0; e < 4; e++)
            o[e] += __shfl_xor(o[e], x);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l; // nothing seen: zero
    // An infinity here comes from a cached one, which the weights' low parts (0, or below it) turn into NaN in some rows
    // and not in others: NaN in all.  Zero times anything finite adds nothing.
    o *= inv;
    if (g == 0 && d < P.hd)
        *(pa_f4 *)(P.out + (size_t)row * P.hd + d) = o + o * 0.0f;
}

// How a call is cut into items.
struct PaPlan {
    int hdp, rwp, rwo;
    int pre_splits, pre_items, xcd_slots, own_blocks, own_splits, own_len, slots;
    size_t rows;
};
static PaPlan pa_plan(size_t prefix_rows, size_t own_rows, size_t n, size_t n_q, size_t n_heads, size_t n_kv,
                      size_t hd, bool ragged) {
    PaPlan p = {};
    const size_t G = n_heads / n_kv, all = n * n_q * G, mine = n_q * G;
    p.hdp = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
    p.rows = n * n_q * n_heads;
    // Rows of a prefix item, 32, 64 or 128: few rows are bound by an item's start and end, many by the matrix cores, whose
    // fragments serve twice as many products a wave at 128.  Measured, heads of 128, in blocks of 64 and of 128: 128 rows
    // a key head against 512 shared rows 13.8 us and 16.4, against 65536 54 and 57; 256 against 4096 20.5 and 24.5; 2048
    // against 16384 166 and 149.  In blocks of 32, 64 and 128, heads of 64: 32 rows against 4096 11.0, 11.6 and 12.9; 128
    // 14.6, 13.8 and 14.5; 512 against 65536 210, 188 and 166; 2048 against 512 51, 48 and 54 (the line is too low
    // there).  Heads of 256: 32 rows against 4096 21.6, 22.8 and 26.8; 256 29.7, 30.6 and 34.3; 2048 117, 87 and 87; 512
    // against 65536 308, 208 and 185.
    p.rwp = all <= 32 ? 1 : all <= 256 ? 2 : 4;
    p.rwo = mine <= 32 ? 1 : 2;
    // the chip's work groups (two to a CU, one at head sizes over 128), shared by the tiles of the two kinds
    const int slots = p.hdp == 256 ? 256 : 512;
    p.own_blocks = (int)((mine + 32 * p.rwo - 1) / (32 * p.rwo));
    const int pre_x = (int)(n_kv * ((all + 32 * p.rwp - 1) / (32 * p.rwp))), own_x = (int)(n * n_kv * p.own_blocks);
    const double pre_work = (double)pre_x * ((prefix_rows + 63) / 64), own_work = (double)own_x * ((own_rows + 127) / 128);
    const double share = prefix_rows ? pre_work / (pre_work + own_work) : 0.0;
    const auto best = [&](size_t rows, int x, int room) {
        int at = 1;
        float least = __builtin_inff();
        for (int s = 1; s <= 64; s++) {
            const float cost = pa_cost((int)rows, s, x, room, (float)p.rows);
            if (cost < least)
                least = cost, at = s;
        }
        return at;
    };
    if (own_rows) {
        const int room = (int)((1.0 - share) * slots);
        p.own_splits = best(own_rows, own_x, room < 8 ? 8 : room);
        p.own_len = pa_split_len((int)own_rows, p.own_splits);
    }
    if (prefix_rows) {
        p.xcd_slots = (int)(share * slots / 8 < 1 ? 1 : share * slots / 8);
        const int s = best(prefix_rows, pre_x, p.xcd_slots * 8);
        p.pre_splits = s;
        if (ragged) { // with fewer live rows there may be more of them: room for up to twice as many
            const int most = (int)((prefix_rows + 127) / 128);
            p.pre_splits = 2 * s + 2 < 64 ? 2 * s + 2 : 64;
            p.pre_splits = p.pre_splits > most ? most : p.pre_splits;
        }
        const int64_t x = (int64_t)pre_x * s, cap = ragged && x < slots ? slots : x;
        p.pre_items = (int)((cap + 7) / 8 * 8);
    }
    p.slots = p.pre_splits + p.own_splits;
    return p;
}
static size_t pa_ws_bytes(const PaPlan &p, size_t hd) {
    return p.slots ? 16 + p.rows * p.slots * (hd * 4 + sizeof(float2)) : 0;
}

template <int HDP>
static void pa_launch(const PaPlan &p, const PrefixAttnParams &P, size_t items, hipStream_t st) {
    const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(items), dim3(PA_THREADS), 0, st, P); };
    if (p.rwp == 1) // all lanes' rows are at most 32, and so are one's
        run(prefix_attn_kernel<HDP, 1, 1>);
    else if (p.rwp == 2)
        p.rwo == 1 ? run(prefix_attn_kernel<HDP, 2, 1>) : run(prefix_attn_kernel<HDP, 2, 2>);
    else
        p.rwo == 1 ? run(prefix_attn_kernel<HDP, 4, 1>) : run(prefix_attn_kernel<HDP, 4, 2>);
}

} // namespace lh

using namespace lh;

constexpr size_t PA_MAX_ROWS = 0x3fffffff;
constexpr size_t PA_MAX_STRIDE = (size_t)1 << 23; // the rows of a tile (128) at 32-bit byte offsets from its first
// The sizes the kernels index in 32 bits.
static bool pa_served(size_t n, size_t n_q, size_t n_heads, size_t n_kv, size_t hd) {
    return n && n <= 65535 && n_q && n_q <= 4096 && n_heads && n_heads <= 65535 && n_kv && n_heads % n_kv == 0 && hd &&
           hd % 8 == 0 && hd <= PA_MAX_HD && n * n_q * n_heads <= 0x2000000;
}

// lanes: how many r holds.  The stride of a dimension of one has no part in the layout.
static int kv_rows_check(const loomhip_kv_rows *r, size_t n_kv, size_t hd, size_t lanes, const char *what) {
    if (!r || r->rows == 0)
        return LOOMHIP_OK;
    if (!r->k || !r->v)
        return fail(LOOMHIP_ERR_ARG, "prefix_attn: %s has no keys or values", what);
    if (r->rows > PA_MAX_ROWS)
        return fail(LOOMHIP_DECLINED, "prefix_attn: %zu %s rows not served", r->rows, what);
    if (r->row_stride < hd && r->rows > 1)
        return fail(LOOMHIP_ERR_ARG, "prefix_attn: %s row stride %zu below a head", what, r->row_stride);
    if (r->row_stride > PA_MAX_STRIDE && r->rows > 1)
        return fail(LOOMHIP_DECLINED, "prefix_attn: %s rows %zu elements apart not served", what, r->row_stride);
    if ((uintptr_t)r->k % 16 || (uintptr_t)r->v % 16 || (r->rows > 1 && r->row_stride % 8) ||
        (n_kv > 1 && r->head_stride % 8) || (lanes > 1 && r->lane_stride % 8))
        return fail(LOOMHIP_DECLINED, "prefix_attn: %s rows not at multiples of 16 bytes", what);
    return LOOMHIP_OK;
}

extern "C" {

size_t loomhip_prefix_attn_ws(size_t prefix_rows, size_t own_rows, size_t n, size_t n_q, size_t n_heads,
                              size_t n_kv_heads, size_t head_dim) {
    if (!pa_served(n, n_q, n_heads, n_kv_heads, head_dim) || prefix_rows > PA_MAX_ROWS || own_rows > PA_MAX_ROWS)
        return 0;
    // the larger of the two plans: with q_len, and without
    const PaPlan p = pa_plan(prefix_rows, own_rows, n, n_q, n_heads, n_kv_heads, head_dim, true);
    return pa_ws_bytes(p, head_dim);
}

int loomhip_prefix_attn_dev(const loomhip_kv_rows *prefix, const loomhip_kv_rows *own, const float *q,
                            const int32_t *own_len, const int32_t *q_len, size_t n, size_t n_q, size_t n_heads,
                            size_t n_kv_heads, size_t head_dim, float scale, float *out, int zero_rest, void *ws,
                            size_t ws_bytes, void *stream) {
    if (n == 0 || n_q == 0)
        return LOOMHIP_OK;
    if (!q || !out || n_heads == 0 || n_kv_heads == 0 || n_heads % n_kv_heads)
        return fail(LOOMHIP_ERR_ARG, "prefix_attn: null argument, or %zu heads over %zu key heads", n_heads, n_kv_heads);
    if (head_dim == 0 || head_dim % 8 || head_dim > PA_MAX_HD)
        return fail(LOOMHIP_DECLINED, "prefix_attn: head size %zu not served", head_dim);
    if (!pa_served(n, n_q, n_heads, n_kv_heads, head_dim))
        return fail(LOOMHIP_DECLINED, "prefix_attn: %zu lanes of %zu tokens, %zu heads not served", n, n_q, n_heads);
    if (int rc = kv_rows_check(prefix, n_kv_heads, head_dim, 1, "prefix"))
        return rc;
    if (int rc = kv_rows_check(own, n_kv_heads, head_dim, n, "own"))
        return rc;
    if (own && own->rows && !own_len)
        return fail(LOOMHIP_ERR_ARG, "prefix_attn: own rows without their lengths");
    if (((uintptr_t)own_len | (uintptr_t)q_len) % 4)
        return fail(LOOMHIP_ERR_ARG, "prefix_attn: lengths not aligned to their elements");
    if ((uintptr_t)q % 16 || (uintptr_t)out % 16)
        return fail(LOOMHIP_DECLINED, "prefix_attn: q or out not at a multiple of 16 bytes");
    const PaPlan p = pa_plan(prefix ? prefix->rows : 0, own ? own->rows : 0, n, n_q, n_heads, n_kv_heads, head_dim,
                             q_len != nullptr);
    const size_t need = pa_ws_bytes(p, head_dim);
    if (need && (!ws || ws_bytes < need || (uintptr_t)ws % 16))
        return fail(LOOMHIP_ERR_ARG, "prefix_attn: the workspace takes %zu bytes at a multiple of 16, got %zu", need,
                    ws_bytes);
    const size_t items = p.pre_items + n * n_kv_heads * p.own_splits * p.own_blocks;
    if (items > 0xffffff)
        return fail(LOOMHIP_DECLINED, "prefix_attn: %zu work items not served", items);
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
    P.zero_rest = zero_rest != 0;
    P.pre_splits = p.pre_splits;
    P.pre_items = p.pre_items;
    P.xcd_slots = p.xcd_slots;
    P.own_blocks = p.own_blocks;
    P.own_splits = p.own_splits;
    P.own_len_split = p.own_len;
    P.slots = p.slots;
    P.cut = (int *)ws;
    P.part = (float *)((char *)ws + 16);
    P.ml = (float2 *)(P.part + p.rows * p.slots * head_dim);
    hipStream_t st = stream_of(stream);
    if (items) {
        if (p.hdp == 64)
            pa_launch<64>(p, P, items, st);
        else if (p.hdp == 128)
            pa_launch<128>(p, P, items, st);
        else
            pa_launch<256>(p, P, items, st);
        note_launch();
    }
    const dim3 mg((p.rows + PA_MERGE_ROWS - 1) / PA_MERGE_ROWS);
    if (p.hdp == 64)
        hipLaunchKernelGGL(prefix_attn_merge_kernel<16>, mg, dim3(PA_THREADS), 0, st, P, (int)p.rows);
    else if (p.hdp == 128)
        hipLaunchKernelGGL(prefix_attn_merge_kernel<32>, mg, dim3(PA_THREADS), 0, st, P, (int)p.rows);
    else
        hipLaunchKernelGGL(prefix_attn_merge_kernel<64>, mg, dim3(PA_THREADS), 0, st, P, (int)p.rows);
    note_launch();
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? LOOMHIP_OK : hip_fail(e, "prefix_attn launch");
}

} // extern "C"

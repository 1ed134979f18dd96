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
// Products on the f16 matrix cores (v_mfma_f32_32x32x16_f16), exact to f32's
// standard: the f32 query is scaled by a power of two of its own and split
// into two f16 parts (22 significant bits) against the exact fp16 keys, the
// weights p into two f16 parts against the exact fp16 values, f32 sums.  One
// f16 part alone (11 bits) would leave 2e-4.
//
// S^T = K Q^T: a lane holds one query (column lane % 32) and, of each 32 keys,
// the rows 8 (i / 4) + 4 (lane / 32) + i % 4, i < 16.  These registers are the
// B operand of O^T = V^T P^T as they stand, if its 16 contracted indices
// (lane / 32, j < 8) mean the keys 8 (j / 4) + 4 (lane / 32) + j % 4; the A
// operand's lane then needs 4 + 4 consecutive keys of one value column, which
// the LDS transpose read (ds_read_b64_tr_b16) gives from row-major values.
// The softmax of a query needs one exchange between the two half waves.
#include "runtime.hpp"

namespace lh {

typedef _Float16 pa_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 pa_h2 __attribute__((ext_vector_type(2)));
typedef __fp16 pa_f2 __attribute__((ext_vector_type(2)));
typedef short pa_s4 __attribute__((ext_vector_type(4)));
typedef float pa_f16 __attribute__((ext_vector_type(16)));
typedef float pa_f4 __attribute__((ext_vector_type(4)));

constexpr int PA_THREADS = 256;
constexpr int PA_MAX_HD = 256;
// p = 2^(s - m + PA_SHIFT): the running maximum m moves only where a score
// passes it by more than PA_SLACK (in log2), so most tiles rescale nothing; p
// stays below 2^14 (f16 ends at 2^16) and its low part stays normal down to
// 2^-9 of the maximum, below that off by at most 2^-31 of it.
constexpr float PA_SHIFT = 6.0f, PA_SLACK = 8.0f;

struct PrefixAttnParams {
    loomhip_kv_rows pre, own;
    const float *q;
    const int32_t *own_len, *q_len;
    int n, n_q, n_heads, n_kv, hd;
    float scale;
    float *out;
    // items: prefix [kv][split][row block], then own [lane][kv][split][row block]
    int pre_blocks, pre_splits, pre_len; // row blocks of all lanes, splits, rows per split
    int own_blocks, own_splits, own_len_split;
    int pre_items;
    int slots;   // pre_splits + own_splits
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

// A work group's four waves as RW row groups of 32 queries by 4 / RW key
// groups: a tile of TK cache rows, KPW of them for each wave.  RW = 4 shares a
// tile among 128 queries; RW = 1 takes up to 32 queries (a lane's own rows, a
// small batch) with its waves side by side along the keys.  AHEAD: the next
// tile's loads are in registers while a tile is multiplied; where the tile's
// 64 registers a thread would not fit beside the query and the sums, its work
// groups' short ranges are loaded as they come.
template <int HDP, int RW>
struct PaCfg {
    static constexpr int KW = 4 / RW, KPW = RW == 4 && HDP < 256 ? 64 : 32, TK = KW * KPW;
    static constexpr bool AHEAD = RW > 1 && HDP < 256;
    static constexpr int CH = HDP / 8;                    // 16-byte chunks of a row
    static constexpr int NCH = TK * CH / PA_THREADS;      // chunks a thread stages, of keys and of values each
    static constexpr int TILE_BYTES = TK * HDP * 2;       // keys, or values
    static constexpr int MERGE_BYTES = KW > 1 ? 4 * 32 * HDP * 4 : 0;
    static constexpr int BYTES = 2 * TILE_BYTES > MERGE_BYTES ? 2 * TILE_BYTES : MERGE_BYTES;
};

// Chunk positions inside an LDS row.  Keys are read as 16 bytes of 32 rows: a
// lane's eight neighbours (eight rows) must fall on different 16-byte columns
// of the 256 bytes of banks.  Values are read by 16 lanes as 32 bytes of four
// rows: the four must fall on different 32-byte columns.
template <int HDP>
__device__ __forceinline__ int pa_k_pos(int row, int ch) {
    return ch ^ (HDP == 64 ? (row >> 1) & 7 : row & 15);
}
template <int HDP>
__device__ __forceinline__ int pa_v_pos(int row, int ch) {
    return ch ^ (HDP == 64 ? ((row >> 1) & 3) << 1 : (row & 7) << 1);
}

// Query rows [row0, row0 + RW * 32) of the item (map: their global row, -1 past the end; lim: the first key each
// does not see) against cache rows [k0, k1) at k / v (one head's rows, `stride` elements apart): records into slot
// `slot`.  border: rows from here on are not seen by every query.
template <int HDP, int RW>
__device__ __forceinline__ void pa_item(const PrefixAttnParams &P, const uint16_t *__restrict__ kp,
                                        const uint16_t *__restrict__ vp, size_t stride, int k0, int k1, int border,
                                        int slot, const int *map, const int *lim, char *smem, int *flag) {
    using C = PaCfg<HDP, RW>;
    constexpr int STEPS = HDP / 16, KB = C::KPW / 32, DB = HDP / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int half = lane >> 5, col = lane & 31;
    const int rw = wave % RW, kw = wave / RW;
    const int row = map[rw * 32 + col], limit = lim[rw * 32 + col] < k1 ? lim[rw * 32 + col] : k1;
    const int hd = P.hd;
    char *const sk = smem, *const sv = smem + C::TILE_BYTES;

    // staging: thread t's chunks are t, t + 256, ..
    uint4 rk[C::NCH], rv[C::NCH];
    const int sch = tid % C::CH, srow = tid / C::CH; // its column of chunks, its first row
    const auto stage_load = [&](const uint16_t *__restrict__ p, uint4 *to, int kt) {
        const int left = sch * 8 < hd ? k1 - kt - srow : 0; // rows from its first on
        const size_t off = (size_t)(kt + srow) * stride + sch * 8;
#pragma unroll
        for (int c = 0; c < C::NCH; c++) {
            constexpr int STEP = PA_THREADS / C::CH;
            to[c] = c * STEP < left ? *(const uint4 *)(p + off + (size_t)(c * STEP) * stride) : uint4{0, 0, 0, 0};
        }
    };
    const auto stage_keys = [&] {
#pragma unroll
        for (int c = 0; c < C::NCH; c++) {
            const int r = srow + c * (PA_THREADS / C::CH);
            *(uint4 *)(sk + (r * C::CH + pa_k_pos<HDP>(r, sch)) * 16) = rk[c];
        }
    };
    // Values that some query does not see are left out of the product where they are not finite: they would reach
    // it as 0 * v.  Returns whether there was one.
    const auto stage_values = [&](int kt, bool edge) {
        bool strange = false;
#pragma unroll
        for (int c = 0; c < C::NCH; c++) {
            const int r = srow + c * (PA_THREADS / C::CH);
            if (edge && kt + r >= border) {
                uint32_t *w = (uint32_t *)&rv[c];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const bool lo = (w[e] & 0x7c00u) == 0x7c00u, hi = (w[e] & 0x7c000000u) == 0x7c000000u;
                    strange |= lo | hi;
                    w[e] &= (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0x0000ffffu : 0xffffffffu);
                }
            }
            *(uint4 *)(sv + (r * C::CH + pa_v_pos<HDP>(r, sch)) * 16) = rv[c];
        }
        return strange;
    };
    if (tid == 0)
        *flag = 0;
    if (C::AHEAD) {
        stage_load(kp, rk, k0);
        stage_load(vp, rv, k0);
    }

    // the query: its largest element brought to 2^13 .. 2^14 by a power of two, split into two f16 parts
    pa_h8 qh[STEPS], ql[STEPS];
    float cs; // scores in log2 units per unit of the split query's
    {
        float v[STEPS][8], amax = 0.0f;
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int d = s * 16 + half * 8;
            const bool in = row >= 0 && d < hd;
            const pa_f4 z = {0.0f, 0.0f, 0.0f, 0.0f};
            const pa_f4 a = in ? *(const pa_f4 *)(P.q + (size_t)row * hd + d) : z;
            const pa_f4 b = in ? *(const pa_f4 *)(P.q + (size_t)row * hd + d + 4) : z;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[s][e] = a[e], v[s][4 + e] = b[e];
                amax = fmaxf(amax, fmaxf(fabsf(a[e]), fabsf(b[e])));
            }
        }
        amax = pa_half_max(amax);
        const int k = amax > 0.0f && amax < __builtin_inff() ? pa_clamp(13 - ilogbf(amax), -120, 120) : 0;
        const float f = ldexpf(P.scale < 0.0f ? -1.0f : 1.0f, k);
        cs = ldexpf(fabsf(P.scale) * 0x1.715476p+0f, -k);
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
    const int k_at = ((kb + col) * C::CH + pa_k_pos<HDP>(kb + col, half)) * 16;
    const int v_row = kb + 4 * half + ((lane & 15) >> 2), v_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const int v_at = (v_row * C::CH + pa_v_pos<HDP>(v_row, v_col / 8)) * 16 + v_col % 8 * 2;
    pa_f16 o[DB];
#pragma unroll
    for (int b = 0; b < DB; b++)
#pragma unroll
        for (int i = 0; i < 16; i++)
            o[b][i] = 0.0f;
    float m = -__builtin_inff(), l = 0.0f;

    for (int kt = k0; kt < k1; kt += C::TK) {
        const bool edge = kt + C::TK > border; // some row of the tile is not seen by every query
        __syncthreads();
        bool strange;
        if constexpr (C::AHEAD) {
            stage_keys();
            strange = stage_values(kt, edge);
        } else {
            stage_load(kp, rk, kt);
            stage_keys();
            stage_load(vp, rv, kt);
            strange = stage_values(kt, edge);
        }
        if (edge && strange)
            *flag = 1;
        __syncthreads();
        if (C::AHEAD && kt + C::TK < k1) {
            stage_load(kp, rk, kt + C::TK);
            stage_load(vp, rv, kt + C::TK);
        }

        // scores of the wave's KPW keys
        pa_f16 s[KB];
#pragma unroll
        for (int b = 0; b < KB; b++) {
#pragma unroll
            for (int i = 0; i < 16; i++)
                s[b][i] = 0.0f;
#pragma unroll
            for (int st = 0; st < STEPS; st++) {
                // pa_k_pos of row kb + b * 32 + col, chunk 2 st + half: the row's part and st's by exclusive or
                const pa_h8 a = *(const pa_h8 *)(sk + ((k_at ^ (st * 32)) + b * 32 * C::CH * 16));
                s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[st], s[b], 0, 0, 0);
                s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[st], s[b], 0, 0, 0);
            }
        }
        if (edge || kt + C::TK > k1) {
            const int seen = limit - kt - kb - 4 * half; // of the lane's keys, counted from its first
#pragma unroll
            for (int b = 0; b < KB; b++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    s[b][i] = b * 32 + 8 * (i / 4) + i % 4 < seen ? s[b][i] : -__builtin_inff();
        }
        // the running maximum
        float mx = s[0][0];
#pragma unroll
        for (int b = 0; b < KB; b++)
#pragma unroll
            for (int i = 0; i < 16; i++)
                mx = fmaxf(mx, s[b][i]);
        mx = pa_half_max(mx) * cs;
        if (__any(mx > m + PA_SLACK)) {
            const float m2 = fmaxf(m, mx);
            const float f = m == m2 ? 1.0f : __builtin_amdgcn_exp2f(m - m2); // -inf before the first seen key: 0
            m = m2;
            l *= f;
#pragma unroll
            for (int b = 0; b < DB; b++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    o[b][i] *= f;
        }
        const float sub = PA_SHIFT - (m == -__builtin_inff() ? 0.0f : m);
        // weights, in two f16 parts
        pa_h8 ph[KB][2], pl[KB][2];
#pragma unroll
        for (int b = 0; b < KB; b++)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], cs, sub));
                const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i + 1], cs, sub));
                l += p0 + p1;
                const pa_h2 h = __builtin_bit_cast(pa_h2, __builtin_amdgcn_cvt_pkrtz(p0, p1));
                const float r0 = __builtin_fmaf((float)h[0], -1.0f, p0), r1 = __builtin_fmaf((float)h[1], -1.0f, p1);
                const pa_h2 g = __builtin_bit_cast(pa_h2, __builtin_amdgcn_cvt_pkrtz(r0, r1));
                ph[b][i / 8][i % 8] = h[0], ph[b][i / 8][i % 8 + 1] = h[1];
                pl[b][i / 8][i % 8] = g[0], pl[b][i / 8][i % 8 + 1] = g[1];
            }
        // O^T += V^T P^T
#pragma unroll
        for (int b = 0; b < KB; b++)
#pragma unroll
            for (int st = 0; st < 2; st++)
#pragma unroll
                for (int db = 0; db < DB; db++) {
                    // rows v_row + b * 32 + st * 16 (+ 8), column db * 32 + v_col: db's part by exclusive or
                    const int at = (v_at ^ (db * 64)) + (b * 32 + st * 16) * C::CH * 16;
                    pa_s4 a[2];
#pragma unroll
                    for (int x = 0; x < 2; x++)
                        a[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) pa_s4 *)(sv + at + x * 8 * C::CH * 16));
                    const pa_h8 va = __builtin_bit_cast(
                        pa_h8, __builtin_shufflevector(a[0], a[1], 0, 1, 2, 3, 4, 5, 6, 7));
                    o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, ph[b][st], o[db], 0, 0, 0);
                    o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pl[b][st], o[db], 0, 0, 0);
                }
    }
    l = pa_half_sum(l);

    // records: o as it stands relative to m (both carry PA_SHIFT)
    if constexpr (C::KW == 1) {
        if (row >= 0) {
            const size_t rec = (size_t)row * P.slots + slot;
            if (half == 0)
                P.ml[rec] = make_float2(m, l);
            float *dst = P.part + rec * hd;
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const int d = db * 32 + 2 * i + 4 * half;
                    if (d < hd)
                        *(pa_f4 *)(dst + d) = pa_f4{o[db][i], o[db][i + 1], o[db][i + 2], o[db][i + 3]};
                }
        }
    } else {
        // the key groups of a row group joined through LDS
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
        for (int at = tid; at < RW * 32 * (HDP / 4); at += PA_THREADS) {
            const int rr = at / (HDP / 4), d = at % (HDP / 4) * 4; // row of the block, its column
            const int R = map[rr];
            if (R < 0 || d >= hd)
                continue;
            const int g = rr / 32, c = rr % 32;
            pa_f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < C::KW; w++)
                v += *(const pa_f4 *)((const float *)smem + (size_t)(g + w * RW) * 32 * HDP + c * HDP +
                                      ((d / 4 + c) % (HDP / 4)) * 4);
            const size_t rec = (size_t)R * P.slots + slot;
            *(pa_f4 *)(P.part + rec * hd + d) = v;
            if (d == 0) {
                float mm = sm[g][c], ll = 0.0f;
#pragma unroll
                for (int w = 1; w < C::KW; w++)
                    mm = fmaxf(mm, sm[g + w * RW][c]);
#pragma unroll
                for (int w = 0; w < C::KW; w++)
                    ll += sl[g + w * RW][c] * (sm[g + w * RW][c] == mm ? 1.0f : __builtin_amdgcn_exp2f(sm[g + w * RW][c] - mm));
                P.ml[rec] = make_float2(mm, ll);
            }
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

// The block's rows of all lanes' live query rows (lane, token < q_len, head of the group), [r0, r0 + R): false if
// the batch has no such rows.  Every thread takes lanes tid, tid + 256, ..; the running sum of their token counts
// tells which of them fall into the block.
template <int R>
__device__ __forceinline__ bool pa_map_all(const PrefixAttnParams &P, int kvh, int r0, int *map, int *scan) {
    const int G = P.n_heads / P.n_kv, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int r = tid; r < R; r += PA_THREADS)
        map[r] = -1;
    __syncthreads();
    if (!P.q_len) {
        const int rows = P.n * P.n_q * G;
        for (int r = tid; r < R; r += PA_THREADS)
            if (r0 + r < rows)
                map[r] = (r0 + r) / G * P.n_heads + kvh * G + (r0 + r) % G;
        __syncthreads();
        return r0 < rows;
    }
    int before = 0; // tokens of the lanes already scanned
    for (int i0 = 0; i0 < P.n; i0 += PA_THREADS) {
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
        const int first = (before + c - L) * G; // the lane's first row
        for (int r = first < r0 ? r0 - first : 0; r < L * G && first + r < r0 + R; r++)
            map[first + r - r0] = (i * P.n_q + r / G) * P.n_heads + kvh * G + r % G;
        before += all;
        if (before * G >= r0 + R)
            break;
    }
    __syncthreads();
    return r0 < before * G;
}

template <int HDP, int RWP, int RWO>
__global__ __launch_bounds__(PA_THREADS, HDP == 256 ? 1 : 2) void prefix_attn_kernel(PrefixAttnParams P) {
    constexpr int BP = PaCfg<HDP, RWP>::BYTES, BO = PaCfg<HDP, RWO>::BYTES;
    __shared__ __attribute__((aligned(16))) char smem[BP > BO ? BP : BO];
    constexpr int RM = (RWP > RWO ? RWP : RWO) * 32;
    __shared__ int map[RM], lim[RM], scan[PA_THREADS / 64], flag;
    const int G = P.n_heads / P.n_kv, tid = threadIdx.x;
    if ((int)blockIdx.x < P.pre_items) {
        // Work groups go to the eight XCDs in turn: the row blocks of one (key head, split) get numbers 8 apart, so
        // they find its rows in one L2.
        const int b = blockIdx.x, at = b >> 3;
        const int ks = (b & 7) + 8 * (at / P.pre_blocks), rb = at % P.pre_blocks;
        if (ks >= P.n_kv * P.pre_splits)
            return;
        const int kvh = ks / P.pre_splits, sp = ks % P.pre_splits;
        if (!pa_map_all<RWP * 32>(P, kvh, rb * RWP * 32, map, scan))
            return;
        const int rows = (int)P.pre.rows, k0 = sp * P.pre_len, k1 = k0 + P.pre_len < rows ? k0 + P.pre_len : rows;
        for (int r = tid; r < RWP * 32; r += PA_THREADS)
            lim[r] = k1;
        __syncthreads();
        pa_item<HDP, RWP>(P, P.pre.k + (size_t)kvh * P.pre.head_stride, P.pre.v + (size_t)kvh * P.pre.head_stride,
                          P.pre.row_stride, k0, k1, k1, sp, map, lim, smem, &flag);
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
            lim[r] = in ? pa_seen(len, L, j) : 0;
        }
        __syncthreads();
        const size_t base = (size_t)i * P.own.lane_stride + (size_t)kvh * P.own.head_stride;
        pa_item<HDP, RWO>(P, P.own.k + base, P.own.v + base, P.own.row_stride, k0, k1, pa_seen(len, L, 0),
                          P.pre_splits + sp, map, lim, smem, &flag);
    }
}

// A row's records joined: M = max m, out = sum 2^(m - M) o / sum 2^(m - M) l, a wave per row.
constexpr int PA_MERGE_ROWS = PA_THREADS / 64;
__global__ __launch_bounds__(PA_THREADS) void prefix_attn_merge_kernel(PrefixAttnParams P, int rows) {
    const int row = blockIdx.x * PA_MERGE_ROWS + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= rows)
        return;
    const int token = row / P.n_heads, i = token / P.n_q, j = token % P.n_q;
    if (j >= pa_q_len(P, i))
        return;
    const int len = pa_own_len(P, i);
    // the slots that were written: the prefix's, and the own splits that start below the lane's length
    const int own = P.own_splits ? (len + P.own_len_split - 1) / P.own_len_split : 0, slots = P.pre_splits + own;
    const float2 *ml = P.ml + (size_t)row * P.slots;
    const float *part = P.part + (size_t)row * P.slots * P.hd;
    float M = -__builtin_inff();
    for (int s = lane; s < slots; s += 64)
        M = fmaxf(M, ml[s].x);
    M = wave_max(M);
    float l = 0.0f;
    pa_f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < slots; s++) {
        const float2 r = ml[s];
        const float w = r.x == M ? 1.0f : __builtin_amdgcn_exp2f(r.x - M);
        l += r.y * w;
        if (lane * 4 < P.hd) {
            const pa_f4 v = *(const pa_f4 *)(part + (size_t)s * P.hd + lane * 4);
            o += v * w;
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l; // nothing seen: zero
    if (lane * 4 < P.hd)
        *(pa_f4 *)(P.out + (size_t)row * P.hd + lane * 4) = o * inv;
}

// How a call is cut into items.
struct PaPlan {
    int hdp, rwp, rwo;
    int pre_blocks, pre_splits, pre_len, own_blocks, own_splits, own_len, slots;
    size_t rows;
};
static PaPlan pa_plan(size_t prefix_rows, size_t own_rows, size_t n, size_t n_q, size_t n_heads, size_t n_kv,
                      size_t hd) {
    PaPlan p = {};
    const size_t G = n_heads / n_kv;
    p.hdp = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
    p.rows = n * n_q * n_heads;
    const size_t all = n * n_q * G, mine = n_q * G;
    p.rwp = all <= 32 ? 1 : all <= 64 ? 2 : 4;
    p.rwo = mine <= 32 ? 1 : 2;
    constexpr size_t ITEMS = 512, MIN_ROWS = 128;
    const auto cut = [](size_t rows, size_t others, int *splits, int *len) {
        if (rows == 0)
            return;
        size_t s = (ITEMS + others - 1) / others, most = (rows + MIN_ROWS - 1) / MIN_ROWS;
        s = s > most ? most : s < 1 ? 1 : s;
        const size_t ln = ((rows + s - 1) / s + MIN_ROWS - 1) / MIN_ROWS * MIN_ROWS;
        *len = (int)ln;
        *splits = (int)((rows + ln - 1) / ln);
    };
    p.pre_blocks = (int)((all + 32 * p.rwp - 1) / (32 * p.rwp));
    p.own_blocks = (int)((mine + 32 * p.rwo - 1) / (32 * p.rwo));
    cut(prefix_rows, n_kv * p.pre_blocks, &p.pre_splits, &p.pre_len);
    cut(own_rows, n * n_kv * p.own_blocks, &p.own_splits, &p.own_len);
    p.slots = p.pre_splits + p.own_splits;
    return p;
}

template <int HDP, int RWP>
static void pa_launch(const PaPlan &p, const PrefixAttnParams &P, size_t items, hipStream_t st) {
    if (p.rwo == 1)
        hipLaunchKernelGGL((prefix_attn_kernel<HDP, RWP, 1>), dim3(items), dim3(PA_THREADS), 0, st, P);
    else
        hipLaunchKernelGGL((prefix_attn_kernel<HDP, RWP, 2>), dim3(items), dim3(PA_THREADS), 0, st, P);
}
template <int HDP>
static void pa_launch(const PaPlan &p, const PrefixAttnParams &P, size_t items, hipStream_t st) {
    if (p.rwp == 1)
        pa_launch<HDP, 1>(p, P, items, st);
    else if (p.rwp == 2)
        pa_launch<HDP, 2>(p, P, items, st);
    else
        pa_launch<HDP, 4>(p, P, items, st);
}

} // namespace lh

using namespace lh;

constexpr size_t PA_MAX_ROWS = 0x3fffffff;
// The sizes the kernels index in 32 bits.
static bool pa_served(size_t n, size_t n_q, size_t n_heads, size_t n_kv, size_t hd) {
    return n && n <= 65535 && n_q && n_q <= 4096 && n_heads && n_heads <= 65535 && n_kv && n_heads % n_kv == 0 && hd &&
           hd % 8 == 0 && hd <= PA_MAX_HD && n * n_q * n_heads <= 0x2000000;
}

static int kv_rows_check(const loomhip_kv_rows *r, size_t n_kv, size_t hd, bool lanes, const char *what) {
    if (!r || r->rows == 0)
        return LOOMHIP_OK;
    if (!r->k || !r->v)
        return fail(LOOMHIP_ERR_ARG, "prefix_attn: %s has no keys or values", what);
    if (r->rows > PA_MAX_ROWS)
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
    if (!pa_served(n, n_q, n_heads, n_kv_heads, head_dim) || prefix_rows > PA_MAX_ROWS || own_rows > PA_MAX_ROWS)
        return 0;
    const PaPlan p = pa_plan(prefix_rows, own_rows, n, n_q, n_heads, n_kv_heads, head_dim);
    return p.rows * p.slots * (head_dim * 4 + sizeof(float2));
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
    if (!pa_served(n, n_q, n_heads, n_kv_heads, head_dim))
        return fail(LOOMHIP_DECLINED, "prefix_attn: %zu lanes of %zu tokens, %zu heads not served", n, n_q, n_heads);
    if (int rc = kv_rows_check(prefix, n_kv_heads, head_dim, false, "prefix"))
        return rc;
    if (int rc = kv_rows_check(own, n_kv_heads, head_dim, true, "own"))
        return rc;
    if (own && own->rows && !own_len)
        return fail(LOOMHIP_ERR_ARG, "prefix_attn: own rows without their lengths");
    if ((uintptr_t)q % 16 || (uintptr_t)out % 16)
        return fail(LOOMHIP_DECLINED, "prefix_attn: q or out not at a multiple of 16 bytes");
    const PaPlan p = pa_plan(prefix ? prefix->rows : 0, own ? own->rows : 0, n, n_q, n_heads, n_kv_heads, head_dim);
    const size_t need = p.rows * p.slots * (head_dim * 4 + sizeof(float2));
    if (need && (!ws || ws_bytes < need || (uintptr_t)ws % 16))
        return fail(LOOMHIP_ERR_ARG, "prefix_attn: the workspace takes %zu bytes at a multiple of 16, got %zu", need,
                    ws_bytes);
    const size_t pre_items = p.pre_splits ? (n_kv_heads * p.pre_splits + 7) / 8 * 8 * p.pre_blocks : 0;
    const size_t items = pre_items + n * n_kv_heads * p.own_splits * p.own_blocks;
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
    P.pre_blocks = p.pre_blocks;
    P.pre_splits = p.pre_splits;
    P.pre_len = p.pre_len;
    P.own_blocks = p.own_blocks;
    P.own_splits = p.own_splits;
    P.own_len_split = p.own_len;
    P.pre_items = (int)pre_items;
    P.slots = p.slots;
    P.part = (float *)ws;
    P.ml = (float2 *)((char *)ws + p.rows * p.slots * head_dim * 4);
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
    hipLaunchKernelGGL(prefix_attn_merge_kernel, dim3((p.rows + PA_MERGE_ROWS - 1) / PA_MERGE_ROWS), dim3(PA_THREADS), 0,
                       st, P, (int)p.rows);
    note_launch();
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? LOOMHIP_OK : hip_fail(e, "prefix_attn launch");
}

} // extern "C"

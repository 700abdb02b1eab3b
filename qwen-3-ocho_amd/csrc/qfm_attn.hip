// qfm_attn.hip -- attention of drafted rows over the quantised cache
// (qfm_tree_attn).
//
// One workgroup of four waves takes up to 16 RB rows (nodes x the query heads
// that share a key/value head) and a range of 32-token tiles; the waves take
// the tiles in turn, each with a running maximum, sum and result of its own,
// joined through LDS at the end and, where a sequence's keys are split over
// workgroups, once more by k_tree_join. No wave waits for another inside the
// loop, and every cached byte enters the registers of one wave only, straight
// from memory:
//   S^T = K Q^T   the MFMA's rows are tokens. A lane's 16 bytes of a key row
//                 (d = 64 c + 16 g + 0..15, g = lane / 16) are two k-steps; Q is
//                 laid out to match.
//   O^T = V^T P^T lane (g, r) of S^T holds tokens 4 g + i of both 16-token halves
//                 for row r, which is the layout the second product wants of
//                 P^T when its inner index runs over (half, 4 g + i) in that
//                 order: no exchange between lanes. V's layout (four tokens of
//                 a channel side by side) gives a lane the same tokens of 4
//                 channels in 16 bytes.
// Codes are widened to fp16 exactly (int8 and E4M3 both fit); a row of Q is
// scaled to [2^14, 2^15) by a power of two; p times the value's scale is kept
// within fp16 by a power of two of the largest value scale so far. Q is one fp16
// number (two for F32 rows: bf16 and fp16 fit one), p one for BF16 rows, whose
// results are rounded to 2^-8 anyway, and two for F16 and F32.
//
// The bound of a large call is its cache: 37 users of 2 to 4 thousand tokens,
// 124 MB of codes and scales, take 33.0 us (3.8 TB/s, a plain sum over as much
// memory reads 4.0). Many rows a head are bound by the softmax between the two
// products, which costs a wave about half as long again as their MFMAs (61-node trees of five users, 26 GFLOP: 64 us; k_tree_wide below). Few
// rows and short contexts are bound by the chain of a launch, the page table,
// the first tile, a join through LDS and one through memory (1021 tokens: 9.8
// us); what is there to fill the GPU is the split of the keys.
#include "qfm_kv.h"
#include "qfm_mfma.h"
#include "qfm_internal.h"
#include <algorithm>

namespace qfm {

constexpr int kAttnWaves = 4;
constexpr int kMaxSplits = 128;    // two a lane in the join
constexpr long kMaxTokens = (1l << 31) - (1 << 16);   // 32 x a tile's number stays an int, past the last one too
constexpr float kNoMax = -3.402823466e38f;
constexpr float kLazy = 8.0f;      // the maximum may be exceeded by 2^8 before sums and results are rescaled
constexpr int kVeMin = -118;       // least exponent of the value scale that the products are kept relative to

struct AttnArgs {
    const uint8_t *q;
    uint8_t *out;
    int G, T, max_nodes, splits;   // splits: 1, or workgroups a sequence on average
    int dealt, rows;               // rows: what po and pml have room for
    long qrs, qhs, ors, ohs;
    const int *row_start, *ctx;
    const uint64_t *tree;
    float scale;
    float *po;                     // [rows][q_heads][D], normalised
    float2 *pml;                   // [rows][q_heads] {maximum (base 2), sum}
    int2 *parts;                   // [n_seq] {splits, first row of po and pml}
};

// the rows of sequence s: first row, count
__device__ __forceinline__ int2 seq_rows(const int *row_start, int s, int T, int max_nodes) {
    const int r0 = row_start[s], r1 = min(row_start[s + 1], T);
    return make_int2(r0, r0 < 0 || r1 <= r0 ? 0 : min(r1 - r0, max_nodes));
}

// inclusive sums over the lanes
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);      // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);      // row_bcast 15, 31
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}
// sum and maximum (of values from 0 on) over the lanes, as scalars
__device__ __forceinline__ int wave_add(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }
__device__ __forceinline__ int wave_top(int v) {
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));
    return __builtin_amdgcn_readlane(v, 63);
}

// A workgroup's share: tiles t0 .. t1 - 1 of sequence seq (rows r0 .. r0 + m - 1,
// ctx tokens before them, len with them), which is split n ways; row: its first
// row of the partial results, first: that of the sequence. m = 0: nothing.
struct Share { int seq, r0, m, ctx, len, t0, t1, n, row, first; };
constexpr int kDealSeqs = 256;     // four a lane
// Sequences differ in length, so the workgroups along x are dealt out by tiles:
// chunks of as few tiles as still give every chunk a workgroup, found by bisection
// between total / workgroups and what is enough whatever the remainders (a chunk
// at most 1/8 of that range longer than need be). Every wave works this out for
// itself from all the lengths, one to four a lane: about 1 us of a call (16 users
// of 4000 tokens 31.9 -> 33.4), for which 61-node trees of five users take 64 us
// instead of 71 and one user of 131071 tokens among 36 of 1000 64 instead of 231.
__device__ __forceinline__ Share share_of(const KvView &c, const AttnArgs &a, int lane) {
    const long cap = min((long)c.max_pages << c.page_log2, kMaxTokens);
    Share w{};
    int nt, per, j;
    if (!a.dealt) {
        w.seq = (int)blockIdx.z;
        const int2 sr = seq_rows(a.row_start, w.seq, a.T, a.max_nodes);
        w.r0 = sr.x;
        w.m = sr.y;
        w.ctx = (int)min((long)max(a.ctx[w.seq], 0), cap);
        w.n = a.splits;
        j = (int)blockIdx.x;
        nt = ((int)min((long)w.ctx + w.m, cap) + 31) >> 5;
        per = (nt + w.n - 1) / w.n;
        w.row = w.n * w.r0;
    } else {
        constexpr int Q = kDealSeqs / 64;
        const int slots = (int)gridDim.x, slot = (int)blockIdx.x;
        int r0[Q], m[Q], ctx[Q], tiles[Q], total = 0, most = 0, have = 0;
#pragma unroll
        for (int q = 0; q < Q; q++) {
            r0[q] = m[q] = ctx[q] = tiles[q] = 0;
            if (64 * q < c.n_seq) {
                const int s = min(64 * q + lane, c.n_seq - 1);
                const int2 sr = seq_rows(a.row_start, s, a.T, a.max_nodes);
                r0[q] = sr.x;
                m[q] = 64 * q + lane < c.n_seq ? sr.y : 0;
                ctx[q] = (int)min((long)max(a.ctx[s], 0), cap);
                tiles[q] = m[q] ? ((int)min((long)ctx[q] + m[q], cap) + 31) >> 5 : 0;
                total += tiles[q];
                most = max(most, tiles[q]);
                have += (int)__popcll(__ballot(tiles[q] > 0));
            }
        }
        total = wave_add(total);
        most = wave_top(most);
        // lo from below and hi from above by more than the roundings of their quotients (slots > sequences)
        int lo = max(max(1, (int)((float)total * __builtin_amdgcn_rcpf((float)slots) * (1.0f - 0x1p-20f))), (most + kMaxSplits - 1) / kMaxSplits);
        int hi = max(lo, (int)((float)total * __builtin_amdgcn_rcpf((float)(slots - have)) * (1.0f + 0x1p-20f)) + 1);
        int n[Q], mid = hi;
        // n: tiles in chunks of mid, rounded up; at most kMaxSplits, so that the fp32 quotient is off by one at most
        const auto chunks = [&]() {
            const float inv = __builtin_amdgcn_rcpf((float)mid);
            int sum = 0;
#pragma unroll
            for (int q = 0; q < Q; q++)
                if (64 * q < c.n_seq) {
                    const int f = (int)((float)tiles[q] * inv), rest = tiles[q] - f * mid;
                    n[q] = f + (rest > 0) + (rest > mid);
                    sum += n[q];
                }
            return sum;
        };
        for (int i = 0; i < 3 && lo < hi; i++) {
            mid = (lo + hi) >> 1;
            if (wave_add(chunks()) <= slots) hi = mid;
            else lo = mid + 1;
        }
        mid = per = __builtin_amdgcn_readfirstlane(hi);
        chunks();
        nt = j = 0;
        int before = 0, rows = 0;                              // workgroups and rows of the sequences before
#pragma unroll
        for (int q = 0; q < Q; q++)
            if (64 * q < c.n_seq) {
                const int upto = before + wave_scan(n[q]), r = rows + wave_scan(n[q] * m[q]);
                const uint64_t hit = __ballot(slot < upto && slot >= upto - n[q]);
                if (hit) {
                    const int l = __builtin_ctzll(hit);
                    w.seq = 64 * q + l;
                    w.r0 = __builtin_amdgcn_readlane(r0[q], l);
                    w.m = __builtin_amdgcn_readlane(m[q], l);
                    w.ctx = __builtin_amdgcn_readlane(ctx[q], l);
                    w.n = __builtin_amdgcn_readlane(n[q], l);
                    nt = __builtin_amdgcn_readlane(tiles[q], l);
                    j = slot - __builtin_amdgcn_readlane(upto - n[q], l);
                    w.row = __builtin_amdgcn_readlane(r - n[q] * m[q], l);
                }
                before = __builtin_amdgcn_readlane(upto, 63);
                rows = __builtin_amdgcn_readlane(r, 63);
            }
    }
    w.len = (int)min((long)w.ctx + w.m, cap);
    w.t0 = j * per;
    w.t1 = min(nt, w.t0 + per);
    // ranges of rows that overlap would need more room than there is: no share
    if (w.n > 1 && (w.row < 0 || w.row + w.n * w.m > a.rows)) w.m = 0;
    w.first = w.row;
    w.row += j * w.m;
    return w;
}
// what the joins need to know. Behind the loop: a store ahead of it would have the
// page table read through the vector cache, tile by tile behind the keys (61-node
// trees 88 us for 73)
__device__ __forceinline__ void put_parts(const AttnArgs &a, const Share &w) {
    if (a.dealt && blockIdx.y == 0 && w.row == w.first && threadIdx.x == 0) a.parts[w.seq] = make_int2(w.n, w.first);
}
// for the joins: a sequence's splits and first row, 0 splits for none or for
// results that are in place already
template <bool DEALT>
__device__ __forceinline__ int2 parts_of(const AttnArgs &a, int seq, int2 sr) {
    if constexpr (!DEALT) return make_int2(a.splits, a.splits * sr.x);
    const int2 p = a.parts[seq];
    const bool right = sr.y > 0 && p.x > 1 && p.x <= kMaxSplits && p.y >= 0 && p.y <= a.rows && p.x * sr.y <= a.rows - p.y;
    return make_int2(right ? p.x : 0, p.y);
}

template <int FMT>
__device__ __forceinline__ void codes16(u32x4_t w, f16x8_t &a, f16x8_t &b) {
    if constexpr (FMT == QFM_KV_INT8) {
        i8_to_f16(w, a, b);
    } else {
        uint32_t o[8];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            o[2 * q] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[q], 1.0f, 0));
            o[2 * q + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[q], 1.0f, 1));
        }
        a = __builtin_bit_cast(f16x8_t, u32x4_t{o[0], o[1], o[2], o[3]});
        b = __builtin_bit_cast(f16x8_t, u32x4_t{o[4], o[5], o[6], o[7]});
    }
}

__device__ __forceinline__ float max_over_g(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float sum_over_g(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ float pow2_ratio(int d) { return d < -126 ? 0.0f : exp2i(min(d, 127)); }

// the bytes of the first n of four tokens: a NaN code of E4M3 behind them would
// make NaN of a product with 0
__device__ __forceinline__ uint32_t token_bytes(int n) { return n == 4 ? ~0u : (1u << (8 * n)) - 1u; }

// 4 values rounded to the type
template <int DT>
__device__ __forceinline__ void store4(uint8_t *out, long at, float4 v) {
    if constexpr (DT == QFM_DT_F32) *reinterpret_cast<float4 *>(out + at * 4) = v;
    else *reinterpret_cast<uint2 *>(out + at * 2) = make_uint2(pack2<DT>(v.x, v.y), pack2<DT>(v.z, v.w));
}

// One wave's rows: running maximum (base 2), sum and result, and the softmax
// step of a tile. Result element i of o[rb][k][q] is channel 64 k + 16 g + 4 i + q
// of row l16 of block rb.
// how many fp16 numbers an element of Q and a weight p take
constexpr int q_parts(int dt) { return dt == QFM_DT_F32 ? 2 : 1; }
constexpr int p_parts(int dt) { return dt == QFM_DT_BF16 ? 1 : 2; }

template <int RB, int NC, int PP>
struct Rows {
    f32x4_t o[RB][NC][4];
    float m[RB], l[RB], qs[RB];
    uint64_t see[RB];
    int ve;
    __device__ __forceinline__ void clear() {
        ve = kVeMin;
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
            m[rb] = kNoMax;
            l[rb] = 0.0f;
#pragma unroll
            for (int k = 0; k < NC; k++)
#pragma unroll
                for (int q = 0; q < 4; q++) o[rb][k][q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
    }
    // scores s of tokens 4 g + e of half i, without the scales; n4[i]: how many of
    // this lane's four tokens exist, j0[i]: the first one's node number
    __device__ __forceinline__ void hide(f32x4_t (&s)[RB][2], float (&vs)[2][4], const int (&n4)[2], const int (&j0)[2]) const {
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                // a value that is NaN reaches the rows that see it through their scores
                const bool lost = vs[i][e] != vs[i][e];
                const uint32_t nan = lost ? 0x7FC00000u : 0u;
                vs[i][e] = ((e >= n4[i]) | lost) ? 0.0f : vs[i][e];
                const int j = j0[i] + e;
                const uint64_t bit = 1ull << (j & 63);
#pragma unroll
                for (int rb = 0; rb < RB; rb++) {
                    const bool no = (e >= n4[i]) | ((j >= 0) & ((see[rb] & bit) == 0));
                    const float x = __uint_as_float(__float_as_uint(s[rb][i][e]) | nan);
                    s[rb][i][e] = no ? -INFINITY : x;
                }
            }
    }
    // p times the value scales, as the second product's operand
    __device__ __forceinline__ void step(const f32x4_t (&s)[RB][2], float (&vs)[2][4], f16x8_t (&pf)[RB][PP]) {
        bool grow = false;
        float top[RB], vm = 0.0f;
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
            top[rb] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) top[rb] = fmaxf(top[rb], s[rb][i][e]);
            top[rb] *= qs[rb];
            grow |= top[rb] > m[rb] + kLazy;
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) vm = fmaxf(vm, vs[i][e]);
        grow |= vm >= exp2i(ve) * 2.0f;
        if (__any(grow)) {
            const int vn = max(ve, (int)(__float_as_uint(max_over_g(vm)) >> 23) - 127);
            const float vf = pow2_ratio(ve - vn);
            ve = vn;
#pragma unroll
            for (int rb = 0; rb < RB; rb++) {
                const float mn = fmaxf(m[rb], max_over_g(top[rb])), f = __builtin_amdgcn_exp2f(m[rb] - mn);
                m[rb] = mn;
                l[rb] *= f;
#pragma unroll
                for (int k = 0; k < NC; k++)
#pragma unroll
                    for (int q = 0; q < 4; q++) o[rb][k][q] *= f * vf;
            }
        }
        const float vi = exp2i(6 - ve);
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) vs[i][e] *= vi;
#pragma unroll
        for (int rb = 0; rb < RB; rb++)
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(s[rb][i][e], qs[rb], -m[rb]));
                    l[rb] += p;
                    float x = p * vs[i][e];
                    // the rounded product, to both uses: the compiler may else round the exact one for the
                    // first part and take the remainder of the other, a whole fp16 step apart next to a tie
                    if constexpr (PP == 2) asm("" : "+v"(x));
                    const _Float16 hi = (_Float16)x;
                    pf[rb][0][4 * i + e] = hi;
                    if constexpr (PP == 2) pf[rb][1][4 * i + e] = (_Float16)(x - (float)hi);
                }
    }
};

// A row's 16 NC values of this lane (channels 64 k + 16 g + 8 j + e): as they
// come, then as fp16 fragments scaled by a power of two; widen() returns what
// undoes it, times scale log2(e).
template <int NC, int DT>
struct QRow {
    static constexpr int ES = DT == QFM_DT_F32 ? 4 : 2, QP = q_parts(DT);
    u32x4_t raw[NC][2][ES / 2];
    // row r (node r / G, head r % G of the group) of the sequence whose first row is `first`
    __device__ __forceinline__ void load(const AttnArgs &a, int first, int h, int r, int node, int g) {
        const uint8_t *p = a.q + ((first + node) * a.qrs + (long)(h * a.G + r - node * a.G) * a.qhs) * ES;
#pragma unroll
        for (int k = 0; k < NC; k++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int w = 0; w < ES / 2; w++)
                    raw[k][j][w] = *reinterpret_cast<const u32x4_t *>(p + (64 * k + 16 * g + 8 * j) * ES + 16 * w);
    }
    __device__ __forceinline__ float widen(float scale, f16x8_t (&f)[NC][2][QP]) const {
        float v[NC][2][8], m = 0.0f;
#pragma unroll
        for (int k = 0; k < NC; k++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                load8<DT>(&raw[k][j][0], v[k][j]);
#pragma unroll
                for (int e = 0; e < 8; e++) m = fmaxf(m, fabsf(v[k][j][e]));
            }
        const float top = max_over_g(m);
        const int k2 = f16_exp(top);
        // a row with an infinity is NaN wherever it sees a key, also where every score would be -infinity
        const float sc = top < INFINITY ? exp2i(k2) : NAN;
#pragma unroll
        for (int k = 0; k < NC; k++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float x = v[k][j][e] * sc;
                    f[k][j][0][e] = (_Float16)x;
                    if constexpr (QP == 2) f[k][j][1][e] = (_Float16)(x - (float)(_Float16)x);
                }
        return exp2i(-k2) * (scale * 1.4426950408889634f);
    }
};
__device__ __forceinline__ uint64_t node_mask(const AttnArgs &a, int first, int node) {
    return a.tree ? a.tree[first + node] : node == 63 ? ~0ull : (2ull << node) - 1;
}

// a 32-token tile of keys or values, as the lanes hold it; scale (with the keys):
// of key lane (lane < 32) or of value lane - 32
template <int NC>
struct Tile {
    u32x4_t x[2][NC];
    float scale;
};

template <int FMT, int D, int RB, int DT>
__global__ void __launch_bounds__(64 * kAttnWaves, RB * D <= 256 ? 2 : 1)   // 256 registers: beyond, the compiler copies results in and out of accumulation registers
k_tree_attn(KvView c, AttnArgs a) {
    constexpr int NC = D / 64, QP = q_parts(DT), PP = p_parts(DT), ROWS = 16 * RB, LD = D + 4;
    // two tiles in registers, where there are so many
    constexpr bool DEEP = RB * D <= 128;
    __shared__ __attribute__((aligned(16))) float s_sc[kAttnWaves][64];
    __shared__ float s_o[kAttnWaves][ROWS * LD];
    __shared__ float s_m[kAttnWaves][ROWS], s_l[kAttnWaves][ROWS];
    __shared__ int s_ve[kAttnWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int g = lane >> 4, l16 = lane & 15;
    const int h = (int)blockIdx.y % c.heads, blk = (int)blockIdx.y / c.heads;
    const Share w = share_of(c, a, lane);
    const int rows = w.m * a.G, row0 = blk * ROWS;
    if (row0 >= rows) return;
    const int ctx = w.ctx, len = w.len, t1 = w.t1;
    int t = w.t0 + wave;

    // the pages of a tile's halves (-1: none), requested a tile ahead; loads from page 0 in place of none
    const int *table = c.table + (size_t)w.seq * c.max_pages;
    auto pages = [&](int tt) {
        const int p = 32 * tt, last = c.max_pages - 1;
        int x = table[min(p >> c.page_log2, last)], y = table[min((p + 16) >> c.page_log2, last)];
        x = p < len && (unsigned)x < (unsigned)c.n_pages ? x : -1;
        y = p + 16 < len && (unsigned)y < (unsigned)c.n_pages ? y : -1;
        return make_int2(x, y);
    };
    auto half_at = [&](int tt, int i, int2 pg) {
        return c.token0(max(i ? pg.y : pg.x, 0), h) + ((32 * tt + 16 * i) & (c.page() - 1));
    };
    auto load_k = [&](Tile<NC> &w, int tt, int2 pg) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const size_t at = half_at(tt, i, pg);
#pragma unroll
            for (int k = 0; k < NC; k++)
                w.x[i][k] = *reinterpret_cast<const u32x4_t *>(c.k + at * D + l16 * D + 64 * k + 16 * g);
        }
        const size_t at = g & 1 ? half_at(tt, 1, pg) : half_at(tt, 0, pg);
        w.scale = (lane < 32 ? c.ks : c.vs)[at + l16];
    };
    auto load_v = [&](Tile<NC> &w, int tt, int2 pg) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const size_t at = half_at(tt, i, pg);
#pragma unroll
            for (int k = 0; k < NC; k++)
                w.x[i][k] = *reinterpret_cast<const u32x4_t *>(c.v + at * D + 4 * g * D + (64 * k + 4 * l16) * 4);
        }
    };
    // Q: the waves share the row blocks out and leave their fragments in LDS; up to
    // 32 registers of them are then kept, more are read again tile by tile
    constexpr bool QREG = RB * NC * 2 * QP * 4 <= 32;
    f16x8_t *s_q = reinterpret_cast<f16x8_t *>(&s_o[0][0]);        // [RB][NC][2][QP][64], in lane order
    auto frag = [&](int rb, int k, int j, int n) { return ((((rb * NC + k) * 2 + j) * QP + n) << 6) + lane; };
    Rows<RB, NC, PP> R;
    QRow<NC, DT> q[RB];
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        const int r = min(row0 + 16 * rb + l16, rows - 1), node = r / a.G;
        if ((rb & (kAttnWaves - 1)) == wave) q[rb].load(a, w.r0, h, r, node, g);
        R.see[rb] = node_mask(a, w.r0, node);
    }
    Tile<NC> kt[DEEP ? 2 : 1], vt[DEEP ? 2 : 1];
    int2 pg = pages(t);
    if (t < t1) {
        load_k(kt[0], t, pg);
        load_v(vt[0], t, pg);
    }
    int2 pn = pages(t + kAttnWaves);
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        if ((rb & (kAttnWaves - 1)) != wave) continue;
        f16x8_t f[NC][2][QP];
        const float undo = q[rb].widen(a.scale, f);
        if (g == 0) s_m[0][16 * rb + l16] = undo;
#pragma unroll
        for (int k = 0; k < NC; k++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int n = 0; n < QP; n++) s_q[frag(rb, k, j, n)] = f[k][j][n];
    }
    __syncthreads();
    f16x8_t qf[QREG ? RB : 1][QREG ? NC : 1][2][QP];
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        R.qs[rb] = s_m[0][16 * rb + l16];
        if constexpr (QREG)
#pragma unroll
            for (int k = 0; k < NC; k++)
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int n = 0; n < QP; n++) qf[rb][k][j][n] = s_q[frag(rb, k, j, n)];
    }
    auto q_of = [&](int rb, int k, int j, int n, int at) {
        if constexpr (QREG) return qf[rb][k][j][n];
        else return s_q[frag(rb, k, j, n) + at];
    };

    R.clear();
    // One tile. DEEP: its successor is requested first, into registers of its
    // own; else the keys ahead of the softmax and the
    // values behind the second product, into the registers that have just become
    // free.
    auto step = [&](Tile<NC> &kn, Tile<NC> &kx, Tile<NC> &vn, Tile<NC> &vx) {
        const bool more = t + kAttnWaves < t1;
        if (DEEP && more) load_k(kx, t + kAttnWaves, pn);
        if (DEEP && more) load_v(vx, t + kAttnWaves, pn);
        s_sc[wave][lane] = kn.scale;
        int again = 0;                     // what the compiler cannot see through: Q is not to be kept in registers
        asm volatile("" : "+v"(again));
        f32x4_t s[RB][2];
#pragma unroll
        for (int rb = 0; rb < RB; rb++) s[rb][0] = s[rb][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int k = 0; k < NC; k++) {
                f16x8_t ka, kb;
                codes16<FMT>(kn.x[i][k], ka, kb);
#pragma unroll
                for (int n = 0; n < QP; n++) {
#pragma unroll
                    for (int rb = 0; rb < RB; rb++) s[rb][i] = mfma_f16(ka, q_of(rb, k, 0, n, again), s[rb][i]);
#pragma unroll
                    for (int rb = 0; rb < RB; rb++) s[rb][i] = mfma_f16(kb, q_of(rb, k, 1, n, again), s[rb][i]);
                }
            }
        wave_lds_fence();
        float vs[2][4];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const f32x4_t x = *reinterpret_cast<const f32x4_t *>(&s_sc[wave][16 * i + 4 * g]);
            const f32x4_t y = *reinterpret_cast<const f32x4_t *>(&s_sc[wave][32 + 16 * i + 4 * g]);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                vs[i][e] = y[e];
#pragma unroll
                for (int rb = 0; rb < RB; rb++) s[rb][i][e] *= x[e];
            }
        }
        wave_lds_fence();
        if (!DEEP && more) load_k(kx, t + kAttnWaves, pn);
        if (32 * t + 32 > ctx || (pg.x | pg.y) < 0) {
            const int j0[2] = {32 * t + 4 * g, 32 * t + 16 + 4 * g};
            const int n4[2] = {pg.x < 0 ? 0 : min(max(len - j0[0], 0), 4), pg.y < 0 ? 0 : min(max(len - j0[1], 0), 4)};
            const int node0[2] = {j0[0] - ctx, j0[1] - ctx};
            R.hide(s, vs, n4, node0);
            if constexpr (FMT == QFM_KV_E4M3) {
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int k = 0; k < NC; k++)
#pragma unroll
                        for (int q = 0; q < 4; q++) vn.x[i][k][q] &= token_bytes(n4[i]);
            }
        }
        f16x8_t pf[RB][PP];
        R.step(s, vs, pf);
        // results
#pragma unroll
        for (int k = 0; k < NC; k++) {
            f16x8_t a0, b0, a1, b1;
            codes16<FMT>(vn.x[0][k], a0, b0);
            codes16<FMT>(vn.x[1][k], a1, b1);
            const f16x8_t vf[4] = {__builtin_shufflevector(a0, a1, 0, 1, 2, 3, 8, 9, 10, 11),
                                   __builtin_shufflevector(a0, a1, 4, 5, 6, 7, 12, 13, 14, 15),
                                   __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 8, 9, 10, 11),
                                   __builtin_shufflevector(b0, b1, 4, 5, 6, 7, 12, 13, 14, 15)};
#pragma unroll
            for (int q = 0; q < 4; q++)
#pragma unroll
                for (int rb = 0; rb < RB; rb++)
#pragma unroll
                    for (int n = 0; n < PP; n++) R.o[rb][k][q] = mfma_f16(vf[q], pf[rb][n], R.o[rb][k][q]);
        }
        if (!DEEP && more) load_v(vx, t + kAttnWaves, pn);
        t += kAttnWaves;
        pg = pn;
        pn = pages(t + kAttnWaves);
    };
    while (t < t1) {
        step(kt[0], kt[DEEP], vt[0], vt[DEEP]);
        if constexpr (DEEP) {
            if (t >= t1) break;
            step(kt[1], kt[0], vt[1], vt[0]);
        }
    }

    put_parts(a, w);
    // join the waves
    __syncthreads();                       // Q has been read
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        R.l[rb] = sum_over_g(R.l[rb]);
        if (g == 0) {
            s_m[wave][16 * rb + l16] = R.m[rb];
            s_l[wave][16 * rb + l16] = R.l[rb];
        }
    }
    if (lane == 0) s_ve[wave] = R.ve;
    __syncthreads();
    int vn = s_ve[0];
#pragma unroll
    for (int w = 1; w < kAttnWaves; w++) vn = max(vn, s_ve[w]);
    const float vf = pow2_ratio(R.ve - vn);
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        float mn = s_m[0][16 * rb + l16];
#pragma unroll
        for (int w = 1; w < kAttnWaves; w++) mn = fmaxf(mn, s_m[w][16 * rb + l16]);
        const float f = __builtin_amdgcn_exp2f(R.m[rb] - mn) * vf;
#pragma unroll
        for (int k = 0; k < NC; k++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                *reinterpret_cast<float4 *>(&s_o[wave][(16 * rb + l16) * LD + 64 * k + 16 * g + 4 * i]) =
                    make_float4(R.o[rb][k][0][i] * f, R.o[rb][k][1][i] * f, R.o[rb][k][2][i] * f, R.o[rb][k][3][i] * f);
    }
    __syncthreads();
    const float back = exp2i(vn - 6);
    const int heads = c.heads * a.G;
    for (int e = threadIdx.x; e < ROWS * (D / 4); e += 64 * kAttnWaves) {
        const int r = e / (D / 4), d = (e - r * (D / 4)) * 4;
        if (row0 + r >= rows) break;
        float mn = s_m[0][r], sum = 0.0f;
#pragma unroll
        for (int w = 1; w < kAttnWaves; w++) mn = fmaxf(mn, s_m[w][r]);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kAttnWaves; w++) {
            const float4 y = *reinterpret_cast<const float4 *>(&s_o[w][r * LD + d]);
            x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
            sum += s_l[w][r] * exp2f(s_m[w][r] - mn);
        }
        const float inv = sum == 0.0f ? 0.0f : back / sum;
        x.x *= inv; x.y *= inv; x.z *= inv; x.w *= inv;
        const int node = (row0 + r) / a.G, head = h * a.G + (row0 + r) - node * a.G;
        if (w.n == 1) {
            store4<DT>(a.out, (w.r0 + node) * a.ors + head * a.ohs + d, x);
        } else {
            const size_t at = (size_t)(w.row + node) * heads + head;
            *reinterpret_cast<float4 *>(a.po + at * D + d) = x;
            if (d == 0) a.pml[at] = make_float2(mn, sum);
        }
    }
}

// The same for many rows of a key/value head: eight waves of 16 RB rows each,
// which take every tile together. It is widened to fp16 once, by all waves, and laid into LDS in the order
// of the MFMA operands (16-byte reads and writes, no two lanes on a bank); each
// step's tiles are requested a step ahead of being widened and widened a step
// ahead of their use, one barrier a step.
constexpr int kWideWaves = 8;

template <int FMT, int D, int RB, int DT>
__global__ void __launch_bounds__(64 * kWideWaves)
k_tree_wide(KvView c, AttnArgs a) {
    constexpr int NC = D / 64, QP = q_parts(DT), PP = p_parts(DT), ROWS = 16 * RB * kWideWaves;
    constexpr int NF = 8 * NC;                              // fragments a tile: 4 NC of K, then 4 NC of V
    constexpr int UNITS = 4 * NC, UN = (UNITS + kWideWaves - 1) / kWideWaves, LJ = 68;
    constexpr int TILES = 2 * NF * 64 * 16, JOIN = kWideWaves * 16 * LJ * 4;
    __shared__ __attribute__((aligned(16))) uint8_t s_buf[TILES > JOIN ? TILES : JOIN];
    __shared__ float s_sc[2][64];                           // 32 key scales, 32 value scales
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int g = lane >> 4, l16 = lane & 15;
    const int h = (int)blockIdx.y % c.heads, blk = (int)blockIdx.y / c.heads;
    const Share w = share_of(c, a, lane);
    const int rows = w.m * a.G, row0 = blk * ROWS;
    if (row0 >= rows) return;
    const int ctx = w.ctx, len = w.len, t0 = w.t0, t1 = w.t1;
    const int lim = min(len, 32 * t1);                      // tokens from here on are no keys of this workgroup
    const bool live = row0 + 16 * RB * wave < rows;           // this wave has rows

    const int *table = c.table + (size_t)w.seq * c.max_pages;
    auto pages = [&](int tt) {
        const int p = 32 * tt, last = c.max_pages - 1;
        int x = table[min(p >> c.page_log2, last)], y = table[min((p + 16) >> c.page_log2, last)];
        x = p < lim && (unsigned)x < (unsigned)c.n_pages ? x : -1;
        y = p + 16 < lim && (unsigned)y < (unsigned)c.n_pages ? y : -1;
        return make_int2(x, y);
    };
    // token index of half i of tile tt, on page 0 where there is none
    auto half_at = [&](int tt, int i, int2 pg) {
        return c.token0(max(i ? pg.y : pg.x, 0), h) + ((32 * tt + 16 * i) & (c.page() - 1));
    };
    u32x4_t raw[UN];
    float raw_sc;
    auto request = [&](int tt, int2 pg) {
#pragma unroll
        for (int n = 0; n < UN; n++) {
            const int r = wave + kWideWaves * n, i = (r % (2 * NC)) / NC, k = r % NC;
            if (r >= UNITS) break;
            const size_t at = half_at(tt, i, pg);
            const uint8_t *src = r < 2 * NC ? c.k + at * D + l16 * D + 64 * k + 16 * g
                                            : c.v + at * D + 4 * g * D + (64 * k + 4 * l16) * 4;
            raw[n] = *reinterpret_cast<const u32x4_t *>(src);
        }
        if (wave == 0) {
            const size_t at = half_at(tt, (lane >> 4) & 1, pg) + l16;
            raw_sc = (lane < 32 ? c.ks : c.vs)[at];
        }
    };
    auto widen = [&](int tt, int2 pg) {
        uint8_t *buf = s_buf + (tt & 1) * (TILES / 2);
#pragma unroll
        for (int n = 0; n < UN; n++) {
            const int r = wave + kWideWaves * n, i = (r % (2 * NC)) / NC, k = r % NC;
            if (r >= UNITS) break;
            uint8_t *dst = buf + lane * 16;
            f16x8_t x, y;
            if (r < 2 * NC) {
                codes16<FMT>(raw[n], x, y);
                *reinterpret_cast<f16x8_t *>(dst + ((i * NC + k) * 2) * 1024) = x;
                *reinterpret_cast<f16x8_t *>(dst + ((i * NC + k) * 2 + 1) * 1024) = y;
            } else {
                if constexpr (FMT == QFM_KV_E4M3) {
                    const int j0 = 32 * tt + 16 * i + 4 * g;
                    const uint32_t keep = token_bytes((i ? pg.y : pg.x) < 0 ? 0 : min(max(lim - j0, 0), 4));
#pragma unroll
                    for (int q = 0; q < 4; q++) raw[n][q] &= keep;
                }
                codes16<FMT>(raw[n], x, y);
                const u32x4_t p = __builtin_bit_cast(u32x4_t, x), q = __builtin_bit_cast(u32x4_t, y);
                dst += (4 * NC + 4 * k) * 1024 + 8 * i;
                *reinterpret_cast<u32x2_t *>(dst) = u32x2_t{p[0], p[1]};
                *reinterpret_cast<u32x2_t *>(dst + 1024) = u32x2_t{p[2], p[3]};
                *reinterpret_cast<u32x2_t *>(dst + 2 * 1024) = u32x2_t{q[0], q[1]};
                *reinterpret_cast<u32x2_t *>(dst + 3 * 1024) = u32x2_t{q[2], q[3]};
            }
        }
        if (wave == 0) s_sc[tt & 1][lane] = raw_sc;
    };
    Rows<RB, NC, PP> R;
    QRow<NC, DT> q[RB];
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        const int r = min(row0 + 16 * (RB * wave + rb) + l16, rows - 1), node = r / a.G;
        q[rb].load(a, w.r0, h, r, node, g);
        R.see[rb] = node_mask(a, w.r0, node);
    }
    int2 pc = pages(t0), pn = pages(t0 + 1), pf2 = pages(t0 + 2);   // of this tile and the next two
    if (t0 < t1) request(t0, pc);
    f16x8_t qf[RB][NC][2][QP];
#pragma unroll
    for (int rb = 0; rb < RB; rb++) R.qs[rb] = q[rb].widen(a.scale, qf[rb]);
    R.clear();
    if (t0 < t1) widen(t0, pc);
    if (t0 + 1 < t1) request(t0 + 1, pn);
    // the next tile: half of the waves widen their part of it before this tile's
    // products and half behind them, so that the two waves of a SIMD are not both at
    // their conversions and both at their MFMAs (61-node trees 75.2 -> 73.2 us)
    auto ahead = [&](int t) {
        if (t + 1 < t1) widen(t + 1, pn);
        if (t + 2 < t1) request(t + 2, pf2);
    };
    __syncthreads();
    for (int t = t0; t < t1; t++) {
        if (wave < kWideWaves / 2) ahead(t);
        if (live) {
            const uint8_t *buf = s_buf + (t & 1) * (TILES / 2) + lane * 16;
            f32x4_t s[RB][2];
#pragma unroll
            for (int rb = 0; rb < RB; rb++) s[rb][0] = s[rb][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int k = 0; k < NC; k++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const f16x8_t kf = *reinterpret_cast<const f16x8_t *>(buf + ((i * NC + k) * 2 + j) * 1024);
#pragma unroll
                        for (int n = 0; n < QP; n++)
#pragma unroll
                            for (int rb = 0; rb < RB; rb++) s[rb][i] = mfma_f16(kf, qf[rb][k][j][n], s[rb][i]);
                    }
            float vs[2][4];
            const float *sc = s_sc[t & 1];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float4 x = *reinterpret_cast<const float4 *>(sc + 16 * i + 4 * g);
                const float4 y = *reinterpret_cast<const float4 *>(sc + 32 + 16 * i + 4 * g);
                const float ks[4] = {x.x, x.y, x.z, x.w};
                vs[i][0] = y.x; vs[i][1] = y.y; vs[i][2] = y.z; vs[i][3] = y.w;
#pragma unroll
                for (int rb = 0; rb < RB; rb++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[rb][i][e] *= ks[e];
            }
            if (32 * t + 32 > min(ctx, lim) || (pc.x | pc.y) < 0) {
                const int j0[2] = {32 * t + 4 * g, 32 * t + 16 + 4 * g};
                const int n4[2] = {pc.x < 0 ? 0 : min(max(lim - j0[0], 0), 4), pc.y < 0 ? 0 : min(max(lim - j0[1], 0), 4)};
                const int node0[2] = {j0[0] - ctx, j0[1] - ctx};
                R.hide(s, vs, n4, node0);
            }
            f16x8_t pf[RB][PP];
            R.step(s, vs, pf);
#pragma unroll
            for (int k = 0; k < NC; k++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const f16x8_t vf = *reinterpret_cast<const f16x8_t *>(buf + (4 * NC + 4 * k + q) * 1024);
#pragma unroll
                    for (int n = 0; n < PP; n++)
#pragma unroll
                        for (int rb = 0; rb < RB; rb++) R.o[rb][k][q] = mfma_f16(vf, pf[rb][n], R.o[rb][k][q]);
                }
        }
        if (wave >= kWideWaves / 2) ahead(t);
        pc = pn;
        pn = pf2;
        pf2 = pages(t + 3);
        __syncthreads();
    }

    put_parts(a, w);
    // 4 channels of a row, to the results or the workspace; 64 channels of a row
    // a turn, brought side by side through LDS
    const int heads = c.heads * a.G;
    struct Place { long t; int head; size_t at; };
    auto place = [&](int r) {
        const int node = r / a.G, head = h * a.G + r - node * a.G;
        return Place{w.r0 + node, head, (size_t)(w.row + node) * heads + head};
    };
    auto put = [&](const Place &p, int d, float4 x) {
        if (w.n == 1) store4<DT>(a.out, p.t * a.ors + p.head * a.ohs + d, x);
        else *reinterpret_cast<float4 *>(a.po + p.at * D + d) = x;
    };
    float *s_j = reinterpret_cast<float *>(s_buf) + wave * (16 * LJ);
    if (!live) return;
#pragma unroll
    for (int rb = 0; rb < RB; rb++) R.l[rb] = sum_over_g(R.l[rb]);
    const float back = exp2i(R.ve - 6);
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        const int r0 = row0 + 16 * (RB * wave + rb);
        const float inv = R.l[rb] == 0.0f ? 0.0f : back / R.l[rb];
        if (w.n > 1 && g == 0 && r0 + l16 < rows) a.pml[place(r0 + l16).at] = make_float2(R.m[rb], R.l[rb]);
        Place p[4];
#pragma unroll
        for (int n = 0; n < 4; n++) p[n] = place(min(r0 + 4 * n + g, rows - 1));
#pragma unroll
        for (int k = 0; k < NC; k++) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                *reinterpret_cast<float4 *>(&s_j[l16 * LJ + 16 * g + 4 * i]) =
                    make_float4(R.o[rb][k][0][i] * inv, R.o[rb][k][1][i] * inv, R.o[rb][k][2][i] * inv, R.o[rb][k][3][i] * inv);
            wave_lds_fence();
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const float4 x = *reinterpret_cast<const float4 *>(&s_j[(4 * n + g) * LJ + 4 * l16]);
                if (r0 + 4 * n + g < rows) put(p[n], 64 * k + 4 * l16, x);
            }
            wave_lds_fence();
        }
    }
}

// out(t, h) = sum_s w_s o_s / sum_s w_s, w_s = sum_s 2^(max_s - max): one block 64
// channels of a row and head, a thread 4 of them of every 16th split, so that all
// splits are requested at once (131072 tokens in 128 splits, 48 rows and heads of
// 256 channels: 4.6 us; a block a row and head, 11.6).
template <int D, int DT, bool DEALT>
__global__ void __launch_bounds__(256)
k_tree_join(AttnArgs a, int heads) {
    constexpr int TD = 16, NG = 256 / TD, U = kMaxSplits / NG;
    __shared__ float s_w[kMaxSplits], s_part[NG][4 * TD];
    const int2 sr = seq_rows(a.row_start, (int)blockIdx.z, a.T, a.max_nodes);
    const int2 parts = parts_of<DEALT>(a, (int)blockIdx.z, sr);
    if ((int)blockIdx.y >= sr.y || !parts.x) return;
    const int head = (int)blockIdx.x / (D / 64), dl = (int)threadIdx.x % TD * 4, d = (int)blockIdx.x % (D / 64) * 64 + dl, grp = (int)threadIdx.x / TD, lane = threadIdx.x & 63;
    const long t = sr.x + (int)blockIdx.y;
    const size_t row = (size_t)(parts.y + (int)blockIdx.y) * heads + head, step = (size_t)sr.y * heads;
    // every wave finds the weights, two splits a lane
    float2 ml[2];
#pragma unroll
    for (int i = 0; i < 2; i++) ml[i] = lane + 64 * i < parts.x ? a.pml[(lane + 64 * i) * step + row] : make_float2(kNoMax, 0.0f);
    float4 y[U];
#pragma unroll
    for (int i = 0; i < U; i++)
        if (grp + NG * i < parts.x) y[i] = *reinterpret_cast<const float4 *>(a.po + ((grp + NG * i) * step + row) * D + d);
    float mn = fmaxf(ml[0].x, ml[1].x);
#pragma unroll
    for (int o = 32; o; o >>= 1) mn = fmaxf(mn, __shfl_xor(mn, o));
    const float w0 = ml[0].y * __builtin_amdgcn_exp2f(ml[0].x - mn), w1 = ml[1].y * __builtin_amdgcn_exp2f(ml[1].x - mn);
    float sum = w0 + w1;
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (threadIdx.x < 64) {
        s_w[lane] = w0;
        s_w[lane + 64] = w1;
    }
    __syncthreads();
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < U; i++) {
        const float w = s_w[grp + NG * i];
        if (w == 0.0f) continue;                            // no such split, or one without keys, which wrote no result
        x.x = fmaf(w, y[i].x, x.x); x.y = fmaf(w, y[i].y, x.y); x.z = fmaf(w, y[i].z, x.z); x.w = fmaf(w, y[i].w, x.w);
    }
    *reinterpret_cast<float4 *>(&s_part[grp][dl]) = x;
    __syncthreads();
    if (grp) return;
#pragma unroll
    for (int i = 1; i < NG; i++) {
        const float4 z = *reinterpret_cast<const float4 *>(&s_part[i][dl]);
        x.x += z.x; x.y += z.y; x.z += z.z; x.w += z.w;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    store4<DT>(a.out, t * a.ors + head * a.ohs + d, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
}

// The same where the splits are few (kFewSplits on average): a thread 4 channels
// of a row and head over all splits, kFewSplits at a time, 1024 / D rows and heads
// a block.
constexpr int kFewSplits = 8;
template <int D, int DT, bool DEALT>
__global__ void __launch_bounds__(256)
k_tree_join_few(AttnArgs a, int heads) {
    constexpr int TD = D / 4;
    const int2 sr = seq_rows(a.row_start, (int)blockIdx.z, a.T, a.max_nodes);
    const int2 parts = parts_of<DEALT>(a, (int)blockIdx.z, sr);
    const int i = (int)blockIdx.x * (256 / TD) + (int)threadIdx.x / TD, node = i / heads, head = i - node * heads;
    if (node >= sr.y || !parts.x) return;
    const int d = (int)threadIdx.x % TD * 4;
    const size_t row = (size_t)(parts.y + node) * heads + head, step = (size_t)sr.y * heads;
    float m = kNoMax, sum = 0.0f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    const auto add = [&](int s0, bool more) {
        float2 ml[kFewSplits];
        float4 y[kFewSplits];
#pragma unroll
        for (int s = 0; s < kFewSplits; s++) {
            ml[s] = make_float2(kNoMax, 0.0f);
            y[s] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (s0 + s < parts.x) {
                ml[s] = a.pml[(s0 + s) * step + row];
                y[s] = *reinterpret_cast<const float4 *>(a.po + ((s0 + s) * step + row) * D + d);
            }
        }
        float mn = m;
#pragma unroll
        for (int s = 0; s < kFewSplits; s++) mn = fmaxf(mn, ml[s].x);
        if (more) {
            const float old = __builtin_amdgcn_exp2f(m - mn);
            sum *= old;
            x.x *= old; x.y *= old; x.z *= old; x.w *= old;
        }
        m = mn;
#pragma unroll
        for (int s = 0; s < kFewSplits; s++) {
            const float w = ml[s].y * __builtin_amdgcn_exp2f(ml[s].x - mn);
            sum += w;
            // a split without keys wrote no result
            const bool none = w == 0.0f;
            x.x = none ? x.x : fmaf(w, y[s].x, x.x); x.y = none ? x.y : fmaf(w, y[s].y, x.y);
            x.z = none ? x.z : fmaf(w, y[s].z, x.z); x.w = none ? x.w : fmaf(w, y[s].w, x.w);
        }
    };
    add(0, false);
    if constexpr (DEALT)
        for (int s0 = kFewSplits; s0 < parts.x; s0 += kFewSplits) add(s0, true);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    store4<DT>(a.out, (long)(sr.x + node) * a.ors + head * a.ohs + d, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
}

// How a call is laid out: 16 rb rows a wave, in k_tree_attn or k_tree_wide, and
// the splits of a sequence's keys.
// block: rows a workgroup; slots: workgroups along the keys for a head's block of rows
struct AttnPlan { int rb, block, splits, slots; bool wide; };
// what a wave holds within 256 registers
constexpr int few_blocks(int D, bool f32) { return D == 256 && f32 ? 1 : 2; }
constexpr int wide_blocks(int D, bool f32) { return D == 64 || (D == 128 && !f32) ? 2 : 1; }
// workgroups that a CU holds at once, by their registers
constexpr int few_resident(int D, int rb) { return rb == 1 ? (D == 64 ? 3 : 2) : D == 256 ? 1 : 2; }

// Microseconds that a layout takes, as fitted to 130 shapes (contexts 1 to 131071,
// 1 to 64 nodes, every head layout and type) in up to 40 layouts each: rounds of
// resident workgroups (fractions of one for the most part: sequences differ in
// length), each a prologue and its tiles; a step is as long as its loads' latency
// or as what the CU's workgroups compute together; a join and its partial results.
// What it picks takes 1.2% more than the best layout on average; one round of
// resident workgroups with the widest rows took 21% more. Each form is there for
// what the others lose without it: 16 rows a wave 16%, 32 rows 3%, k_tree_wide 3%
// (61-node trees of five users: 84 us, 75 with it, before the keys were dealt out).
static float attn_cost(const AttnPlan &p, int D, int dtype, long groups, int rows, long tiles) {
    const float d = D / 128.0f, each = p.wide ? 1 : kAttnWaves;
    const bool f32 = dtype == QFM_DT_F32, f16 = dtype == QFM_DT_F16;
    const int resident = p.wide ? 1 : few_resident(D, p.rb);
    const long all = groups * p.splits, whole = (all + 256 * resident - 1) / (256 * resident);
    const float rounds = 0.24f * whole + 0.76f * std::max(1.0f, all / (256.0f * resident));
    const float occ = (float)std::min<long>(resident, (all + 255) / 256);
    const float steps = (float)(long)((tiles + p.splits * (long)each - 1) / (p.splits * (long)each));
    const float busy = occ * d * (p.rb == 1 ? 0.66f : 0.83f) * (f32 ? 0.89f : f16 ? 0.69f : 1.0f);
    const float wait = (0.37f + 0.55f * d) * (p.rb * D > 128 ? 1.14f : 1.0f);
    const float step = p.wide ? 0.15f + 0.43f * d * p.rb * (f32 ? 1.9f : f16 ? 1.19f : 1.0f) : std::max(wait, busy);
    float us = 3.9f + rounds * ((p.wide ? 2.2f : 1.1f) + 1.1f * d * p.rb + steps * step);
    if (p.splits > 1) us += 3.1f + (p.splits > kFewSplits ? 1.4f : 0.0f) + (float)all * std::min(p.block, rows) * D * 8 / 5.4e6f;
    return us;
}

// whether the keys of so many sequences may be dealt out by length
static bool dealt_seqs(int n_seq) { return n_seq > 1 && n_seq <= kDealSeqs; }

// What is left of the CUs, all of them or each a further time, is dealt out, too.
static void attn_slots(AttnPlan &p, int kv_heads, int n_seq, int rows) {
    p.slots = n_seq * p.splits;
    if (p.splits == 1 || !dealt_seqs(n_seq)) return;
    const long groups = (long)kv_heads * ((rows + p.block - 1) / p.block);
    const long fill = (groups * p.slots + 255) / 256 * 256 / groups;
    p.slots = (int)std::min<long>(std::max<long>(p.slots, fill), (long)n_seq * (p.splits + 1) - 1);
}

static AttnPlan attn_plan(int D, int kv_heads, int n_seq, int q_heads, int max_nodes, int max_ctx, int dtype) {
    static const int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, kMaxSplits};
    const int rows = max_nodes * (q_heads / kv_heads);
    const long tiles = ((long)max_ctx + max_nodes + 31) / 32;
    const bool f32 = dtype == QFM_DT_F32;
    AttnPlan best{};
    float least = 0.0f;
    for (int form = 0; form < 3; form++) {                  // rb 1, rb 2, wide
        AttnPlan p{};
        p.wide = form == 2;
        p.rb = p.wide ? wide_blocks(D, f32) : form + 1;
        if (form == 1 && few_blocks(D, f32) < 2) continue;
        if (form && rows <= 16) break;
        p.block = 16 * p.rb * (p.wide ? kWideWaves : 1);
        const long groups = (long)n_seq * kv_heads * ((rows + p.block - 1) / p.block);
        for (int n : kSplits) {
            if (n > 1 && n > tiles) break;
            p.splits = n;
            const float us = attn_cost(p, D, dtype, groups, rows, tiles);
            if (!best.rb || us < least) {
                best = p;
                least = us;
            }
        }
    }
    // half the work may be one sequence's: a second workgroup for it where a join is little beside that
    if (best.splits == 1 && dealt_seqs(n_seq) && least > 100.0f && tiles > 1) best.splits = 2;
    attn_slots(best, kv_heads, n_seq, rows);
    return best;
}

static int attn_shape(const qfm_kv_cache *c, int n_seq, int T, int q_heads, int max_nodes, int max_ctx) {
    if (!c || (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) || c->kv_heads < 1 || c->kv_heads > 1024 ||
        n_seq < 1 || n_seq > 65535 || T < 0 || T > 1 << 22 || q_heads < 1 || q_heads > 4096 || q_heads % c->kv_heads ||
        max_nodes < 1 || max_nodes > 64 || max_ctx < 0)
        return -1;
    return (long)c->kv_heads * ((max_nodes * (q_heads / c->kv_heads) + 15) / 16) > 65535 ? -1 : 0;
}

// rows of partial results: every split of a sequence has all its rows
static long attn_rows(const AttnPlan &p, int n_seq, int T, int max_nodes) {
    if (p.splits == 1) return 0;
    const long even = (long)p.splits * T;
    return dealt_seqs(n_seq) ? std::max(even, std::min((long)p.slots * max_nodes, std::min<long>(p.slots, kMaxSplits) * T)) : even;
}
static size_t attn_ws(const qfm_kv_cache *c, long rows, int n_seq, int q_heads) {
    return rows ? (size_t)rows * q_heads * (c->head_dim + 2) * 4 + (size_t)n_seq * 8 : 0;
}

template <int FMT, int D, int DT>
static void attn_launch(const KvView &v, const AttnArgs &a, const AttnPlan &p, dim3 g, hipStream_t s) {
    constexpr bool F32 = DT == QFM_DT_F32;
    constexpr int RB = wide_blocks(D, F32);
    const dim3 b(64 * kAttnWaves), bw(64 * kWideWaves);
    if (p.wide) hipLaunchKernelGGL((k_tree_wide<FMT, D, RB, DT>), g, bw, 0, s, v, a);
    else if (p.rb == 1) hipLaunchKernelGGL((k_tree_attn<FMT, D, 1, DT>), g, b, 0, s, v, a);
    else if constexpr (few_blocks(D, F32) == 2) hipLaunchKernelGGL((k_tree_attn<FMT, D, 2, DT>), g, b, 0, s, v, a);
}
template <int D, int DT, bool DEALT>
static void attn_join(const AttnArgs &a, int heads, int n_seq, hipStream_t s) {
    if (a.splits <= kFewSplits) {
        const dim3 gj((unsigned)((heads * a.max_nodes + 1024 / D - 1) / (1024 / D)), 1, (unsigned)n_seq);
        hipLaunchKernelGGL((k_tree_join_few<D, DT, DEALT>), gj, dim3(256), 0, s, a, heads);
    } else {
        const dim3 gj((unsigned)(heads * (D / 64)), (unsigned)a.max_nodes, (unsigned)n_seq);
        hipLaunchKernelGGL((k_tree_join<D, DT, DEALT>), gj, dim3(256), 0, s, a, heads);
    }
}
template <int D, int DT>
static void attn_launch(const KvView &v, const AttnArgs &a, const AttnPlan &p, int fmt, int n_seq, hipStream_t s) {
    const int rows = a.max_nodes * a.G, heads = v.heads * a.G;
    const dim3 g((unsigned)(a.dealt ? p.slots : p.splits), (unsigned)(v.heads * ((rows + p.block - 1) / p.block)),
                 a.dealt ? 1u : (unsigned)n_seq);
    if (fmt == QFM_KV_INT8) attn_launch<QFM_KV_INT8, D, DT>(v, a, p, g, s);
    else attn_launch<QFM_KV_E4M3, D, DT>(v, a, p, g, s);
    if (a.splits == 1) return;
    if (a.dealt) attn_join<D, DT, true>(a, heads, n_seq, s);
    else attn_join<D, DT, false>(a, heads, n_seq, s);
}
template <int D>
static void attn_launch(const KvView &v, const AttnArgs &a, const AttnPlan &p, int dtype, int fmt, int n_seq, hipStream_t s) {
    if (dtype == QFM_DT_F32) attn_launch<D, QFM_DT_F32>(v, a, p, fmt, n_seq, s);
    else if (dtype == QFM_DT_BF16) attn_launch<D, QFM_DT_BF16>(v, a, p, fmt, n_seq, s);
    else attn_launch<D, QFM_DT_F16>(v, a, p, fmt, n_seq, s);
}

}  // namespace qfm

using namespace qfm;

extern "C" {

size_t qfm_tree_attn_ws_bytes(const qfm_kv_cache *c, int n_seq, int T, int q_heads, int max_nodes, int max_ctx) {
    if (attn_shape(c, n_seq, T, q_heads, max_nodes, max_ctx)) return 0;
    long rows = 0;
    for (int dtype : {QFM_DT_F32, QFM_DT_BF16, QFM_DT_F16})
        rows = std::max(rows, attn_rows(attn_plan(c->head_dim, c->kv_heads, n_seq, q_heads, max_nodes, max_ctx, dtype), n_seq, T, max_nodes));
    return attn_ws(c, rows, n_seq, q_heads);
}

int qfm_tree_attn(const qfm_kv_cache *c, const qfm_kv_seqs *sq, const void *q, void *out, int dtype, int q_heads,
                  long q_row_stride, long q_head_stride, long out_row_stride, long out_head_stride, const int *row_start,
                  const int *ctx, const uint64_t *tree, int T, int max_nodes, int max_ctx, float scale, void *ws,
                  size_t ws_bytes, hipStream_t s) {
    const char *who = "qfm_tree_attn";
    KvView v;
    if (kv_view(c, sq, &v, who)) return -1;
    if (attn_shape(c, sq->n_seq, T, q_heads, max_nodes, max_ctx)) {
        set_error(-1, "%s: T = %d, %d query heads over %d, %d nodes (1..64), max_ctx %d", who, T, q_heads, c->kv_heads,
                  max_nodes, max_ctx);
        return -1;
    }
    if (dtype != QFM_DT_F32 && dtype != QFM_DT_BF16 && dtype != QFM_DT_F16) {
        set_error(-1, "%s: element type %d", who, dtype);
        return -1;
    }
    if (!q || !out || !row_start || !ctx) { set_error(-1, "%s: null argument", who); return -1; }
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15 || reinterpret_cast<uintptr_t>(tree) & 7) {
        set_error(-1, "%s: q and out are 16-byte aligned, the masks 8", who);
        return -1;
    }
    if (q_row_stride < 0 || q_head_stride < 0 || q_row_stride % 8 || q_head_stride % 8 || out_row_stride % 8 ||
        out_head_stride % 8 || out_row_stride < c->head_dim || out_head_stride < c->head_dim) {
        set_error(-1, "%s: strides %ld %ld %ld %ld (multiples of 8, those of out at least %d)", who, q_row_stride,
                  q_head_stride, out_row_stride, out_head_stride, c->head_dim);
        return -1;
    }
    if (!(scale > 0.0f) || !(scale < 3.4e38f)) { set_error(-1, "%s: scale %g", who, (double)scale); return -1; }
    const int D = c->head_dim, G = q_heads / c->kv_heads;
    const AttnPlan p = attn_plan(D, c->kv_heads, sq->n_seq, q_heads, max_nodes, max_ctx, dtype);
    const long rows = attn_rows(p, sq->n_seq, T, max_nodes);
    const size_t need = attn_ws(c, rows, sq->n_seq, q_heads);
    if (need && (!ws || ws_bytes < need || reinterpret_cast<uintptr_t>(ws) & 15)) {
        set_error(-1, "%s: workspace of %zu bytes (16-byte aligned), %zu needed", who, ws ? ws_bytes : (size_t)0, need);
        return -1;
    }
    if (T == 0) return 0;
    AttnArgs a{};
    a.q = static_cast<const uint8_t *>(q);
    a.out = static_cast<uint8_t *>(out);
    a.G = G; a.T = T; a.max_nodes = max_nodes; a.splits = p.splits;
    a.qrs = q_row_stride; a.qhs = q_head_stride; a.ors = out_row_stride; a.ohs = out_head_stride;
    a.row_start = row_start; a.ctx = ctx; a.tree = tree; a.scale = scale;
    if (p.splits > 1) {
        // (the sum of all tiles stays an int)
        const long most = (std::min((long)sq->max_pages * c->page, kMaxTokens) >> 5) + 1;
        a.dealt = dealt_seqs(sq->n_seq) && most * sq->n_seq < 1l << 31;
        a.rows = (int)rows;
        a.po = static_cast<float *>(ws);
        a.pml = reinterpret_cast<float2 *>(a.po + (size_t)rows * q_heads * D);
        a.parts = reinterpret_cast<int2 *>(a.pml + (size_t)rows * q_heads);
    }
    if (D == 64) attn_launch<64>(v, a, p, dtype, c->fmt, sq->n_seq, s);
    else if (D == 128) attn_launch<128>(v, a, p, dtype, c->fmt, sq->n_seq, s);
    else attn_launch<256>(v, a, p, dtype, c->fmt, sq->n_seq, s);
    return check_launch(who) ? -3 : 0;
}

}  // extern "C"

// qfm_kv.hip -- the quantised key/value cache: rows in (qfm_kv_write) and rows
// back (qfm_kv_read).
//
// A row of one head is D values with one scale: amax over the row, then one
// quotient a value. Both kernels are bound by bytes (2 or 4 in and 1 out a
// value, or the reverse: 8038 rows of 8 x 128 in 13.8 us written, 11.9 read,
// 50 MB at 3.6 and 4.2 TB/s) and, at a few rows, by the chain of dependent loads
// row -> sequence and position -> page (3.3 us alone; a call costs the host 4).
#include "qfm_kv.h"
#include "qfm_internal.h"

namespace qfm {

constexpr int kKvThreads = 256;

// v / s as IEEE division gives it. With r = 1 / s rounded correctly, q = v r and
// q + (v - q s) r, the residual exact by fma, round to the quotient itself (P.
// Markstein) while nothing underflows: three operations in place of the ten of
// a division, which bound the kernel (8038 rows of 8 x 128: 29.2 us with
// divisions and byte stores).
__device__ __forceinline__ float quotient(float v, float s, float r) {
    const float q = v * r;
    return fmaf(fmaf(-q, s, v), r, q);
}

// 4 codes as one word
template <int FMT>
__device__ __forceinline__ uint32_t kv_codes(float a, float b, float c, float d) {
    if constexpr (FMT == QFM_KV_INT8) {
        const auto code = [](float q) { return (uint32_t)(int)rintf(fminf(127.0f, fmaxf(-127.0f, q))); };
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(code(d), code(c), 0x0c0c0400u),
                                     __builtin_amdgcn_perm(code(b), code(a), 0x0c0c0400u), 0x05040100u);
    } else {
        const auto lim = [](float q) { return fminf(448.0f, fmaxf(-448.0f, q)); };
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(lim(a), lim(b), 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(lim(c), lim(d), w, true);
    }
}

// VL = D / 16 values of a row, widened to fp32 (p aligned to their size, to 16 bytes at most)
template <int DT, int VL>
__device__ __forceinline__ void load_row(const uint8_t *p, float (&v)[VL]) {
    if constexpr (VL == 4 && DT != QFM_DT_F32) {
        const uint2 w = *reinterpret_cast<const uint2 *>(p);
        const uint32_t d[2] = {w.x, w.y};
#pragma unroll
        for (int i = 0; i < 2; i++) {
            v[2 * i] = DT == QFM_DT_BF16 ? bf16_lo(d[i]) : (float)as_h2(d[i]).x;
            v[2 * i + 1] = DT == QFM_DT_BF16 ? bf16_hi(d[i]) : (float)as_h2(d[i]).y;
        }
    } else if constexpr (VL == 4) {
        const float4 a = *reinterpret_cast<const float4 *>(p);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
#pragma unroll
        for (int i = 0; i < VL / 8; i++) load8<DT>(p + i * 8 * (DT == QFM_DT_F32 ? 4 : 2), *reinterpret_cast<float(*)[8]>(&v[8 * i]));
    }
}

// codes (VL / 4 words) and scale of this lane's part of a row; LPR lanes a row
template <int FMT, int VL, int LPR>
__device__ __forceinline__ float quantise(const float (&v)[VL], uint32_t (&code)[VL / 4]) {
    constexpr float kInv = FMT == QFM_KV_INT8 ? 1.0f / 127.0f : 1.0f / 448.0f;
    // the largest magnitude as bits: NaN and infinity above every number
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < VL; i++) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
#pragma unroll
    for (int o = LPR / 2; o; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
    const bool fine = m < 0x7F800000u;
    float s = __uint_as_float(m) * kInv;
    if (s == 0.0f) s = 1.0f;
    float q[VL];
    if (__any(s < 0x1p-60f)) {             // where the residual may underflow
#pragma unroll
        for (int i = 0; i < VL; i++) q[i] = v[i] / s;
    } else {
        const float r = 1.0f / s;
#pragma unroll
        for (int i = 0; i < VL; i++) q[i] = quotient(v[i], s, r);
    }
#pragma unroll
    for (int i = 0; i < VL / 4; i++) {
        const uint32_t w = kv_codes<FMT>(q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]);
        code[i] = fine ? w : 0u;
    }
    return fine ? s : __uint_as_float(0x7FC00000u);
}

// Bytes c of the lanes j, j + 16, j + 32, j + 48 (rows 0..3) -> in lane 16 r + j
// the four rows' byte r: a 4 x 4 transpose in two exchanges.
__device__ __forceinline__ uint32_t transpose_rows(uint32_t x, int r) {
    const uint32_t y = (uint32_t)__shfl_xor((int)x, 16);
    // byte selectors: 0..3 of the second operand, 4..7 of the first
    const uint32_t z = r & 1 ? __builtin_amdgcn_perm(x, y, 0x07030501u) : __builtin_amdgcn_perm(y, x, 0x06020400u);
    const uint32_t w = (uint32_t)__shfl_xor((int)z, 32);
    return r & 2 ? __builtin_amdgcn_perm(z, w, 0x07060302u) : __builtin_amdgcn_perm(w, z, 0x05040100u);
}

// Few rows (up to kFewRows): what counts is the chain row -> place -> stores, so
// keys and values are rows of their own, 8 values a lane, every value code a byte
// store (8 rows of 2 x 256: 4.2 us a call, 5.4 in fours as below).
constexpr int kFewRows = 64;
template <int DT, int FMT, int D>
__global__ void __launch_bounds__(kKvThreads)
k_kv_write_few(KvView c, const uint8_t *__restrict__ k, const uint8_t *__restrict__ v, long rs, long hs,
               const int *__restrict__ seq, const int *__restrict__ pos, int T) {
    constexpr int LPR = D / 8, ES = DT == QFM_DT_F32 ? 4 : 2;
    const int u = ((int)blockIdx.x * kKvThreads + (int)threadIdx.x) / LPR, j = (int)threadIdx.x % LPR, kv = u & 1;
    const int t = (u >> 1) / c.heads, h = (u >> 1) - t * c.heads;
    if (t >= T) return;                                     // whole rows: LPR lanes leave together
    float x[8];
    load8<DT>((kv ? v : k) + (t * rs + h * hs + 8 * j) * ES, x);
    const int sq = seq[t], p = pos[t];
    const int page = (unsigned)sq < (unsigned)c.n_seq ? c.page_of(sq, p) : -1;
    const int tok = p & (c.page() - 1);
    uint32_t code[2];
    const float s = quantise<FMT, 8, LPR>(x, code);
    if (page < 0) return;
    const size_t at = c.token0(page, h);
    if (j == 0) (kv ? c.vs : c.ks)[at + tok] = s;
    if (kv) {
        uint8_t *o = c.v + (at + (tok & ~3)) * D + (8 * j) * 4 + (tok & 3);
#pragma unroll
        for (int q = 0; q < 8; q++) o[4 * q] = (uint8_t)(code[q / 4] >> (8 * (q % 4)));
    } else {
        *reinterpret_cast<uint2 *>(c.k + (at + tok) * D + 8 * j) = make_uint2(code[0], code[1]);
    }
}

// One wave takes 4 rows of a head, 16 lanes a row. Keys go as they are. Values
// lie four tokens to a word: where 4 rows in a row fill such a word (positions 4
// n .. 4 n + 3 of one sequence) the wave in whose rows the first one is takes
// those four and writes words; the other rows' values go byte by byte.
template <int DT, int FMT, int D>
__global__ void __launch_bounds__(kKvThreads)
k_kv_write(KvView c, const uint8_t *__restrict__ k, const uint8_t *__restrict__ v, long rs, long hs,
           const int *__restrict__ seq, const int *__restrict__ pos, int T) {
    constexpr int VL = D / 16, ES = DT == QFM_DT_F32 ? 4 : 2;
    const int lane = threadIdx.x & 63, j = lane & 15, r = lane >> 4;
    const long u = (long)blockIdx.x * (kKvThreads / 64) + (threadIdx.x >> 6);
    const int h = (int)(u % c.heads), b = (int)(u / c.heads) * 4;
    if (b >= T) return;
    const uint8_t *kp = k + (h * hs + VL * j) * ES, *vp = v + (h * hs + VL * j) * ES;
    const int t = min(b + r, T - 1);
    float x[VL], y[VL];
    load_row<DT, VL>(kp + (long)t * rs * ES, x);
    // rows b - 3 .. b + 12: which continue their predecessor's sequence
    const int ti = b - 3 + j;
    const int ts = ti >= 0 && ti < T ? seq[ti] : -1, tp = ti >= 0 && ti < T ? pos[ti] : -1;
    const int bs = __shfl(ts, j - 1), bp = __shfl(tp, j - 1);                  // (every lane takes part)
    const uint32_t cont = (uint32_t)__ballot(j > 0 && tp > 0 && ts == bs && tp == bp + 1) & 0xFFFFu;   // bit j: row b - 3 + j
    const uint32_t first = (uint32_t)__ballot(tp >= 0 && (tp & 3) == 0) & 0xFFFFu & cont >> 1 & cont >> 2 & cont >> 3;
    // first: rows that begin four in a row; the one among this wave's own, if any
    const uint32_t mine = first >> 3 & 0xFu;
    const int q0 = mine ? __builtin_ctz(mine) : 0;

    const int sq = __shfl(ts, r + 3), p = __shfl(tp, r + 3);
    const int page = b + r < T && (unsigned)sq < (unsigned)c.n_seq ? c.page_of(sq, p) : -1;
    const int tok = p & (c.page() - 1);
    uint32_t code[VL / 4];
    float s = quantise<FMT, VL, 16>(x, code);
    load_row<DT, VL>(vp + (long)(mine ? min(b + q0 + r, T - 1) : t) * rs * ES, y);
    if (page >= 0) {
        const size_t at = c.token0(page, h) + tok;
        uint32_t *o = reinterpret_cast<uint32_t *>(c.k + at * D + VL * j);
#pragma unroll
        for (int i = 0; i < VL / 4; i++) o[i] = code[i];
        if (j == 0) c.ks[at] = s;
    }
    if (mine) {
        s = quantise<FMT, VL, 16>(y, code);
        const int qs = __shfl(ts, q0 + 3), qp = __shfl(tp, q0 + 3);
        const int pg = (unsigned)qs < (unsigned)c.n_seq ? c.page_of(qs, qp) : -1;
        const size_t at = c.token0(max(pg, 0), h) + (qp & (c.page() - 1));
#pragma unroll
        for (int i = 0; i < VL / 4; i++) {
            const uint32_t w = transpose_rows(code[i], r);
            if (pg >= 0) *reinterpret_cast<uint32_t *>(c.v + at * D + (VL * j + 4 * i + r) * 4) = w;
        }
        if (pg >= 0 && j == 0) c.vs[at + r] = s;
    }
    // this row in no such four: bit 3 + r of first, or of the three rows before it
    const uint32_t part = first | first << 1 | first << 2 | first << 3;
    const bool single = page >= 0 && !(part >> (3 + r) & 1);
    if (!__any(single)) return;
    if (mine) load_row<DT, VL>(vp + (long)t * rs * ES, y);
    s = quantise<FMT, VL, 16>(y, code);
    if (!single) return;
    const size_t at = c.token0(page, h);
    uint8_t *o = c.v + (at + (tok & ~3)) * D + VL * j * 4 + (tok & 3);
#pragma unroll
    for (int i = 0; i < VL; i++) o[4 * i] = (uint8_t)(code[i / 4] >> (8 * (i % 4)));
    if (j == 0) c.vs[at + tok] = s;
}

// D / 8 lanes a row and head, 8 values a lane; keys, then values.
template <int DT, int FMT, int D>
__global__ void __launch_bounds__(kKvThreads)
k_kv_read(KvView c, uint8_t *__restrict__ k, uint8_t *__restrict__ v, long rs, long hs, const int *__restrict__ seq,
          const int *__restrict__ pos, int T) {
    constexpr int LPR = D / 8, ES = DT == QFM_DT_F32 ? 4 : 2;
    const long u = ((long)blockIdx.x * kKvThreads + threadIdx.x) / LPR;
    const int j = threadIdx.x % LPR;
    const long t = u / c.heads;
    const int h = (int)(u - t * c.heads);
    if (t >= T) return;
    const int sq = seq[t], p = pos[t];
    const int page = (unsigned)sq < (unsigned)c.n_seq ? c.page_of(sq, p) : -1;
    if (page < 0) return;
    const int tok = p & (c.page() - 1);
    const size_t at = c.token0(page, h);
    const long o = (t * rs + h * hs + 8 * j) * ES;
    float x[8];
    if (k) {
        const uint2 w = *reinterpret_cast<const uint2 *>(c.k + (at + tok) * D + 8 * j);
        const float s = c.ks[at + tok];
#pragma unroll
        for (int q = 0; q < 8; q++) x[q] = code_value<FMT>(q < 4 ? w.x : w.y, q & 3) * s;
        store8<DT>(k + o, x);
    }
    if (v) {
        const uint4 *w = reinterpret_cast<const uint4 *>(c.v + (at + (tok & ~3)) * D + 32 * j);
        const uint4 a = w[0], b = w[1];
        const uint32_t d[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        const float s = c.vs[at + tok];
#pragma unroll
        for (int q = 0; q < 8; q++) x[q] = code_value<FMT>(d[q], tok & 3) * s;
        store8<DT>(v + o, x);
    }
}

int kv_view(const qfm_kv_cache *c, const qfm_kv_seqs *sq, KvView *out, const char *who) {
    if (!c || !sq || !c->k || !c->v || !c->ks || !c->vs || !sq->table) {
        set_error(-1, "%s: null cache, page table or buffer", who);
        return -1;
    }
    if (c->page < 16 || c->page > 256 || (c->page & (c->page - 1))) {
        set_error(-1, "%s: page of %d tokens (16, 32, 64, 128 or 256)", who, c->page);
        return -1;
    }
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
        set_error(-1, "%s: head_dim %d (64, 128 or 256)", who, c->head_dim);
        return -1;
    }
    if (c->fmt != QFM_KV_INT8 && c->fmt != QFM_KV_E4M3) {
        set_error(-1, "%s: cache format %d", who, c->fmt);
        return -1;
    }
    if (c->n_pages < 1 || c->kv_heads < 1 || c->kv_heads > 1024 || sq->n_seq < 1 || sq->n_seq > 65535 ||
        sq->max_pages < 1) {
        set_error(-1, "%s: %d pages, %d heads (1..1024), %d sequences (1..65535), %d pages a sequence", who, c->n_pages,
                  c->kv_heads, sq->n_seq, sq->max_pages);
        return -1;
    }
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15 ||
        (reinterpret_cast<uintptr_t>(c->ks) | reinterpret_cast<uintptr_t>(c->vs)) & 15) {
        set_error(-1, "%s: cache buffers are 16-byte aligned", who);
        return -1;
    }
    *out = KvView{static_cast<uint8_t *>(c->k), static_cast<uint8_t *>(c->v), c->ks, c->vs, sq->table, c->n_pages,
                  __builtin_ctz((unsigned)c->page), c->kv_heads, sq->n_seq, sq->max_pages};
    return 0;
}

static int rows_check(const void *k, const void *v, int dtype, long rs, long hs, long least, const int *seq,
                      const int *pos, int T, const char *who) {
    if (dtype != QFM_DT_F32 && dtype != QFM_DT_BF16 && dtype != QFM_DT_F16) {
        set_error(-1, "%s: element type %d", who, dtype);
        return -1;
    }
    if (!seq || !pos || T < 0 || T > 1 << 24) {
        set_error(-1, "%s: null sequences or positions, or T = %d", who, T);
        return -1;
    }
    if (rs < least || hs < least || rs % 8 || hs % 8) {
        set_error(-1, "%s: strides %ld and %ld (multiples of 8, at least %ld)", who, rs, hs, least);
        return -1;
    }
    if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) {
        set_error(-1, "%s: rows are 16-byte aligned", who);
        return -1;
    }
    return 0;
}

}  // namespace qfm

using namespace qfm;

#define QFM_KV_D(KERNEL, DT, FMT)                                                                                  \
    switch (c->head_dim) {                                                                                         \
        case 64: hipLaunchKernelGGL((KERNEL<DT, FMT, 64>), g, b, 0, s, QFM_KV_ARGS); break;                        \
        case 128: hipLaunchKernelGGL((KERNEL<DT, FMT, 128>), g, b, 0, s, QFM_KV_ARGS); break;                      \
        default: hipLaunchKernelGGL((KERNEL<DT, FMT, 256>), g, b, 0, s, QFM_KV_ARGS); break;                       \
    }
#define QFM_KV_LAUNCH(KERNEL)                                                                                      \
    switch (dtype * 2 + c->fmt) {                                                                                  \
        case QFM_DT_F32 * 2 + QFM_KV_INT8: QFM_KV_D(KERNEL, QFM_DT_F32, QFM_KV_INT8) break;                        \
        case QFM_DT_F32 * 2 + QFM_KV_E4M3: QFM_KV_D(KERNEL, QFM_DT_F32, QFM_KV_E4M3) break;                        \
        case QFM_DT_BF16 * 2 + QFM_KV_INT8: QFM_KV_D(KERNEL, QFM_DT_BF16, QFM_KV_INT8) break;                      \
        case QFM_DT_BF16 * 2 + QFM_KV_E4M3: QFM_KV_D(KERNEL, QFM_DT_BF16, QFM_KV_E4M3) break;                      \
        case QFM_DT_F16 * 2 + QFM_KV_INT8: QFM_KV_D(KERNEL, QFM_DT_F16, QFM_KV_INT8) break;                        \
        default: QFM_KV_D(KERNEL, QFM_DT_F16, QFM_KV_E4M3) break;                                                  \
    }

extern "C" {

int qfm_kv_write(const qfm_kv_cache *c, const qfm_kv_seqs *sq, const void *k, const void *v, int dtype,
                 long row_stride, long head_stride, const int *seq, const int *pos, int T, hipStream_t s) {
    const char *who = "qfm_kv_write";
    KvView w;
    if (kv_view(c, sq, &w, who)) return -1;
    if (!k || !v) { set_error(-1, "%s: null rows", who); return -1; }
    if (rows_check(k, v, dtype, row_stride, head_stride, 0, seq, pos, T, who)) return -1;
    if (T == 0) return 0;
    const long waves = (long)((T + 3) / 4) * w.heads;
    const dim3 g((unsigned)((waves + kKvThreads / 64 - 1) / (kKvThreads / 64))), b(kKvThreads);
#define QFM_KV_ARGS w, static_cast<const uint8_t *>(k), static_cast<const uint8_t *>(v), row_stride, head_stride, seq, pos, T
    if (T <= kFewRows) {
        const dim3 g((unsigned)((T * w.heads * 2 * (c->head_dim / 8) + kKvThreads - 1) / kKvThreads));
        QFM_KV_LAUNCH(k_kv_write_few)
    } else {
        QFM_KV_LAUNCH(k_kv_write)
    }
#undef QFM_KV_ARGS
    return check_launch(who) ? -3 : 0;
}

int qfm_kv_read(const qfm_kv_cache *c, const qfm_kv_seqs *sq, void *k, void *v, int dtype, long row_stride,
                long head_stride, const int *seq, const int *pos, int T, hipStream_t s) {
    const char *who = "qfm_kv_read";
    KvView w;
    if (kv_view(c, sq, &w, who)) return -1;
    if (!k && !v) { set_error(-1, "%s: null rows", who); return -1; }
    if (rows_check(k, v, dtype, row_stride, head_stride, c->head_dim, seq, pos, T, who)) return -1;
    if (T == 0) return 0;
    const dim3 g((unsigned)(((long)T * w.heads * (c->head_dim / 8) + kKvThreads - 1) / kKvThreads)), b(kKvThreads);
#define QFM_KV_ARGS w, static_cast<uint8_t *>(k), static_cast<uint8_t *>(v), row_stride, head_stride, seq, pos, T
    QFM_KV_LAUNCH(k_kv_read)
#undef QFM_KV_ARGS
    return check_launch(who) ? -3 : 0;
}

}  // extern "C"

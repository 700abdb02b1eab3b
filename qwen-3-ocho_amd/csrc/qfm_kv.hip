// qfm_kv.hip -- the quantised key/value cache: rows in (qfm_kv_write) and rows
// back (qfm_kv_read).
//
// A row of one head is D values with one scale: amax over the row, then one
// division a value. Both kernels are bound by bytes (2 or 4 in and 1 out a
// value, or the reverse) and, at a few rows, by the chain of dependent loads
// row -> sequence and position -> page.
#include "qfm_kv.h"
#include "qfm_internal.h"

namespace qfm {

constexpr int kKvThreads = 256;

// code of v / s in the low byte
template <int FMT>
__device__ __forceinline__ uint32_t kv_code(float v, float s) {
    const float q = v / s;
    if constexpr (FMT == QFM_KV_INT8) return (uint32_t)(int)fminf(127.0f, fmaxf(-127.0f, rintf(q))) & 0xFFu;
    else return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(fminf(448.0f, fmaxf(-448.0f, q)), 0.0f, 0, false) & 0xFFu;
}

// D / 8 lanes a row and head, 8 values a lane; keys, then values.
template <int DT, int FMT, int D>
__global__ void __launch_bounds__(kKvThreads)
k_kv_write(KvView c, const uint8_t *__restrict__ k, const uint8_t *__restrict__ v, long rs, long hs,
           const int *__restrict__ seq, const int *__restrict__ pos, int T) {
    constexpr int LPR = D / 8, ES = DT == QFM_DT_F32 ? 4 : 2;
    constexpr float kInv = FMT == QFM_KV_INT8 ? 1.0f / 127.0f : 1.0f / 448.0f;
    const long u = ((long)blockIdx.x * kKvThreads + threadIdx.x) / LPR;
    const int j = threadIdx.x % LPR;
    const long t = u / c.heads;
    const int h = (int)(u - t * c.heads);
    if (t >= T) return;                                     // whole rows: LPR lanes leave together
    float x[2][8];
    load8<DT>(k + (t * rs + h * hs + 8 * j) * ES, x[0]);
    load8<DT>(v + (t * rs + h * hs + 8 * j) * ES, x[1]);
    const int sq = seq[t], p = pos[t];
    const int page = (unsigned)sq < (unsigned)c.n_seq ? c.page_of(sq, p) : -1;
    const int tok = p & (c.page() - 1);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        // the largest magnitude as bits: NaN and infinity above every number
        uint32_t m = 0;
#pragma unroll
        for (int q = 0; q < 8; q++) m = max(m, __float_as_uint(x[i][q]) & 0x7FFFFFFFu);
#pragma unroll
        for (int o = LPR / 2; o; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
        const bool fine = m < 0x7F800000u;
        float s = __uint_as_float(m) * kInv;
        if (s == 0.0f) s = 1.0f;
        uint32_t code[8];
#pragma unroll
        for (int q = 0; q < 8; q++) code[q] = fine ? kv_code<FMT>(x[i][q], s) : 0u;
        if (page < 0) continue;
        const size_t at = c.token0(page, h);
        if (j == 0) (i ? c.vs : c.ks)[at + tok] = fine ? s : __uint_as_float(0x7FC00000u);
        if (i == 0) {
            *reinterpret_cast<uint2 *>(c.k + (at + tok) * D + 8 * j) =
                make_uint2(code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24,
                           code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24);
        } else {
            uint8_t *o = c.v + (at + (tok & ~3)) * D + (8 * j) * 4 + (tok & 3);
#pragma unroll
            for (int q = 0; q < 8; q++) o[4 * q] = (uint8_t)code[q];
        }
    }
}

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
    const dim3 g((unsigned)(((long)T * w.heads * (c->head_dim / 8) + kKvThreads - 1) / kKvThreads)), b(kKvThreads);
#define QFM_KV_ARGS w, static_cast<const uint8_t *>(k), static_cast<const uint8_t *>(v), row_stride, head_stride, seq, pos, T
    QFM_KV_LAUNCH(k_kv_write)
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

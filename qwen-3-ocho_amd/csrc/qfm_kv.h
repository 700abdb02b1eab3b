// qfm_kv.h -- the key/value cache as its kernels see it (qfm_kv.hip, qfm_attn.hip).
#pragma once
#include "qfm_dev.h"
#include "../../include/qf_attn.h"

namespace qfm {

// A checked qfm_kv_cache and qfm_kv_seqs, passed to kernels by value.
struct KvView {
    uint8_t *k, *v;
    float *ks, *vs;
    const int *table;
    int n_pages, page_log2, heads, n_seq, max_pages;
    __device__ __forceinline__ int page() const { return 1 << page_log2; }
    // the page that holds position p of sequence s (s checked), or -1
    __device__ __forceinline__ int page_of(int s, long p) const {
        const long i = p >> page_log2;
        if (p < 0 || i >= max_pages) return -1;
        const int g = table[(long)s * max_pages + i];
        return (unsigned)g < (unsigned)n_pages ? g : -1;
    }
    // token index of (page, head, token 0): k and v codes lie at D times it
    __device__ __forceinline__ size_t token0(int page_id, int head) const {
        return ((size_t)page_id * heads + head) << page_log2;
    }
};

// 0 and the view, or -1 with the error latched
int kv_view(const qfm_kv_cache *c, const qfm_kv_seqs *sq, KvView *out, const char *who);
inline size_t dt_size(int dtype) { return dtype == QFM_DT_F32 ? 4 : 2; }

// 8 values of a row, widened to fp32 (p 16-byte aligned)
template <int DT>
__device__ __forceinline__ void load8(const void *p, float (&v)[8]) {
    if constexpr (DT == QFM_DT_F32) {
        const float4 a = static_cast<const float4 *>(p)[0], b = static_cast<const float4 *>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 w = *static_cast<const uint4 *>(p);
        const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (DT == QFM_DT_BF16) {
                v[2 * i] = bf16_lo(d[i]);
                v[2 * i + 1] = bf16_hi(d[i]);
            } else {
                v[2 * i] = (float)as_h2(d[i]).x;
                v[2 * i + 1] = (float)as_h2(d[i]).y;
            }
        }
    }
}
// two values rounded to nearest even, as one word
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    static_assert(DT != QFM_DT_F32, "16-bit types");
    if constexpr (DT == QFM_DT_BF16) return (uint32_t)f32_to_bf16(a) | ((uint32_t)f32_to_bf16(b) << 16);
    const f16x2_t h = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, h);
}
template <int DT>
__device__ __forceinline__ void store8(void *p, const float (&v)[8]) {
    if constexpr (DT == QFM_DT_F32) {
        static_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        static_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *static_cast<uint4 *>(p) = make_uint4(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]),
                                              pack2<DT>(v[6], v[7]));
    }
}

// byte j of w as a cache value without its scale
template <int FMT>
__device__ __forceinline__ float code_value(uint32_t w, int j) {
    if constexpr (FMT == QFM_KV_INT8) return (float)((int)((w >> (8 * j) ^ 0x80u) & 0xFFu) - 128);
    else return __builtin_amdgcn_cvt_f32_fp8((int)(w >> (8 * j) & 0xFFu), 0);
}

}  // namespace qfm

// qfm_lora.hip -- low-rank adapters of many requests beside the projections
// that their rows share (qfm_lora_rows).
//
//   k_lora_in   h[t] = A[e] x[t]           (fp32, into the workspace)
//   k_lora_out  y[t] = base[t] + scale[e] B[e] h[t]
//
// Rows are taken 16 at a time as the columns of an MFMA, whatever their
// adapters: a column's result depends on that row alone, so a workgroup runs
// the product once for each distinct adapter of its 16 rows and keeps the
// columns that have it. Neighbours of one prompt share an adapter (one pass); a
// decode batch has up to 16 (EACH: a workgroup for each, none of which waits
// for the others). No sorting of rows, no atomics, one writer a value.
#include "qfm_dev.h"
#include "qfm_mfma.h"
#include "qfm_internal.h"
#include "../../include/qf_attn.h"
#include "../../include/qf_dense.h"

namespace qfm {

struct LoraArgs {
    const void *a[4], *b[4];
    const float *base[4];
    float *y[4];
    const int *rank, *slot;
    const float *scale;
    const void *x;
    float *h;                          // [T][n R]
    long xs;
    int rows[4], n, K, R, slots, T;
};

template <int DT>
__device__ __forceinline__ f32x4_t lora_mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
    if constexpr (DT == QFM_DT_BF16) return mfma_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c);
    else return mfma_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c);
}

// The slot of this lane's row (lane % 16) of block b, -1 for none, and the next
// distinct slot of the block's rows not yet in `left` (16 bits).
__device__ __forceinline__ int lora_slot(const LoraArgs &a, int b, int l16) {
    const int t = 16 * b + l16, e = t < a.T ? a.slot[t] : -1;
    return (unsigned)e < (unsigned)a.slots ? e : -1;
}
__device__ __forceinline__ int next_slot(int e, uint32_t &left) {
    const int cur = __builtin_amdgcn_readlane(e, __builtin_ctz(left));
    left &= ~(uint32_t)__ballot(e == cur);
    return cur;
}

constexpr int kLoraInWaves = 8;

// One 16-row tile of A a workgroup (blockIdx.y over the n projections' tiles);
// the waves take the chunks of 64 inner values in turn.
template <int DT, bool EACH>
__global__ void __launch_bounds__(64 * kLoraInWaves)
k_lora_in(LoraArgs a) {
    __shared__ f32x4_t s_acc[kLoraInWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, l16 = lane & 15;
    const int tiles = (a.R + 15) >> 4, i = (int)blockIdx.y / tiles, r0 = ((int)blockIdx.y - i * tiles) * 16;
    const int e = lora_slot(a, (int)blockIdx.x, l16);
    uint32_t left = (uint32_t)__ballot(e >= 0) & 0xFFFFu;
    int skip = EACH ? (int)blockIdx.z : 0;
    const uint16_t *x = static_cast<const uint16_t *>(a.x) + (size_t)min(16 * (int)blockIdx.x + l16, a.T - 1) * a.xs + 16 * g;
    while (left) {
        const int cur = next_slot(e, left);
        if (EACH && skip--) continue;
        const uint16_t *w = static_cast<const uint16_t *>(a.a[i]) + ((size_t)cur * a.R + min(r0 + l16, a.R - 1)) * a.K + 16 * g;
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
        for (int k = 64 * wave; k < a.K; k += 64 * kLoraInWaves) {
            const u32x4_t *wp = reinterpret_cast<const u32x4_t *>(w + k), *xp = reinterpret_cast<const u32x4_t *>(x + k);
            acc = lora_mfma<DT>(wp[0], xp[0], acc);
            acc = lora_mfma<DT>(wp[1], xp[1], acc);
        }
        s_acc[wave][lane] = acc;
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int v = 1; v < kLoraInWaves; v++) acc += s_acc[v][lane];
            const int rank = a.rank[cur];
            const int r = r0 + 4 * g;
            if (e == cur && r < a.R) {
                float4 o = make_float4(acc[0], acc[1], acc[2], acc[3]);
                if (r + 0 >= rank) o.x = 0.0f;
                if (r + 1 >= rank) o.y = 0.0f;
                if (r + 2 >= rank) o.z = 0.0f;
                if (r + 3 >= rank) o.w = 0.0f;
                *reinterpret_cast<float4 *>(a.h + (size_t)(16 * (int)blockIdx.x + l16) * (a.n * a.R) + i * a.R + r) = o;
            }
        }
        if (EACH) return;
        __syncthreads();
    }
}

constexpr int kLoraOutWaves = 4, kLoraOutTiles = 4;   // tiles of 16 outputs a wave

// blockIdx.y: 256 outputs of one projection (first: the projections' first such
// block). KS: 32-value steps of the rank.
struct LoraFirst { int v[5]; };
template <int DT, int KS, bool EACH>
__global__ void __launch_bounds__(64 * kLoraOutWaves)
k_lora_out(LoraArgs a, LoraFirst first) {
    constexpr int NP = DT == QFM_DT_BF16 ? 3 : 2;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, l16 = lane & 15;
    int i = 0;
    while (i < 3 && (int)blockIdx.y >= first.v[i + 1]) i++;
    const int N = a.rows[i], o0 = (((int)blockIdx.y - first.v[i]) * kLoraOutWaves + wave) * (16 * kLoraOutTiles);
    const int t = 16 * (int)blockIdx.x + l16, e = lora_slot(a, (int)blockIdx.x, l16);
    uint32_t left = (uint32_t)__ballot(e >= 0) & 0xFFFFu;
    int skip = EACH ? (int)blockIdx.z : 0;
    bool mine = t < a.T && (EACH ? e < 0 && skip == 0 : true);      // columns that this wave writes
    f32x4_t acc[kLoraOutTiles];
#pragma unroll
    for (int q = 0; q < kLoraOutTiles; q++) acc[q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float factor = 0.0f;
    while (left) {
        const int cur = next_slot(e, left);
        if (EACH && skip--) continue;
        const bool here = e == cur;
        if (EACH) mine |= here;
        // this row's inner values, whole, as 16-bit numbers
        float v[KS][8], m = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; s++) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[s][j] = 0.0f;
            if (here && 32 * s + 8 * g < a.R) {
                const float4 *p = reinterpret_cast<const float4 *>(a.h + (size_t)t * (a.n * a.R) + i * a.R + 32 * s + 8 * g);
                const float4 c = p[0], d = p[1];
                v[s][0] = c.x; v[s][1] = c.y; v[s][2] = c.z; v[s][3] = c.w; v[s][4] = d.x; v[s][5] = d.y; v[s][6] = d.z; v[s][7] = d.w;
            }
#pragma unroll
            for (int j = 0; j < 8; j++) m = fmaxf(m, fabsf(v[s][j]));
        }
        float sc = 1.0f, back = 1.0f;
        if constexpr (DT == QFM_DT_F16) {
            m = fmaxf(m, __shfl_xor(m, 16));
            const int k = f16_exp(fmaxf(m, __shfl_xor(m, 32)));
            sc = exp2i(k);
            back = exp2i(-k);
        }
        u32x4_t hp[KS][NP];
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float c = v[s][2 * j] * sc, d = v[s][2 * j + 1] * sc;
#pragma unroll
                for (int p = 0; p < NP; p++) {
                    if constexpr (DT == QFM_DT_BF16) {
                        const uint32_t u = (uint32_t)f32_to_bf16(c) | ((uint32_t)f32_to_bf16(d) << 16);
                        hp[s][p][j] = u;
                        c -= bf16_lo(u);
                        d -= bf16_hi(u);
                    } else {
                        const f16x2_t u = {(_Float16)c, (_Float16)d};
                        hp[s][p][j] = __builtin_bit_cast(uint32_t, u);
                        c -= (float)u.x;
                        d -= (float)u.y;
                    }
                }
            }
        const int rank = min(max(a.rank[cur], 0), a.R);
        if (here) factor = a.scale[cur] * back;
        const uint16_t *w = static_cast<const uint16_t *>(a.b[i]) + (size_t)cur * N * a.R;
#pragma unroll
        for (int q = 0; q < kLoraOutTiles; q++) {
            const uint16_t *wr = w + (size_t)min(o0 + 16 * q + l16, N - 1) * a.R;
            f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const int k = 32 * s + 8 * g, keep = rank - k;      // columns from rank on count as zeros
                u32x4_t b = {0u, 0u, 0u, 0u};
                if (keep > 0) b = *reinterpret_cast<const u32x4_t *>(wr + k);
                if (keep < 8) {
#pragma unroll
                    for (int j = 0; j < 4; j++) b[j] &= keep >= 2 * j + 2 ? ~0u : keep == 2 * j + 1 ? 0xFFFFu : 0u;
                }
#pragma unroll
                for (int p = 0; p < NP; p++) sum = lora_mfma<DT>(b, hp[s][p], sum);
            }
            // chosen, not added: an infinite weight times another row's zeros is NaN
#pragma unroll
            for (int j = 0; j < 4; j++) acc[q][j] = here ? sum[j] : acc[q][j];
        }
        if (EACH) break;
    }
    if (!mine) return;
    const bool whole = N % 4 == 0;
#pragma unroll
    for (int q = 0; q < kLoraOutTiles; q++) {
        const int o = o0 + 16 * q + 4 * g;
        if (o >= N) break;
        const size_t at = (size_t)t * N + o;
        float *y = a.y[i] + at;
        const float *base = a.base[i] ? a.base[i] + at : nullptr;
        if (whole) {
            float4 v = base ? *reinterpret_cast<const float4 *>(base) : make_float4(0.f, 0.f, 0.f, 0.f);
            v.x = fmaf(factor, acc[q][0], v.x); v.y = fmaf(factor, acc[q][1], v.y);
            v.z = fmaf(factor, acc[q][2], v.z); v.w = fmaf(factor, acc[q][3], v.w);
            *reinterpret_cast<float4 *>(y) = v;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (o + j < N) y[j] = fmaf(factor, acc[q][j], base ? base[j] : 0.0f);
        }
    }
}

// up to here a workgroup for each of a block's up to 16 adapters
constexpr int kLoraEachRows = 256;

static int lora_check(const qfm_lora *l, int T, const char *who) {
    if (!l || l->n < 1 || l->n > 4 || l->K < 64 || l->K > 65536 || l->K % 64 || l->R < 8 || l->R > 128 || l->R % 8 ||
        l->slots < 1 || T < 0 || T > 1 << 20 || (l->dtype != QFM_DT_BF16 && l->dtype != QFM_DT_F16)) {
        if (who)
            set_error(-1, "%s: n 1..4, K a multiple of 64 up to 65536, R a multiple of 8 up to 128, slots, T up to 2^20, a 16-bit type",
                      who);
        return -1;
    }
    return 0;
}

template <int DT, bool EACH>
static void lora_launch(const LoraArgs &a, const LoraFirst &f, hipStream_t s) {
    const unsigned blocks = (unsigned)((a.T + 15) / 16), z = EACH ? 16u : 1u;
    hipLaunchKernelGGL((k_lora_in<DT, EACH>), dim3(blocks, (unsigned)(a.n * ((a.R + 15) / 16)), z), dim3(64 * kLoraInWaves), 0, s, a);
    const dim3 g(blocks, (unsigned)f.v[4], z), b(64 * kLoraOutWaves);
    if (a.R <= 32) hipLaunchKernelGGL((k_lora_out<DT, 1, EACH>), g, b, 0, s, a, f);
    else if (a.R <= 64) hipLaunchKernelGGL((k_lora_out<DT, 2, EACH>), g, b, 0, s, a, f);
    else hipLaunchKernelGGL((k_lora_out<DT, 4, EACH>), g, b, 0, s, a, f);
}

}  // namespace qfm

using namespace qfm;

extern "C" {

size_t qfm_lora_ws_bytes(const qfm_lora *l, int T) {
    return lora_check(l, T, nullptr) ? 0 : (size_t)T * l->n * l->R * 4;
}

int qfm_lora_rows(const qfm_lora *l, const void *x, long x_stride, const int *slot, int T, void *ws, size_t ws_bytes,
                  hipStream_t s) {
    const char *who = "qfm_lora_rows";
    if (lora_check(l, T, who)) return -1;
    LoraArgs a{};
    LoraFirst f{};
    uintptr_t align = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(ws);
    bool null = !x || !slot || !l->rank || !l->scale;
    for (int i = 0; i < l->n; i++) {
        null |= !l->a[i] || !l->b[i] || !l->y[i];
        if (l->rows[i] < 1 || l->rows[i] > 1 << 20) { set_error(-1, "%s: projection of %d outputs", who, l->rows[i]); return -1; }
        align |= reinterpret_cast<uintptr_t>(l->a[i]) | reinterpret_cast<uintptr_t>(l->b[i]) |
                 reinterpret_cast<uintptr_t>(l->base[i]) | reinterpret_cast<uintptr_t>(l->y[i]);
        a.a[i] = l->a[i]; a.b[i] = l->b[i]; a.base[i] = l->base[i]; a.y[i] = l->y[i]; a.rows[i] = l->rows[i];
    }
    if (null) { set_error(-1, "%s: null argument", who); return -1; }
    if (align & 15) { set_error(-1, "%s: x, the adapters, base, y and ws are 16-byte aligned", who); return -1; }
    if (x_stride < 0 || x_stride % 8) { set_error(-1, "%s: x_stride %ld (a multiple of 8)", who, x_stride); return -1; }
    const size_t need = qfm_lora_ws_bytes(l, T);
    if (need && (!ws || ws_bytes < need)) {
        set_error(-1, "%s: workspace of %zu bytes, %zu needed", who, ws ? ws_bytes : (size_t)0, need);
        return -1;
    }
    constexpr int per = 16 * kLoraOutTiles * kLoraOutWaves;
    for (int i = 0; i < 4; i++) f.v[i + 1] = f.v[i] + (i < l->n ? (l->rows[i] + per - 1) / per : 0);
    if (f.v[4] > 65535) { set_error(-1, "%s: %d blocks of %d outputs", who, f.v[4], per); return -1; }
    if (T == 0) return 0;
    a.rank = l->rank; a.scale = l->scale; a.slot = slot; a.x = x; a.h = static_cast<float *>(ws);
    a.xs = x_stride; a.n = l->n; a.K = l->K; a.R = l->R; a.slots = l->slots; a.T = T;
    const bool each = T <= kLoraEachRows;
    if (l->dtype == QFM_DT_BF16) each ? lora_launch<QFM_DT_BF16, true>(a, f, s) : lora_launch<QFM_DT_BF16, false>(a, f, s);
    else each ? lora_launch<QFM_DT_F16, true>(a, f, s) : lora_launch<QFM_DT_F16, false>(a, f, s);
    return check_launch(who) ? -3 : 0;
}

}  // extern "C"

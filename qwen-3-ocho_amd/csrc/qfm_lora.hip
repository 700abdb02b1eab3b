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
// for the others). No sorting of rows, no atomics, one writer a value. The
// smallest calls take both products in one launch (k_lora_few).
//
// What it has to move is base and y (8 bytes an output and row), x and the
// adapters in use: 97.5 MB for 2050 rows of K 2048 to 4096 + 512 + 512 outputs at
// rank 64, of which k_lora_in takes 16.4 us and k_lora_out 22.6 (3.7 TB/s). A decode
// batch is bound by the chain launch, slots, A and x, sums, launch, h, B, base
// (37 rows of 24 adapters, 7 MB: 11.3 us).
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

// RT 16-row tiles of A a workgroup (blockIdx.y over the n projections' tiles)
// against CB 16-row blocks of x; the waves take the chunks of 64 inner values in
// turn, their sums meet in LDS. Rows of A and x lie K apart, so a fragment read
// straight from memory would take a cache line a lane (2050 rows: 27.6 us); a
// wave reads 8 rows of 128 bytes a request instead, U chunks together, and turns
// them in an LDS area of its own.
template <int DT, int RT, int CB>
__global__ void __launch_bounds__(64 * kLoraInWaves)
k_lora_in(LoraArgs a) {
    constexpr int U = RT * CB > 1 ? 2 : 4, NA = 2 * RT, NX = 2 * CB, PART = (NA + NX) * 1024;
    __shared__ __attribute__((aligned(16))) uint8_t s_buf[kLoraInWaves * (PART > RT * CB * 1024 ? PART : RT * CB * 1024)];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), g = lane >> 4, l16 = lane & 15;
    const int l8 = lane >> 3, ch = lane & 7, tiles = (a.R + 15) >> 4, most = a.n * tiles - 1;
    uint8_t *s_w = s_buf + wave * PART, *s_x = s_w + NA * 1024;
    f32x4_t *s_acc = reinterpret_cast<f32x4_t *>(s_buf);             // [waves][RT CB][64], once the chunks are done
    int e[CB];
    uint32_t left[CB], some = 0;
#pragma unroll
    for (int c = 0; c < CB; c++) {
        e[c] = lora_slot(a, (int)blockIdx.x * CB + c, l16);
        left[c] = (uint32_t)__ballot(e[c] >= 0) & 0xFFFFu;
        some |= left[c];
    }
    const uint16_t *x[NX];
#pragma unroll
    for (int n = 0; n < NX; n++)
        x[n] = static_cast<const uint16_t *>(a.x) + (size_t)min(16 * CB * (int)blockIdx.x + 8 * n + l8, a.T - 1) * a.xs + 8 * ch;
    // the adapters of these rows, every gridDim.z-th of them here
    for (int pass = 0; some; pass++) {
        // the next adapter: the first left block's first left row has it
        int cur = -1;
#pragma unroll
        for (int c = 0; c < CB; c++)
            if (cur < 0 && left[c]) cur = __builtin_amdgcn_readlane(e[c], __builtin_ctz(left[c]));
        some = 0;
#pragma unroll
        for (int c = 0; c < CB; c++) {
            left[c] &= ~(uint32_t)__ballot(e[c] == cur);
            some |= left[c];
        }
        if (pass % (int)gridDim.z != (int)blockIdx.z) continue;
        const uint16_t *w[NA];
#pragma unroll
        for (int n = 0; n < NA; n++) {
            const int y = min((int)blockIdx.y * RT + n / 2, most), i = y / tiles, r = (y - i * tiles) * 16 + (n & 1) * 8 + l8;
            w[n] = static_cast<const uint16_t *>(a.a[i]) + ((size_t)cur * a.R + min(r, a.R - 1)) * a.K + 8 * ch;
        }
        f32x4_t acc[RT][CB];
#pragma unroll
        for (int q = 0; q < RT; q++)
#pragma unroll
            for (int c = 0; c < CB; c++) acc[q][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        const int chunks = a.K / 64;
        for (int k0 = wave; k0 < chunks; k0 += U * kLoraInWaves) {
            u32x4_t wv[U][NA], xv[U][NX];
#pragma unroll
            for (int v = 0; v < U; v++) {
                const size_t at = 64 * (size_t)min(k0 + v * kLoraInWaves, chunks - 1);
#pragma unroll
                for (int n = 0; n < NA; n++) wv[v][n] = *reinterpret_cast<const u32x4_t *>(w[n] + at);
#pragma unroll
                for (int n = 0; n < NX; n++) xv[v][n] = *reinterpret_cast<const u32x4_t *>(x[n] + at);
            }
#pragma unroll
            for (int v = 0; v < U; v++) {
                if (k0 + v * kLoraInWaves >= chunks) break;
#pragma unroll
                for (int n = 0; n < NA; n++) *reinterpret_cast<u32x4_t *>(s_w + lds_at<128>(8 * n + l8, ch)) = wv[v][n];
#pragma unroll
                for (int n = 0; n < NX; n++) *reinterpret_cast<u32x4_t *>(s_x + lds_at<128>(8 * n + l8, ch)) = xv[v][n];
                wave_lds_fence();
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    u32x4_t xf[CB];
#pragma unroll
                    for (int c = 0; c < CB; c++) xf[c] = *reinterpret_cast<const u32x4_t *>(s_x + lds_at<128>(16 * c + l16, 4 * j + g));
#pragma unroll
                    for (int q = 0; q < RT; q++) {
                        const u32x4_t wf = *reinterpret_cast<const u32x4_t *>(s_w + lds_at<128>(16 * q + l16, 4 * j + g));
#pragma unroll
                        for (int c = 0; c < CB; c++) acc[q][c] = lora_mfma<DT>(wf, xf[c], acc[q][c]);
                    }
                }
                wave_lds_fence();
            }
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < RT; q++)
#pragma unroll
            for (int c = 0; c < CB; c++) s_acc[(wave * RT * CB + q * CB + c) * 64 + lane] = acc[q][c];
        const int rank = a.rank[cur];
        __syncthreads();
#pragma unroll
        for (int p = 0; p < RT * CB; p++) {
            if (p % kLoraInWaves != wave) continue;
            f32x4_t sum = s_acc[p * 64 + lane];
#pragma unroll
            for (int v = 1; v < kLoraInWaves; v++) sum += s_acc[(v * RT * CB + p) * 64 + lane];
            const int q = p / CB, c = p % CB, y = (int)blockIdx.y * RT + q, i = y / tiles, r = (y - i * tiles) * 16 + 4 * g;
            if (y <= most && e[c] == cur && r < a.R) {
                const float4 o = make_float4(r + 0 < rank ? sum[0] : 0.0f, r + 1 < rank ? sum[1] : 0.0f,
                                             r + 2 < rank ? sum[2] : 0.0f, r + 3 < rank ? sum[3] : 0.0f);
                const size_t t = 16 * (size_t)((int)blockIdx.x * CB + c) + l16;
                *reinterpret_cast<float4 *>(a.h + t * (a.n * a.R) + i * a.R + r) = o;
            }
        }
        __syncthreads();
    }
}

// A row's inner values (of the lanes l16 + 16 g: 8 g .. 8 g + 7 of each 32), whole,
// as 16-bit numbers; returns what undoes their common factor.
constexpr int inner_count(int dt) { return dt == QFM_DT_BF16 ? 3 : 2; }
template <int DT, int KS, int NP>
__device__ __forceinline__ float inner_parts(const float (&v)[KS][8], u32x4_t (&hp)[KS][NP]) {
    float sc = 1.0f, back = 1.0f;
    if constexpr (DT == QFM_DT_F16) {
        float m = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int j = 0; j < 8; j++) m = fmaxf(m, fabsf(v[s][j]));
        m = fmaxf(m, __shfl_xor(m, 16));
        const int k = f16_exp(fmaxf(m, __shfl_xor(m, 32)));
        sc = exp2i(k);
        back = exp2i(-k);
    }
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float c = v[s][2 * j] * sc, d = v[s][2 * j + 1] * sc;
#pragma unroll
            for (int p = 0; p < NP; p++) {
                if constexpr (DT == QFM_DT_BF16) {
                    // cut off after 8 bits, three times: 24 bits, nothing lost
                    const uint32_t u = pack_bf16_hi(c, d);
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
    return back;
}
// 8 columns of a row of B from column k on, those from rank on as zeros
__device__ __forceinline__ u32x4_t rank_columns(u32x4_t b, int keep) {
#pragma unroll
    for (int j = 0; j < 4; j++) b[j] &= keep >= 2 * j + 2 ? ~0u : keep == 2 * j + 1 ? 0xFFFFu : 0u;
    return b;
}

constexpr int kLoraOutWaves = 4, kLoraOutTiles = 4;   // tiles of 16 outputs a wave

// blockIdx.y: 256 outputs of one projection (first: the projections' first such
// block), NB 16-row blocks one after another, so many that all workgroups run
// at once: a first block takes about 12 us, from its slots over the adapter to
// the store, those behind it 4. B's fragments stay in registers from block to
// block while the adapter is the same. KS: 32-value steps of the rank.
struct LoraFirst { int v[5]; };
template <int DT, int KS, bool EACH>
__global__ void __launch_bounds__(64 * kLoraOutWaves)
k_lora_out(LoraArgs a, LoraFirst first, int NB) {
    constexpr int NP = inner_count(DT);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, l16 = lane & 15;
    int i = 0;
    while (i < 3 && (int)blockIdx.y >= first.v[i + 1]) i++;
    const int N = a.rows[i], o0 = (((int)blockIdx.y - first.v[i]) * kLoraOutWaves + wave) * (16 * kLoraOutTiles);
    constexpr int LJ = 68;
    __shared__ __attribute__((aligned(16))) float s_y[kLoraOutWaves][16 * LJ];
    const bool whole = N % 4 == 0;
    const float *base0 = a.base[i];
    const int oc = o0 + 4 * l16;                            // this lane's outputs of rows 4 q + g
    u32x4_t bf[kLoraOutTiles][KS];
    int have = -1;                                          // the adapter in bf
    // a block's slots, inner values and base (4 rows of 256 bytes a request) are
    // requested a block ahead
    auto request = [&](int blk, int &e, f32x4_t (&h)[KS][2], f32x4_t (&bs)[4]) {
        e = lora_slot(a, blk, l16);
        const float *hp = a.h + (size_t)min(16 * blk + l16, a.T - 1) * (a.n * a.R) + i * a.R;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const f32x4_t *p = reinterpret_cast<const f32x4_t *>(hp + min(32 * s + 8 * g, a.R - 8));
            h[s][0] = p[0];
            h[s][1] = p[1];
        }
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int tr = 16 * blk + 4 * q + g;
            bs[q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            if (base0 && tr < a.T && oc < N) {
                const float *p = base0 + (size_t)tr * N + oc;
                if (whole) bs[q] = *reinterpret_cast<const f32x4_t *>(p);
                else bs[q] = f32x4_t{p[0], oc + 1 < N ? p[1] : 0.0f, oc + 2 < N ? p[2] : 0.0f, oc + 3 < N ? p[3] : 0.0f};
            }
        }
    };
    int e, en;
    f32x4_t h[KS][2], hn[KS][2], bs[4], bn[4];
    request((int)blockIdx.x * NB, e, h, bs);
    for (int nb = 0; nb < NB; nb++) {
        const int blk = (int)blockIdx.x * NB + nb, t = 16 * blk + l16;
        if (16 * blk >= a.T) return;
        if constexpr (!EACH) request(min(blk + 1, (a.T - 1) / 16), en, hn, bn);
        uint32_t left = (uint32_t)__ballot(e >= 0) & 0xFFFFu;
        int skip = EACH ? (int)blockIdx.z : 0;
        bool mine = t < a.T && (EACH ? e < 0 && skip == 0 : true);      // rows that this wave writes
        f32x4_t acc[kLoraOutTiles];
#pragma unroll
        for (int q = 0; q < kLoraOutTiles; q++) acc[q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        float factor = 0.0f;
        while (left) {
            const int cur = next_slot(e, left);
            if (EACH && skip--) continue;
            const bool here = e == cur;
            if (EACH) mine |= here;
            if (cur != have) {
                have = cur;
                const int rank = min(max(a.rank[cur], 0), a.R);
                const uint16_t *w = static_cast<const uint16_t *>(a.b[i]) + (size_t)cur * N * a.R;
#pragma unroll
                for (int q = 0; q < kLoraOutTiles; q++) {
                    const uint16_t *wr = w + (size_t)min(o0 + 16 * q + l16, N - 1) * a.R;
#pragma unroll
                    for (int s = 0; s < KS; s++) {
                        const int k = 32 * s + 8 * g;
                        bf[q][s] = rank_columns(*reinterpret_cast<const u32x4_t *>(wr + min(k, a.R - 8)), rank - k);
                    }
                }
            }
            float v[KS][8];
#pragma unroll
            for (int s = 0; s < KS; s++) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[s][j] = 0.0f;
                if (here && 32 * s + 8 * g < a.R) {
#pragma unroll
                    for (int j = 0; j < 8; j++) v[s][j] = h[s][j / 4][j % 4];
                }
            }
            u32x4_t hp[KS][NP];
            const float back = inner_parts<DT, KS, NP>(v, hp);
            if (here) factor = a.scale[cur] * back;
#pragma unroll
            for (int q = 0; q < kLoraOutTiles; q++) {
                f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < KS; s++)
#pragma unroll
                    for (int p = 0; p < NP; p++) sum = lora_mfma<DT>(bf[q][s], hp[s][p], sum);
                // chosen, not added: an infinite weight times another row's zeros is NaN
#pragma unroll
                for (int j = 0; j < 4; j++) acc[q][j] = here ? sum[j] : acc[q][j];
            }
            if (EACH) break;
        }
        const uint32_t rows = (uint32_t)__ballot(mine) & 0xFFFFu;
        float *sy = s_y[wave];
#pragma unroll
        for (int q = 0; q < kLoraOutTiles; q++)
            *reinterpret_cast<float4 *>(&sy[l16 * LJ + 16 * q + 4 * g]) =
                make_float4(factor * acc[q][0], factor * acc[q][1], factor * acc[q][2], factor * acc[q][3]);
        wave_lds_fence();
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const float4 d = *reinterpret_cast<const float4 *>(&sy[(4 * q + g) * LJ + 4 * l16]);
            if (!(rows >> (4 * q + g) & 1) || oc >= N) continue;
            const float4 v = make_float4(bs[q][0] + d.x, bs[q][1] + d.y, bs[q][2] + d.z, bs[q][3] + d.w);
            float *y = a.y[i] + (size_t)(16 * blk + 4 * q + g) * N + oc;
            if (whole && !EACH) {
                // more than the caches keep: past them (2050 rows 44.1 -> 38.1 us; with a reader of y behind it 61.2 -> 60.4)
                __builtin_nontemporal_store(f32x4_t{v.x, v.y, v.z, v.w}, reinterpret_cast<f32x4_t *>(y));
            } else if (whole) {
                *reinterpret_cast<float4 *>(y) = v;
            } else {
                y[0] = v.x;
                if (oc + 1 < N) y[1] = v.y;
                if (oc + 2 < N) y[2] = v.z;
                if (oc + 3 < N) y[3] = v.w;
            }
        }
        wave_lds_fence();
        if constexpr (EACH) return;
        e = en;
#pragma unroll
        for (int s = 0; s < KS; s++) {
            h[s][0] = hn[s][0];
            h[s][1] = hn[s][1];
        }
#pragma unroll
        for (int q = 0; q < 4; q++) bs[q] = bn[q];
    }
}

// Both products in one launch, for few rows and small adapters: 256 outputs of a
// projection, 16 rows and the blockIdx.z-th of their adapters a workgroup, which
// finds the inner rows by itself (A is read N / 256 times, from the caches but for
// the first). Everything that depends on the slots alone (x, A, B, base) is
// requested together.
template <int DT, int KS>
__global__ void __launch_bounds__(64 * kLoraInWaves)
k_lora_few(LoraArgs a, LoraFirst first) {
    constexpr int NP = inner_count(DT), RT = 2 * KS, NA = 2 * RT, PART = (NA + 2) * 1024, U = KS == 1 ? 4 : 2;
    constexpr int TL = 2, LH = 32 * KS + 4, LJ = 16 * TL + 4;             // tiles of 16 outputs a wave
    __shared__ __attribute__((aligned(16))) uint8_t s_buf[kLoraInWaves * PART];
    __shared__ __attribute__((aligned(16))) float s_h[16 * LH];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), g = lane >> 4, l16 = lane & 15;
    const int l8 = lane >> 3, ch = lane & 7, blk = (int)blockIdx.x;
    int i = 0;
    while (i < 3 && (int)blockIdx.y >= first.v[i + 1]) i++;
    const int N = a.rows[i], o0 = (((int)blockIdx.y - first.v[i]) * kLoraInWaves + wave) * (16 * TL);
    const bool whole = N % 4 == 0;
    // base, 8 rows of 128 bytes a request
    const int oc = o0 + 4 * ch;
    f32x4_t bs[2];
#pragma unroll
    for (int q = 0; q < 2; q++) {
        const int tr = 16 * blk + 8 * q + l8;
        bs[q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        if (a.base[i] && tr < a.T && oc < N) {
            const float *p = a.base[i] + (size_t)tr * N + oc;
            if (whole) bs[q] = *reinterpret_cast<const f32x4_t *>(p);
            else bs[q] = f32x4_t{p[0], oc + 1 < N ? p[1] : 0.0f, oc + 2 < N ? p[2] : 0.0f, oc + 3 < N ? p[3] : 0.0f};
        }
    }
    const int e = lora_slot(a, blk, l16);
    uint32_t left = (uint32_t)__ballot(e >= 0) & 0xFFFFu;
    int cur = -1;
    for (int skip = (int)blockIdx.z; left; skip--) {
        const int c = next_slot(e, left);
        if (skip == 0) {
            cur = c;
            break;
        }
    }
    const bool mine = 16 * blk + l16 < a.T && (e == cur || (e < 0 && blockIdx.z == 0));    // (cur -1: those without)
    const uint32_t rows = (uint32_t)__ballot(mine) & 0xFFFFu;
    if (!rows || (cur < 0 && blockIdx.z)) return;            // the same for every wave
    f32x4_t acc[TL];
#pragma unroll
    for (int q = 0; q < TL; q++) acc[q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float factor = 0.0f;
    if (cur >= 0) {
        const int rank = min(max(a.rank[cur], 0), a.R);
        const float scale = a.scale[cur];
        u32x4_t bf[TL][KS];
#pragma unroll
        for (int q = 0; q < TL; q++)
#pragma unroll
            for (int s = 0; s < KS; s++)
                bf[q][s] = *reinterpret_cast<const u32x4_t *>(static_cast<const uint16_t *>(a.b[i]) +
                                                              ((size_t)cur * N + min(o0 + 16 * q + l16, N - 1)) * a.R + min(32 * s + 8 * g, a.R - 8));
        uint8_t *s_w = s_buf + wave * PART, *s_x = s_w + NA * 1024;
        const uint16_t *x[2], *w[NA];
#pragma unroll
        for (int n = 0; n < 2; n++)
            x[n] = static_cast<const uint16_t *>(a.x) + (size_t)min(16 * blk + 8 * n + l8, a.T - 1) * a.xs + 8 * ch;
#pragma unroll
        for (int n = 0; n < NA; n++)
            w[n] = static_cast<const uint16_t *>(a.a[i]) + ((size_t)cur * a.R + min(8 * n + l8, a.R - 1)) * a.K + 8 * ch;
        f32x4_t h[RT];
#pragma unroll
        for (int q = 0; q < RT; q++) h[q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        const int chunks = a.K / 64;
        for (int k0 = wave; k0 < chunks; k0 += U * kLoraInWaves) {
            u32x4_t wv[U][NA], xv[U][2];
#pragma unroll
            for (int v = 0; v < U; v++) {
                const size_t at = 64 * (size_t)min(k0 + v * kLoraInWaves, chunks - 1);
#pragma unroll
                for (int n = 0; n < NA; n++) wv[v][n] = *reinterpret_cast<const u32x4_t *>(w[n] + at);
#pragma unroll
                for (int n = 0; n < 2; n++) xv[v][n] = *reinterpret_cast<const u32x4_t *>(x[n] + at);
            }
#pragma unroll
            for (int v = 0; v < U; v++) {
                if (k0 + v * kLoraInWaves >= chunks) break;
#pragma unroll
                for (int n = 0; n < NA; n++) *reinterpret_cast<u32x4_t *>(s_w + lds_at<128>(8 * n + l8, ch)) = wv[v][n];
#pragma unroll
                for (int n = 0; n < 2; n++) *reinterpret_cast<u32x4_t *>(s_x + lds_at<128>(8 * n + l8, ch)) = xv[v][n];
                wave_lds_fence();
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const u32x4_t xf = *reinterpret_cast<const u32x4_t *>(s_x + lds_at<128>(l16, 4 * j + g));
#pragma unroll
                    for (int q = 0; q < RT; q++)
                        h[q] = lora_mfma<DT>(*reinterpret_cast<const u32x4_t *>(s_w + lds_at<128>(16 * q + l16, 4 * j + g)), xf, h[q]);
                }
                wave_lds_fence();
            }
        }
        // the waves' sums meet: lane (g, l16) holds inner values 4 g .. of row l16
        f32x4_t *s_acc = reinterpret_cast<f32x4_t *>(s_buf);
        __syncthreads();
#pragma unroll
        for (int q = 0; q < RT; q++) s_acc[(wave * RT + q) * 64 + lane] = h[q];
        __syncthreads();
        if (wave < RT) {
            f32x4_t sum = s_acc[wave * 64 + lane];
#pragma unroll
            for (int v = 1; v < kLoraInWaves; v++) sum += s_acc[(v * RT + wave) * 64 + lane];
            const int r = 16 * wave + 4 * g;
            *reinterpret_cast<float4 *>(&s_h[l16 * LH + r]) = make_float4(r + 0 < rank ? sum[0] : 0.0f, r + 1 < rank ? sum[1] : 0.0f,
                                                                          r + 2 < rank ? sum[2] : 0.0f, r + 3 < rank ? sum[3] : 0.0f);
        }
        __syncthreads();
        float v[KS][8];
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float4 y = *reinterpret_cast<const float4 *>(&s_h[l16 * LH + 32 * s + 8 * g + 4 * j]);
                v[s][4 * j] = y.x; v[s][4 * j + 1] = y.y; v[s][4 * j + 2] = y.z; v[s][4 * j + 3] = y.w;
            }
        u32x4_t hp[KS][NP];
        factor = inner_parts<DT, KS, NP>(v, hp) * scale;
#pragma unroll
        for (int q = 0; q < TL; q++) {
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const u32x4_t b = rank_columns(bf[q][s], rank - (32 * s + 8 * g));
#pragma unroll
                for (int p = 0; p < NP; p++) acc[q] = lora_mfma<DT>(b, hp[s][p], acc[q]);
            }
            // chosen: the columns of rows with other adapters hold what is none of theirs
#pragma unroll
            for (int j = 0; j < 4; j++) acc[q][j] = e == cur ? factor * acc[q][j] : 0.0f;
        }
    }
    float *sy = reinterpret_cast<float *>(s_buf) + wave * (16 * LJ);
#pragma unroll
    for (int q = 0; q < TL; q++)
        *reinterpret_cast<float4 *>(&sy[l16 * LJ + 16 * q + 4 * g]) = make_float4(acc[q][0], acc[q][1], acc[q][2], acc[q][3]);
    wave_lds_fence();
#pragma unroll
    for (int q = 0; q < 2; q++) {
        const int r = 8 * q + l8;
        const float4 d = *reinterpret_cast<const float4 *>(&sy[r * LJ + 4 * ch]);
        if (!(rows >> r & 1) || oc >= N) continue;
        const float4 v = make_float4(bs[q][0] + d.x, bs[q][1] + d.y, bs[q][2] + d.z, bs[q][3] + d.w);
        float *y = a.y[i] + (size_t)(16 * blk + r) * N + oc;
        if (whole) {
            *reinterpret_cast<float4 *>(y) = v;
        } else {
            y[0] = v.x;
            if (oc + 1 < N) y[1] = v.y;
            if (oc + 2 < N) y[2] = v.z;
            if (oc + 3 < N) y[3] = v.w;
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

// k_lora_few rather than two launches: while its workgroups, with A once each, are
// no more than the CUs, and A is short enough to arrive in two rounds of loads.
// One row to 4096 + 512 + 512 outputs of K 2048, rank 16: 6.2 us, 8.7 with two; 16
// rows of 16 adapters, 2560 of 2560, rank 32: 9.2 and 12.1; but 37 rows of that
// 16.3 and 12.5, one row of K 8192, rank 64, 18.3 and 13.3.
static bool lora_few(const LoraArgs &a, int outs) {
    const int each = a.T < 16 ? a.T : 16;
    return a.R <= 64 && a.K <= 4096 && a.R * a.K <= 1 << 17 && (long)((a.T + 15) / 16) * (each < a.slots ? each : a.slots) * outs <= 256;
}

template <int DT, bool EACH>
static void lora_launch(const LoraArgs &a, const LoraFirst &f, hipStream_t s) {
    constexpr int RT = EACH ? 1 : 4, CB = EACH ? 1 : 2;
    const int blocks = (a.T + 15) / 16, tiles = a.n * ((a.R + 15) / 16);
    if constexpr (EACH) {
        if (lora_few(a, f.v[4])) {
            const dim3 g((unsigned)blocks, (unsigned)f.v[4], 16u), b(64 * kLoraInWaves);
            if (a.R <= 32) hipLaunchKernelGGL((k_lora_few<DT, 1>), g, b, 0, s, a, f);
            else hipLaunchKernelGGL((k_lora_few<DT, 2>), g, b, 0, s, a, f);
            return;
        }
    }
    hipLaunchKernelGGL((k_lora_in<DT, RT, CB>), dim3((unsigned)((blocks + CB - 1) / CB), (unsigned)((tiles + RT - 1) / RT), EACH ? 16u : 2u),
                       dim3(64 * kLoraInWaves), 0, s, a);
    const int nb = EACH ? 1 : (int)(((long)blocks * f.v[4] + 511) / 512);
    const dim3 g((unsigned)((blocks + nb - 1) / nb), (unsigned)f.v[4], EACH ? 16u : 1u), b(64 * kLoraOutWaves);
    if (a.R <= 32) hipLaunchKernelGGL((k_lora_out<DT, 1, EACH>), g, b, 0, s, a, f, nb);
    else if (a.R <= 64) hipLaunchKernelGGL((k_lora_out<DT, 2, EACH>), g, b, 0, s, a, f, nb);
    else hipLaunchKernelGGL((k_lora_out<DT, 4, EACH>), g, b, 0, s, a, f, nb);
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

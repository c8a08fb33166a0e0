// gg_layernorm.h — layer norm over the last axis, forward and backward, with the weight's and the bias's gradients.
//
//   y = (x - mu) rstd w + b           mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps)        over the C features of a row
//   xh = (x - mu) rstd,  g = dy w:    dx = rstd (g - mean(g) - xh mean(g xh)),   dw = sum_rows dy xh,   db = sum_rows dy
//
// All bandwidth: forward reads x and writes y, backward reads x and dy and writes dx. A row lives in the registers of its TPR threads
// (eight features per thread and vector), so the variance is the mean of squared DIFFERENCES from the mean, taken from registers - no
// cancellation, one read. Statistics, sums and gradients are fp32. TPR is the smallest of 16 / 64 / 256 / 1024 threads that holds the
// row in NV vectors a thread: up to 64 threads the row sums are cross-lane adds without LDS or barrier.
//
// Backward: a workgroup walks rows blockIdx, blockIdx + gridDim, ... and keeps dw and db of its columns in registers; its sums go to
// part[block][2][C], and a second launch adds the workgroups' rows in a fixed order (no atomics: the same bits every time).
//
// 65536 x 2048 bf16: forward 103 us (5.2 TB/s), backward 153 us (5.3 TB/s) and 5.0 us for the column sums (medians of five); a large copy
// runs at 5.0 TB/s. 2496 x 512 bf16, forward: 4.1 us.
#pragma once
#include "gg_element.h"

struct GgLnParams {
    const void* x;
    const void* dy;
    const float* w;
    const float* b;
    void* y;            // forward: y; backward: dx (dense rows)
    float* mean;
    float* rstd;
    float* part;        // backward: [gridDim.x][2][C]
    long long rows, ldx, ldy;
    int C;
    float eps;
};

template <int TPR>
GG_DEVICE float gg_ln_row_sum(float v, float* red) {
    if constexpr (TPR == 16) return gg_row16_sum(v);
    else if constexpr (TPR == 64) return gg_wave_sum_all(v);
    else {
        v = gg_wave_sum_all(v);
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) red[wave] = v;
        gg_sync();
        float s = red[0];
        for (int i = 1; i < TPR / 64; ++i) s += red[i];
        return s;
    }
}

template <int T, int TPR, int NV>
GG_KERNEL GG_LAUNCH_BOUNDS(TPR > 256 ? TPR : 256) void gg_layernorm_fwd_kernel(GgLnParams p) {
    typedef typename GgElt<T>::type E;
    constexpr int RPB = TPR > 256 ? 1 : 256 / TPR;
    GG_SHARED float sRed[2][16];
    const int t = threadIdx.x % TPR;
    const long long row0 = (long long)blockIdx.x * RPB + threadIdx.x / TPR;
    const long long row = row0 < p.rows ? row0 : p.rows - 1;          // (every lane takes part in the sums)
    const E* xr = (const E*)p.x + row * p.ldx;
    GgRaw8<T> raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * 8;
        raw[i] = gg_raw8_load<T>(xr + (c < p.C ? c : 0), p.C - c);
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) s += gg_raw8_get<T>(raw[i], e);
    const float mean = gg_ln_row_sum<TPR>(s, sRed[0]) / (float)p.C;
    float s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float d = gg_raw8_get<T>(raw[i], e) - mean;
            s2 += c + e < p.C ? d * d : 0.f;
        }
    }
    const float rstd = 1.f / sqrtf(gg_ln_row_sum<TPR>(s2, sRed[1]) / (float)p.C + p.eps);
    if (row0 >= p.rows) return;
    if (t == 0 && p.mean) {
        p.mean[row] = mean;
        p.rstd[row] = rstd;
    }
    E* yr = (E*)p.y + row * p.C;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * 8, n = p.C - c;
        if (n <= 0) break;
        const GgRaw8<GG_ELT_F32> w = gg_raw8_load<GG_ELT_F32>(p.w + c, n);
        GgRaw8<GG_ELT_F32> b = {};
        if (p.b) b = gg_raw8_load<GG_ELT_F32>(p.b + c, n);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            v[e] = gg_fmaf((gg_raw8_get<T>(raw[i], e) - mean) * rstd, gg_raw8_get<GG_ELT_F32>(w, e), gg_raw8_get<GG_ELT_F32>(b, e));
        gg_raw8_set<T>(raw[i], v);
        gg_raw8_store<T>(yr + c, raw[i], n);
    }
}

template <int T, int TPR, int NV>
GG_KERNEL GG_LAUNCH_BOUNDS(TPR > 256 ? TPR : 256) void gg_layernorm_bwd_kernel(GgLnParams p) {
    typedef typename GgElt<T>::type E;
    constexpr int RPB = TPR > 256 ? 1 : 256 / TPR;
    GG_SHARED float sRed[2][2][16];                                   // (two sets: a row's sums may be read while the next row's are written)
    GG_SHARED float sAcc[RPB > 1 ? 3 * (TPR < 64 ? TPR : 64) * NV * 8 : 1];
    const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    float w[NV][8], dw[NV][8], db[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * 8;
        const GgRaw8<GG_ELT_F32> wr = gg_raw8_load<GG_ELT_F32>(p.w + (c < p.C ? c : 0), p.C - c);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            w[i][e] = gg_raw8_get<GG_ELT_F32>(wr, e);
            dw[i][e] = db[i][e] = 0.f;
        }
    }
    int odd = 0;
    const float inv = 1.f / (float)p.C;
    for (long long base = (long long)blockIdx.x * RPB; base < p.rows; base += (long long)gridDim.x * RPB, odd ^= 1) {
        const bool in = base + sub < p.rows;
        const long long row = in ? base + sub : p.rows - 1;
        const E* xr = (const E*)p.x + row * p.ldx;
        const E* gr = (const E*)p.dy + row * p.ldy;
        GgRaw8<T> x[NV], g[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * 8, cc = c < p.C ? c : 0;
            x[i] = gg_raw8_load<T>(xr + cc, p.C - c);
            g[i] = gg_raw8_load<T>(gr + cc, p.C - c);
        }
        const float mean = p.mean[row], rstd = p.rstd[row];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float gw = gg_raw8_get<T>(g[i], e) * w[i][e];
                s1 += gw;
                s2 = gg_fmaf(gw, (gg_raw8_get<T>(x[i], e) - mean) * rstd, s2);
            }
        s1 = gg_ln_row_sum<TPR>(s1, sRed[odd][0]) * inv;
        s2 = gg_ln_row_sum<TPR>(s2, sRed[odd][1]) * inv;
        if (!in) continue;      // (the last rows' tail: the lanes come back together at the sums below)
        E* dr = (E*)p.y + row * p.C;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * 8, n = p.C - c;
            if (n <= 0) break;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float gv = gg_raw8_get<T>(g[i], e), xh = (gg_raw8_get<T>(x[i], e) - mean) * rstd;
                v[e] = rstd * (gv * w[i][e] - s1 - xh * s2);
                dw[i][e] = gg_fmaf(gv, xh, dw[i][e]);
                db[i][e] += gv;
            }
            GgRaw8<T> o;
            gg_raw8_set<T>(o, v);
            gg_raw8_store<T>(dr + c, o, n);
        }
    }
    // the workgroup's rows added up: lanes of one wave that share columns first, then the waves in order
    if constexpr (TPR < 64) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                for (int o = TPR; o < 64; o <<= 1) {
                    dw[i][e] += gg_shfl_xor(dw[i][e], o);
                    db[i][e] += gg_shfl_xor(db[i][e], o);
                }
    }
    if constexpr (RPB > 1) {
        constexpr int COLS = (TPR < 64 ? TPR : 64) * NV * 8;
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
        for (int which = 0; which < 2; ++which) {
            float (*acc)[8] = which ? db : dw;
            gg_sync();
            if (wave && lane < (TPR < 64 ? TPR : 64))
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    for (int e = 0; e < 8; ++e) sAcc[(wave - 1) * COLS + (i * 8 + e) * (TPR < 64 ? TPR : 64) + lane] = acc[i][e];
            gg_sync();
            if (wave == 0 && lane < (TPR < 64 ? TPR : 64))
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    for (int e = 0; e < 8; ++e)
                        for (int k = 0; k < 3; ++k) acc[i][e] += sAcc[k * COLS + (i * 8 + e) * (TPR < 64 ? TPR : 64) + lane];
        }
        if (threadIdx.x >= (TPR < 64 ? TPR : 64)) return;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * 8, n = p.C - c;
        if (n <= 0) break;
        GgRaw8<GG_ELT_F32> o;
        float* row = p.part + (long long)blockIdx.x * 2 * p.C + c;
        gg_raw8_set<GG_ELT_F32>(o, dw[i]);
        gg_raw8_store<GG_ELT_F32>(row, o, n);
        gg_raw8_set<GG_ELT_F32>(o, db[i]);
        gg_raw8_store<GG_ELT_F32>(row + p.C, o, n);
    }
}

// column sums of the [blocks][2 C] partial rows: 32 columns x 32 row strides per workgroup (eight loads in flight a thread, then the
// strides in order)
GG_KERNEL GG_LAUNCH_BOUNDS(1024) void gg_layernorm_finish_kernel(const float* part, float* dw, float* db, int blocks, int C) {
    GG_SHARED float sSum[32][33];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), r0 = threadIdx.x >> 5;
    float s = 0.f;
    if (col < 2 * C) {
#pragma unroll 8
        for (int r = r0; r < blocks; r += 32) s += part[(long long)r * 2 * C + col];
    }
    sSum[r0][threadIdx.x & 31] = s;
    gg_sync();
    // strides of column r0 side by side in one half-wave
    s = sSum[threadIdx.x & 31][r0];
    for (int o = 1; o < 32; o <<= 1) s += gg_shfl_xor(s, o);
    const int out = blockIdx.x * 32 + r0;
    if ((threadIdx.x & 31) == 0 && out < 2 * C) {
        if (out < C) dw[out] = s;
        else if (db) db[out - C] = s;
    }
}

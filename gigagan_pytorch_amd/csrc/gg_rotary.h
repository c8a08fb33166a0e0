// gg_rotary.h — rotary positions with several axes (time, height, width): feature pair i of a head turns by the angle
// position[axis(i)] * freq(i), queries and keys in one pass.
//
//   (a, b) -> (a cos - b sin, a sin + b cos)          the gradient is the same turn by the opposite angle
//
// Pairs are (i, i + pairs) or, interleaved, (2i, 2i + 1); features behind the last pair are copied. The product position * freq is
// taken in fp64, in turns (freq / 2 pi), and only its fraction goes on to sine and cosine in fp32: at position 10^6 an fp32 angle would
// be off by 0.06 rad. A workgroup computes the sines of its TB tokens once into LDS (a pair's angle is the same for all heads), then its
// threads walk the tokens' features in memory order, eight pairs each: bound by reading and writing q and k once. 57600 tokens, 24 + 8 heads
// of 128, fp16: 169 us (5.6 TB/s); 32 maps of 32 x 32, 8 + 8 heads of 64, bf16: 28 us (4.8 TB/s); medians.
#pragma once
#include "gg_element.h"

#define GG_ROT_MAX_PAIRS 128
#define GG_ROT_LDS_PAIRS 1024       // pairs x tokens of a workgroup

struct GgRotParams {
    const void* x[2];               // q, k (k null: h[1] = 0)
    void* y[2];                     // dense [B][n][h][d]
    long long sb[2], sh[2], sn[2];  // element strides of x: batch, head, token
    int h[2];
    const void* pos;
    long long pb, pn, pa;           // element strides of the positions: batch, token, axis
    int pos_type;                   // 0 int32, 1 int64, 2 fp32
    int B, n, d, pairs, tb;
    int interleaved, inverse;
    double turns[GG_ROT_MAX_PAIRS];
    unsigned char axis[GG_ROT_MAX_PAIRS];
};

template <int T>
GG_KERNEL GG_LAUNCH_BOUNDS(256) void gg_rotary_kernel(GgRotParams p) {
    typedef typename GgElt<T>::type E;
    GG_SHARED __attribute__((aligned(16))) float sCos[GG_ROT_LDS_PAIRS];
    GG_SHARED __attribute__((aligned(16))) float sSin[GG_ROT_LDS_PAIRS];
    const GgRotParams* kp = gg_late_params(p);          // (the two tables are indexed per lane: read where they lie)
    const int tiles = (p.n - 1) / p.tb + 1;
    const int b = blockIdx.x / tiles;
    const int t0 = (blockIdx.x - b * tiles) * p.tb;
    const int nt = p.n - t0 < p.tb ? p.n - t0 : p.tb;
    for (int i = threadIdx.x; i < nt * p.pairs; i += 256) {
        const int tok = i / p.pairs, pr = i - tok * p.pairs;
        const long long at = b * p.pb + (long long)(t0 + tok) * p.pn + kp->axis[pr] * p.pa;
        const double pos = p.pos_type == 0 ? (double)((const int*)p.pos)[at]
                         : p.pos_type == 1 ? (double)((const long long*)p.pos)[at] : (double)((const float*)p.pos)[at];
        const double turn = pos * kp->turns[pr];
        const float frac = (float)(turn - rint(turn));              // -1/2 .. 1/2
        float s, c;
        gg_sincospi(2.f * frac, &s, &c);
        sCos[i] = c;
        sSin[i] = p.inverse ? -s : s;
    }
    gg_sync();
    const int rot = (p.pairs + 7) / 8, rest = p.d - 2 * p.pairs, per = rot + (rest + 7) / 8;
    const int heads = p.h[0] + p.h[1];
    const int items = nt * heads * per;
    for (int i = threadIdx.x; i < items; i += 256) {
        const int th = i / per, ch = i - th * per;
        const int tok = th / heads;
        int hd = th - tok * heads;
        const int which = hd >= p.h[0];
        if (which) hd -= p.h[0];
        const E* xr = (const E*)p.x[which] + b * p.sb[which] + hd * p.sh[which] + (long long)(t0 + tok) * p.sn[which];
        E* yr = (E*)p.y[which] + (((long long)b * p.n + t0 + tok) * p.h[which] + hd) * p.d;
        if (ch >= rot) {
            const int c = 2 * p.pairs + (ch - rot) * 8, left = p.d - c;
            gg_raw8_store<T>(yr + c, gg_raw8_load<T>(xr + c, left), left);
            continue;
        }
        const int i0 = ch * 8, np = p.pairs - i0 < 8 ? p.pairs - i0 : 8;
        float u[8], v[8], cs[8], sn[8];
        for (int e = 0; e < 8; ++e) {
            const int at = tok * p.pairs + i0 + (e < np ? e : 0);
            cs[e] = sCos[at];
            sn[e] = sSin[at];
        }
        const int ca = p.interleaved ? 2 * i0 : i0, cb = p.interleaved ? ca + 8 : i0 + p.pairs;
        const int na = p.interleaved ? 2 * np : np, nb = p.interleaved ? 2 * np - 8 : np;
        GgRaw8<T> ra = gg_raw8_load<T>(xr + ca, na), rb = gg_raw8_load<T>(xr + (nb > 0 ? cb : ca), nb);
        for (int e = 0; e < 8; ++e) { u[e] = gg_raw8_get<T>(ra, e); v[e] = gg_raw8_get<T>(rb, e); }
        if (p.interleaved) {
            for (int e = 0; e < 4; ++e) {
                const float a = u[2 * e], c = u[2 * e + 1], a2 = v[2 * e], c2 = v[2 * e + 1];
                u[2 * e] = a * cs[e] - c * sn[e];
                u[2 * e + 1] = a * sn[e] + c * cs[e];
                v[2 * e] = a2 * cs[4 + e] - c2 * sn[4 + e];
                v[2 * e + 1] = a2 * sn[4 + e] + c2 * cs[4 + e];
            }
        } else {
            for (int e = 0; e < 8; ++e) {
                const float a = u[e], c = v[e];
                u[e] = a * cs[e] - c * sn[e];
                v[e] = a * sn[e] + c * cs[e];
            }
        }
        gg_raw8_set<T>(ra, u);
        gg_raw8_set<T>(rb, v);
        gg_raw8_store<T>(yr + ca, ra, na);
        if (nb > 0) gg_raw8_store<T>(yr + cb, rb, nb);
    }
}

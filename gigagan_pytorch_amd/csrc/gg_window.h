// gg_window.h — attention with a sliding window and sinks, forward, backward and its few-query form.
//
// Query i of batch item b sits at position p = len_b - n + i (the queries are the last n of the sequence's len_b <= m keys) and sees
//     key j   when   j < len_b,   j <= p + right,   j >= p - left or j < sinks,   keep[b][j]
// (a query at a negative position is padding and sees nothing).
//     o_i = sum_j P_ij v_j,   P = softmax over the seen keys of scale q_i.k_j;   a query that sees no key gets zeros and no gradient.
//     backward: D_i = dO_i.o_i,  dS_ij = P_ij (dO_i.v_j - D_i),  dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,  dv_j = sum_i P_ij dO_i
//
// Grouped heads: g = h / hk query heads read one key head. The kernels' ROWS are the (token, head of the group) pairs of one (batch,
// key head), r = token * g + head, so a tile of rows spans 1/g of the tokens a tile of one head would: K and V are read once for the
// whole group, fewer tiles are cut by the window's edges, and dk / dv of a shared head are one sum in registers.
//
// Contractions are issued transposed (S^T = K Q^T, O^T = V^T P^T; v_mfma_f32_32x32x16): a lane owns one query (backward dk / dv: one key)
// and 16 scores of it, the softmax statistics are lane-local plus one exchange with lane ^ 32, and the packed probabilities are the next
// contraction's B operand as they lie, with the reduction slots re-labelled (slot (c, hi, e) <-> row 16c + 4hi + (e & 3) + 8(e >> 2)).
// Key tiles outside the window are not visited; the tiles a wave sees entirely take no mask arithmetic.
//
// NaN and infinities. Where a row does not see a key its probability is an exact zero, but zero times a NaN in the shared tile is NaN.
// Keys that no row of the workgroup sees are staged as zeros. For the rest every kernel looks at its own result once, at the end: if
// something in it is not finite, the tiles are walked a second time with every non-finite vector taken out of the tile and accounted
// for by itself, key by key, for the rows that see it. Finite inputs never take the second walk.
#pragma once
#include "gg_element.h"

#define GGW_NONE 0x20000000          // "no bound" of a window side, and (negated, doubled) the position of a row that is not there
#define GGW_LOG2E 1.4426950408889634f
#define GGW_TAU 8.0f                 // the running maximum moves when a score exceeds it by 2^8: fewer rescales of the output, P <= 2^8

struct GgWinParams {
    const unsigned short *q, *k, *v, *d_o;
    unsigned short *o, *dq, *dk, *dv;       // dense: o, dq [B][n][h][D]; dk, dv [B][m][hk][D]
    float* lse;                             // [B*hk][n*g]: log2 of the row's sum of 2^(scale log2e s); +inf for a row that sees nothing
    float* dvec;                            // [B*hk][n*g]: D_i
    long long qb, qh, qn, kb, kh, kn, vb, vh, vn, gb, gh, gn;      // element strides of q, k, v, dO
    const int* lengths;                     // [B] or null (= m)
    const unsigned char* keep;              // [B][m], batch stride keep_b, or null
    long long keep_b;
    float* part_o;                          // key splits: [split][B*hk][n*g][D] and [split][B*hk][n*g][2] (m, l)
    float* part_ml;
    int B, n, m, h, hk, g;
    int left, right, sinks;
    float scale;
    int splits;
    int row_tiles;                          // row (dk / dv: key) tiles per (batch, key head)
    int sink_tiles, sink_chunks;            // dk / dv: key tiles that hold sinks, and the row chunks each of them is split into
};

// ---- shared pieces -----------------------------------------------------------------------------------------------

template <int T>
GG_DEVICE f32x16 ggw_mfma(u16x8 a, u16x8 b, f32x16 c) {
    if constexpr (T == GG_ELT_BF16) return gg_mfma_32x32x16_bf16(a, b, c);
    else return gg_mfma_32x32x16_f16(a, b, c);
}
// registers 8c .. 8c + 7 of a result, rounded to 16 bits: the B operand of the follow-up contraction (P and dS are rounded to the operands'
// type for the matrix pipe, as any 16-bit attention does; their sums stay fp32)
template <int T>
GG_DEVICE u16x8 ggw_pack8(const f32x16& v, int c) {
    u16x8 f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = gg_elt<T>(v[8 * c + e]);
    return f;
}
// eight 16-bit values of which one is NaN or infinite
template <int T>
GG_DEVICE bool ggw_bad8(u16x8 x) {
    constexpr unsigned short E = T == GG_ELT_BF16 ? 0x7f80 : 0x7c00;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) bad = bad || (x[e] & E) == E;
    return bad;
}
template <int N>
GG_DEVICE bool ggw_not_finite(const f32x16* v) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s = gg_fmaf(v[i][r], 0.f, s);
    return s != s;
}
template <int D> struct GgwTile { static constexpr int PITCH = 2 * D + 32; static constexpr int BYTES = 64 * PITCH; };

// A operand, rows as they lie: lane l -> row row0 + (l & 31), features kk*16 + 8(l >> 5) + 0..7
template <int D>
GG_DEVICE u16x8 ggw_frag(const char* tile, int row0, int kk, int lane) {
    return *(const u16x8*)(tile + (row0 + (lane & 31)) * GgwTile<D>::PITCH + (kk * 16 + 8 * (lane >> 5)) * 2);
}
// A operand of the tile's transpose: lane l -> feature d0 + (l & 31), slots (hi, e) <-> rows rb + 4hi + (e & 3) + 8(e >> 2)
template <int D>
GG_DEVICE u16x8 ggw_frag_tr(const char* tile, int d0, int rb, int lane) {
    const int i = lane & 15, gq = lane >> 4;
    const char* p = tile + (rb + 4 * (gq >> 1) + (i >> 2)) * GgwTile<D>::PITCH + (d0 + (gq & 1) * 16 + 4 * (i & 3)) * 2;
    const u16x4 a = gg_lds_read_tr16((const bf16_t*)p), b = gg_lds_read_tr16((const bf16_t*)(p + 8 * GgwTile<D>::PITCH));
    return u16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// consecutive items (tiles of one (batch, key head), which share keys) go to one XCD and its L2: the dispatcher deals workgroups out to
// the eight XCDs in turn
GG_DEVICE int ggw_item() {
    const int total = (int)gridDim.x, lin = (int)blockIdx.x;
    const int xq = total >> 3, xr = total & 7, xcd = lin & 7, pos = lin >> 3;
    return (xcd < xr ? xcd * (xq + 1) : xr * (xq + 1) + (xcd - xr) * xq) + pos;
}

GG_DEVICE int ggw_len(const GgWinParams& p, int b) {
    if (!p.lengths) return p.m;
    const int v = p.lengths[b];
    return v < 0 ? 0 : (v > p.m ? p.m : v);
}

// the keys that the rows of tokens t0 .. t1 see between them, in tiles of TK keys: first the `st` tiles that hold sinks, then the window's
struct GgwRange {
    int klo, khi;       // window keys klo .. khi
    int st, w0, nt;     // sink tiles, the window's first tile behind them, tiles in all
};
template <int TK>
GG_DEVICE GgwRange ggw_range(const GgWinParams& p, int len, int t0, int t1) {
    GgwRange r = {0, -1, 0, 0, 0};
    const int shift = len - p.n;
    const int plo = t0 + shift < 0 ? 0 : t0 + shift, phi = t1 + shift;
    if (phi < 0 || phi < plo) return r;
    r.khi = phi + p.right < len - 1 ? phi + p.right : len - 1;
    r.klo = plo - p.left > 0 ? plo - p.left : 0;
    const int s_hi = p.sinks - 1 < r.khi ? p.sinks - 1 : r.khi;
    r.st = s_hi >= 0 ? s_hi / TK + 1 : 0;
    const int wl = r.klo / TK, wh = r.khi / TK;
    r.w0 = wl > r.st ? wl : r.st;
    r.nt = r.st + (wh >= r.w0 ? wh - r.w0 + 1 : 0);
    return r;
}
GG_DEVICE int ggw_tile_at(const GgwRange& r, int i) { return i < r.st ? i : r.w0 + i - r.st; }
// a key that some row of the range sees (key mask apart): others are staged as zeros, so that what lies there (stale cache slots,
// NaN padding) never meets a zero probability in a product
GG_DEVICE bool ggw_in_range(const GgwRange& r, int sinks, int j) { return j <= r.khi && (j >= r.klo || j < sinks); }

// a 64-row tile on its way from memory to LDS: 256 threads, 16 bytes each per step
template <int D> struct GgwRegs { u16x8 v[D / 32]; };
template <int D>
GG_DEVICE void ggw_store_tile(const GgwRegs<D>& r, char* tile) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const int v = threadIdx.x + 256 * i, row = v / (D / 8), c8 = v % (D / 8);
        *(u16x8*)(tile + row * GgwTile<D>::PITCH + c8 * 16) = r.v[i];
    }
}
// the second walk: vectors with a NaN or an infinity are taken out and marked, bad[row][vector]
template <int T, int D>
GG_DEVICE void ggw_take_bad(GgwRegs<D>& r, unsigned char* bad, bool add) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const bool b = ggw_bad8<T>(r.v[i]);
        if (b) r.v[i] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
        const int at = threadIdx.x + 256 * i;               // = row * (D / 8) + vector
        bad[at] = (unsigned char)((add ? bad[at] : 0) | b);
    }
}
template <int D>
GG_DEVICE bool ggw_any_bad(const unsigned char* bad, int row) {
    unsigned any = 0;
#pragma unroll
    for (int c = 0; c < D / 8; c += 4) any |= *(const unsigned*)(bad + row * (D / 8) + c);
    return any != 0;
}
// forward: what the vectors that were taken out of a key tile give the rows that see their keys. K and V are read where they lie.
template <int T, int D, class See>
GG_DEVICE void ggw_add_bad(f32x16* ot, const unsigned char* bad, int tk, int j0, const unsigned short* kb, long long kn, const unsigned short* vb,
                           long long vn, const u16x8* qf, float a2, float m, int hi, See see) {
    for (int jr = 0; jr < tk; ++jr) {
        if (!ggw_any_bad<D>(bad, jr)) continue;             // (workgroup- or wave-uniform; a marked key lies inside the range)
        const int j = j0 + jr;
        float s = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            const u16x8 kv = *(const u16x8*)(kb + (long long)j * kn + kk * 16 + 8 * hi);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = gg_fmaf(gg_elt_f<T>(qf[kk][e]), gg_elt_f<T>(kv[e]), s);
        }
        s = gg_sum_xor32(s);
        const float pj = see(j, jr) ? gg_exp2f(gg_fmaf(s, a2, -m)) : 0.f;
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
            if (bad[jr * (D / 8) + c]) {
                const u16x4 v4 = *(const u16x4*)(vb + (long long)j * vn + c * 8 + 4 * hi);
#pragma unroll
                for (int e = 0; e < 4; ++e) ot[c / 4][4 * (c % 4) + e] += pj > 0.f ? pj * gg_elt_f<T>(v4[e]) : 0.f;
            }
    }
}
// keys j0 .. j0 + 63 of one (batch, key head)
template <int D>
GG_DEVICE GgwRegs<D> ggw_load_keys(const unsigned short* base, long long stride, int j0, const GgwRange& rg, int sinks, const unsigned char* keep) {
    GgwRegs<D> r;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const int v = threadIdx.x + 256 * i, j = j0 + v / (D / 8), c8 = v % (D / 8);
        r.v[i] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
        if (ggw_in_range(rg, sinks, j) && (!keep || keep[j])) r.v[i] = *(const u16x8*)(base + (long long)j * stride + c8 * 8);
    }
    return r;
}

// this lane's row of the tile that starts at row r0, and the wave's 32 rows
struct GgwRow {
    int token, head, pos;       // head within the group
    bool in;                    // the row exists and is not padding
};
GG_DEVICE GgwRow ggw_row(const GgWinParams& p, int r, int len) {
    GgwRow w;
    const int rows = p.n * p.g;
    const int rc = r < rows ? r : rows - 1;
    w.token = (int)((unsigned)rc / (unsigned)p.g);
    w.head = rc - w.token * p.g;
    w.pos = w.token + len - p.n;
    w.in = r < rows && w.pos >= 0;
    return w;
}

// ---- forward -------------------------------------------------------------------------------------------------------
// workgroup: 4 waves x 32 rows, key tiles of 64 staged once for all four, double buffered (one barrier a tile).
// SPLIT: the tiles are dealt out to p.splits workgroups, which leave (m, l, O) for gg_win_join_kernel.
template <int T, int D, bool SPLIT>
GG_KERNEL GG_LAUNCH_BOUNDS(256) void gg_win_fwd_kernel(GgWinParams p) {
    constexpr int KK = D / 16, DB = D / 32;
    GG_SHARED __attribute__((aligned(16))) char sK[2][GgwTile<D>::BYTES];
    GG_SHARED __attribute__((aligned(16))) char sV[2][GgwTile<D>::BYTES];
    GG_SHARED unsigned char sKeep[2][64];
    GG_SHARED __attribute__((aligned(16))) unsigned char sBad[2][64 * (D / 8)];
    GG_SHARED int sAgain;

    const int lane = threadIdx.x & 63, wave = gg_uniform(threadIdx.x >> 6), hi = lane >> 5;
    int item = ggw_item();
    int split = 0;
    if (SPLIT) { split = item % p.splits; item /= p.splits; }
    const int bkv = item / p.row_tiles, tile = item - bkv * p.row_tiles;
    const int b = bkv / p.hk, kvh = bkv - b * p.hk;
    const int rows = p.n * p.g;
    const int len = ggw_len(p, b);
    const int r0 = tile * 128, rl = r0 + 127 < rows - 1 ? r0 + 127 : rows - 1;
    const GgwRange rg = ggw_range<64>(p, len, r0 / p.g, rl / p.g);
    const int ta = SPLIT ? (int)((long long)rg.nt * split / p.splits) : 0, tb = SPLIT ? (int)((long long)rg.nt * (split + 1) / p.splits) : rg.nt;

    const int wr0 = r0 + wave * 32;
    const GgwRow row = ggw_row(p, wr0 + (lane & 31), len);
    const bool whole = wr0 + 31 < rows && wr0 / p.g + len - p.n >= 0;          // (wave-uniform) 32 rows, none of them padding
    const int wlo = wr0 / p.g + len - p.n, whi = (wr0 + 31 < rows ? wr0 + 31 : rows - 1) / p.g + len - p.n;
    const int lo = row.pos - p.left, hij = row.in ? (row.pos + p.right < len - 1 ? row.pos + p.right : len - 1) : -1;
    const int whij = whi + p.right < len - 1 ? whi + p.right : len - 1, wlij = wlo + p.right < len - 1 ? wlo + p.right : len - 1;

    const unsigned short* kb = p.k + b * p.kb + kvh * p.kh;
    const unsigned short* vb = p.v + b * p.vb + kvh * p.vh;
    const unsigned char* keep = p.keep ? p.keep + b * p.keep_b : nullptr;
    u16x8 qf[KK];
    {
        const unsigned short* qr = p.q + b * p.qb + (long long)(kvh * p.g + row.head) * p.qh + (long long)row.token * p.qn + 8 * hi;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) qf[kk] = *(const u16x8*)(qr + kk * 16);
    }
    const float a2 = p.scale * GGW_LOG2E;
    float m, l;
    f32x16 ot[DB];

    GgwRegs<D> rk, rv;
    unsigned char rkeep = 1;
    auto load = [&](int i) {
        const int j0 = ggw_tile_at(rg, i) * 64;
        rk = ggw_load_keys<D>(kb, p.kn, j0, rg, p.sinks, keep);
        rv = ggw_load_keys<D>(vb, p.vn, j0, rg, p.sinks, keep);
        if (keep && threadIdx.x < 64) rkeep = j0 + (int)threadIdx.x < len ? keep[j0 + threadIdx.x] : 0;
    };
    bool again = false;             // the second walk (workgroup-uniform)
    auto store = [&](int buf) {
        if (again) ggw_take_bad<T, D>(rv, sBad[buf], false);
        ggw_store_tile<D>(rk, sK[buf]);
        ggw_store_tile<D>(rv, sV[buf]);
        if (keep && threadIdx.x < 64) sKeep[buf][threadIdx.x] = rkeep;
    };
walk:
    m = -1.0e30f;
    l = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) ot[db][r] = 0.f;
    if (ta < tb) {
        load(ta);
        store(0);
        if (ta + 1 < tb) load(ta + 1);
    }
    if (threadIdx.x == 0) sAgain = 0;
    gg_sync();
    for (int i = ta, buf = 0; i < tb; ++i, buf ^= 1) {
        if (i + 1 < tb) {
            store(buf ^ 1);         // (free since the barrier that ended the last tile)
            if (i + 2 < tb) load(i + 2);
        }
        const int j0 = ggw_tile_at(rg, i) * 64;
        if (j0 <= whij && (j0 + 63 >= wlo - p.left || j0 < p.sinks) && wr0 < rows) {
            f32x16 st[2];
#pragma unroll
            for (int jb = 0; jb < 2; ++jb) {
#pragma unroll
                for (int r = 0; r < 16; ++r) st[jb][r] = 0.f;
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) st[jb] = ggw_mfma<T>(ggw_frag<D>(sK[buf], jb * 32, kk, lane), qf[kk], st[jb]);
            }
            if (!(whole && !keep && j0 + 63 <= wlij && (j0 >= whi - p.left || j0 + 63 < p.sinks))) {
                unsigned long long bits = ~0ull;
                if (keep) bits = gg_ballot(sKeep[buf][lane] != 0);
                bits >>= 4 * hi;
#pragma unroll
                for (int jb = 0; jb < 2; ++jb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int jr = jb * 32 + (r & 3) + 8 * (r >> 2), j = j0 + jr + 4 * hi;
                        const bool see = j <= hij && (j >= lo || j < p.sinks) && ((bits >> jr) & 1);
                        st[jb][r] = see ? st[jb][r] : -__builtin_inff();
                    }
            }
            float mx = -__builtin_inff();
#pragma unroll
            for (int jb = 0; jb < 2; ++jb)
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[jb][r]);
            mx = gg_max_xor32(mx) * a2;
            if (gg_wave_any(mx > m + GGW_TAU)) {
                const float mn = fmaxf(m, mx), corr = gg_exp2f(m - mn);
                l *= corr;
                m = mn;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int r = 0; r < 16; ++r) ot[db][r] *= corr;
            }
            float sum = 0.f;
#pragma unroll
            for (int jb = 0; jb < 2; ++jb)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    st[jb][r] = gg_exp2f(gg_fmaf(st[jb][r], a2, -m));
                    sum += st[jb][r];
                }
            l += sum;
#pragma unroll
            for (int jb = 0; jb < 2; ++jb)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const u16x8 pf = ggw_pack8<T>(st[jb], c);
#pragma unroll
                    for (int db = 0; db < DB; ++db) ot[db] = ggw_mfma<T>(ggw_frag_tr<D>(sV[buf], db * 32, jb * 32 + 16 * c, lane), pf, ot[db]);
                }
            if (again)
                ggw_add_bad<T, D>(ot, sBad[buf], 64, j0, kb, p.kn, vb, p.vn, qf, a2, m, hi, [&](int j, int jr) {
                    return j <= hij && (j >= lo || j < p.sinks) && (!keep || sKeep[buf][jr]);
                });
        }
        gg_sync();
    }
    if (!again) {
        if (ggw_not_finite<DB>(ot)) sAgain = 1;
        gg_sync();
        if (sAgain) {
            again = true;
            gg_sync();
            goto walk;
        }
    }
    l = gg_sum_xor32(l);
    const int r = wr0 + (lane & 31);
    if (r >= rows) return;
    const long long at = (long long)bkv * rows + r;
    if (SPLIT) {
        const long long sp = (long long)split * p.B * p.hk * rows + at;
        float* po = p.part_o + sp * D;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int gq = 0; gq < 4; ++gq)
                *(f32x4*)(po + db * 32 + 8 * gq + 4 * hi) = f32x4{ot[db][4 * gq], ot[db][4 * gq + 1], ot[db][4 * gq + 2], ot[db][4 * gq + 3]};
        if (hi == 0) { p.part_ml[2 * sp] = m; p.part_ml[2 * sp + 1] = l; }
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    unsigned short* orow = p.o + (((long long)b * p.n + row.token) * p.h + kvh * p.g + row.head) * D;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int gq = 0; gq < 4; ++gq) {
            u16x4 o4;
#pragma unroll
            for (int e = 0; e < 4; ++e) o4[e] = gg_elt<T>(ot[db][4 * gq + e] * inv);
            *(u16x4*)(orow + db * 32 + 8 * gq + 4 * hi) = o4;
        }
    if (hi == 0 && p.lse) p.lse[at] = l == 0.f ? __builtin_inff() : m + log2f(l);
}

// ---- forward with few rows ------------------------------------------------------------------------------------------
// One new token: a handful of rows against a long cache - bound by reading K and V once. The four waves share the 32 rows and take key
// tiles of 32 in turn, each on its own: K goes from memory straight into the score product's operand registers, V through a wave-private
// LDS tile (the transpose read), no barrier in the loop; the waves' (m, l, O) are joined in LDS at the end, the splits' by
// gg_win_join_kernel.
template <int T, int D>
GG_KERNEL GG_LAUNCH_BOUNDS(256) void gg_win_few_kernel(GgWinParams p) {
    constexpr int KK = D / 16, DB = D / 32, PITCH = GgwTile<D>::PITCH;
    GG_SHARED __attribute__((aligned(16))) char sV[4][32 * PITCH];
    GG_SHARED __attribute__((aligned(16))) unsigned char sBad[4][32 * (D / 8)];
    GG_SHARED float sM[4][32], sL[4][32];
    GG_SHARED __attribute__((aligned(16))) float sO[32][D + 4];

    const int lane = threadIdx.x & 63, wave = gg_uniform(threadIdx.x >> 6), hi = lane >> 5;
    int item = ggw_item();
    const int split = item % p.splits;
    item /= p.splits;
    const int bkv = item / p.row_tiles, tile = item - bkv * p.row_tiles;
    const int b = bkv / p.hk, kvh = bkv - b * p.hk;
    const int rows = p.n * p.g;
    const int len = ggw_len(p, b);
    const int r0 = tile * 32, rl = r0 + 31 < rows - 1 ? r0 + 31 : rows - 1;
    const GgwRange rg = ggw_range<32>(p, len, r0 / p.g, rl / p.g);
    const int ta = (int)((long long)rg.nt * split / p.splits), tb = (int)((long long)rg.nt * (split + 1) / p.splits);
    const GgwRow row = ggw_row(p, r0 + (lane & 31), len);
    const int lo = row.pos - p.left, hij = row.in ? (row.pos + p.right < len - 1 ? row.pos + p.right : len - 1) : -1;
    const unsigned short* kb = p.k + b * p.kb + kvh * p.kh;
    const unsigned short* vb = p.v + b * p.vb + kvh * p.vh;
    const unsigned char* keep = p.keep ? p.keep + b * p.keep_b : nullptr;
    u16x8 qf[KK];
    {
        const unsigned short* qr = p.q + b * p.qb + (long long)(kvh * p.g + row.head) * p.qh + (long long)row.token * p.qn + 8 * hi;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) qf[kk] = *(const u16x8*)(qr + kk * 16);
    }
    const float a2 = p.scale * GGW_LOG2E;
    float m, l;
    f32x16 ot[DB];

    u16x8 kf[KK], vr[D / 16];
    bool kept = true;
    auto load = [&](int i) {
        const int j0 = ggw_tile_at(rg, i) * 32, j = j0 + (lane & 31);
        const bool ok = j <= rg.khi;                                            // (0 <= khi < len: the clamped row exists)
        const unsigned short* kr = kb + (long long)(ok ? j : rg.khi) * p.kn + 8 * hi;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) kf[kk] = *(const u16x8*)(kr + kk * 16);
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
            const int v = lane + 64 * s, jv = j0 + v / (D / 8), c8 = v % (D / 8);
            vr[s] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
            if (ggw_in_range(rg, p.sinks, jv) && (!keep || keep[jv])) vr[s] = *(const u16x8*)(vb + (long long)jv * p.vn + c8 * 8);
        }
        if (keep) kept = ok && keep[j];
    };
    bool again = false;             // the second walk (wave-uniform)
walk:
    m = -1.0e30f;
    l = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) ot[db][r] = 0.f;
    if (ta + wave < tb) load(ta + wave);
    for (int i = ta + wave; i < tb; i += 4) {
        const int j0 = ggw_tile_at(rg, i) * 32;
        gg_wave_sync();
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
            const int v = lane + 64 * s;
            if (again) {
                const bool bad = ggw_bad8<T>(vr[s]);
                if (bad) vr[s] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
                sBad[wave][v] = bad;
            }
            *(u16x8*)(sV[wave] + (v / (D / 8)) * PITCH + (v % (D / 8)) * 16) = vr[s];
        }
        gg_wave_sync();
        f32x16 st;
#pragma unroll
        for (int r = 0; r < 16; ++r) st[r] = 0.f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) st = ggw_mfma<T>(kf[kk], qf[kk], st);
        unsigned bits = 0xffffffffu;
        if (keep) bits = (unsigned)gg_ballot(kept);
        bits >>= 4 * hi;
        if (i + 4 < tb) load(i + 4);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int jr = (r & 3) + 8 * (r >> 2), j = j0 + jr + 4 * hi;
            const bool see = j <= hij && (j >= lo || j < p.sinks) && ((bits >> jr) & 1);
            st[r] = see ? st[r] : -__builtin_inff();
        }
        float mx = -__builtin_inff();
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[r]);
        mx = gg_max_xor32(mx) * a2;
        if (gg_wave_any(mx > m + GGW_TAU)) {
            const float mn = fmaxf(m, mx), corr = gg_exp2f(m - mn);
            l *= corr;
            m = mn;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) ot[db][r] *= corr;
        }
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            st[r] = gg_exp2f(gg_fmaf(st[r], a2, -m));
            sum += st[r];
        }
        l += sum;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const u16x8 pf = ggw_pack8<T>(st, c);
#pragma unroll
            for (int db = 0; db < DB; ++db) ot[db] = ggw_mfma<T>(ggw_frag_tr<D>(sV[wave], db * 32, 16 * c, lane), pf, ot[db]);
        }
        if (again)
            ggw_add_bad<T, D>(ot, sBad[wave], 32, j0, kb, p.kn, vb, p.vn, qf, a2, m, hi, [&](int j, int jr) {
                (void)jr;
                return j <= hij && (j >= lo || j < p.sinks) && (!keep || keep[j]);
            });
    }
    if (!again && gg_wave_any(ggw_not_finite<DB>(ot))) {
        again = true;
        goto walk;
    }
    l = gg_sum_xor32(l);
    if (hi == 0) { sM[wave][lane] = m; sL[wave][lane] = l; }
    gg_sync();
    const int q = lane & 31;
    float top = sM[0][q];
    for (int w = 1; w < 4; ++w) top = fmaxf(top, sM[w][q]);
    const float f = gg_exp2f(m - top);
    for (int w = 0; w < 4; ++w) {
        if (wave == w)
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int gq = 0; gq < 4; ++gq) {
                    float* at = &sO[q][db * 32 + 8 * gq + 4 * hi];
                    f32x4 x = {ot[db][4 * gq] * f, ot[db][4 * gq + 1] * f, ot[db][4 * gq + 2] * f, ot[db][4 * gq + 3] * f};
                    if (w) x += *(const f32x4*)at;
                    *(f32x4*)at = x;
                }
        gg_sync();
    }
    // 32 rows x D / 4 quads over the workgroup
    for (int i = threadIdx.x; i < 32 * (D / 4); i += 256) {
        const int rr = i / (D / 4), d = (i % (D / 4)) * 4, r = r0 + rr;
        if (r >= rows) break;
        float mt = sM[0][rr], lt = 0.f;
        for (int w = 1; w < 4; ++w) mt = fmaxf(mt, sM[w][rr]);
        for (int w = 0; w < 4; ++w) lt += sL[w][rr] * gg_exp2f(sM[w][rr] - mt);
        const f32x4 x = *(const f32x4*)&sO[rr][d];
        const long long at = (long long)bkv * rows + r;
        if (p.splits > 1) {
            const long long sp = (long long)split * p.B * p.hk * rows + at;
            *(f32x4*)(p.part_o + sp * D + d) = x;
            if (d == 0) { p.part_ml[2 * sp] = mt; p.part_ml[2 * sp + 1] = lt; }
        } else {
            const float inv = lt == 0.f ? 0.f : 1.f / lt;
            const int token = (int)((unsigned)r / (unsigned)p.g), head = r - token * p.g;
            u16x4 o4;
#pragma unroll
            for (int e = 0; e < 4; ++e) o4[e] = gg_elt<T>(x[e] * inv);
            *(u16x4*)(p.o + (((long long)b * p.n + token) * p.h + kvh * p.g + head) * D + d) = o4;
            if (d == 0 && p.lse) p.lse[at] = lt == 0.f ? __builtin_inff() : mt + log2f(lt);
        }
    }
}

// the splits' (m, l, O) of a row joined: four features a thread
template <int T, int D>
GG_KERNEL GG_LAUNCH_BOUNDS(256) void gg_win_join_kernel(GgWinParams p) {
    const int rows = p.n * p.g;
    const long long all = (long long)p.B * p.hk * rows;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, at = i / (D / 4);
    const int d = (int)(i % (D / 4)) * 4;
    if (at >= all) return;
    float top = -1.0e30f;
#pragma unroll 8
    for (int s = 0; s < p.splits; ++s) top = fmaxf(top, p.part_ml[2 * (s * all + at)]);
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
#pragma unroll 8
    for (int s = 0; s < p.splits; ++s) {
        const float f = gg_exp2f(p.part_ml[2 * (s * all + at)] - top);
        l += f * p.part_ml[2 * (s * all + at) + 1];
        x += f * *(const f32x4*)(p.part_o + (s * all + at) * D + d);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int bkv = (int)(at / rows), r = (int)(at - (long long)bkv * rows);
    const int b = bkv / p.hk, kvh = bkv - b * p.hk, token = r / p.g, head = r - token * p.g;
    u16x4 o4;
#pragma unroll
    for (int e = 0; e < 4; ++e) o4[e] = gg_elt<T>(x[e] * inv);
    *(u16x4*)(p.o + (((long long)b * p.n + token) * p.h + kvh * p.g + head) * D + d) = o4;
    if (d == 0 && p.lse) p.lse[at] = l == 0.f ? __builtin_inff() : top + log2f(l);
}

// ---- backward, part 1: dq and D ---------------------------------------------------------------------------------------
// the forward's mapping: 4 waves x 32 rows, key tiles of 64; K is read as rows (scores) and transposed (dq), V as rows (dP)
template <int T, int D>
GG_KERNEL GG_LAUNCH_BOUNDS(256) void gg_win_dq_kernel(GgWinParams p) {
    constexpr int KK = D / 16, DB = D / 32;
    GG_SHARED __attribute__((aligned(16))) char sK[2][GgwTile<D>::BYTES];
    GG_SHARED __attribute__((aligned(16))) char sV[2][GgwTile<D>::BYTES];
    GG_SHARED unsigned char sKeep[2][64];
    GG_SHARED __attribute__((aligned(16))) unsigned char sBad[2][64 * (D / 8)];
    GG_SHARED int sAgain;

    const int lane = threadIdx.x & 63, wave = gg_uniform(threadIdx.x >> 6), hi = lane >> 5;
    const int item = ggw_item();
    const int bkv = item / p.row_tiles, tile = item - bkv * p.row_tiles;
    const int b = bkv / p.hk, kvh = bkv - b * p.hk;
    const int rows = p.n * p.g;
    const int len = ggw_len(p, b);
    const int r0 = tile * 128, rl = r0 + 127 < rows - 1 ? r0 + 127 : rows - 1;
    const GgwRange rg = ggw_range<64>(p, len, r0 / p.g, rl / p.g);

    const int wr0 = r0 + wave * 32;
    const GgwRow row = ggw_row(p, wr0 + (lane & 31), len);
    const bool whole = wr0 + 31 < rows && wr0 / p.g + len - p.n >= 0;
    const int wlo = wr0 / p.g + len - p.n, whi = (wr0 + 31 < rows ? wr0 + 31 : rows - 1) / p.g + len - p.n;
    const int lo = row.pos - p.left, hij = row.in ? (row.pos + p.right < len - 1 ? row.pos + p.right : len - 1) : -1;
    const int whij = whi + p.right < len - 1 ? whi + p.right : len - 1, wlij = wlo + p.right < len - 1 ? wlo + p.right : len - 1;

    const unsigned short* kb = p.k + b * p.kb + kvh * p.kh;
    const unsigned short* vb = p.v + b * p.vb + kvh * p.vh;
    const unsigned char* keep = p.keep ? p.keep + b * p.keep_b : nullptr;
    const int hq = kvh * p.g + row.head;
    const long long orow = (((long long)b * p.n + row.token) * p.h + hq) * D;
    const int rr = wr0 + (lane & 31);
    const long long at = (long long)bkv * rows + (rr < rows ? rr : rows - 1);
    u16x8 qf[KK], gf[KK];
    float dsum = 0.f;
    {
        const unsigned short* qr = p.q + b * p.qb + hq * p.qh + (long long)row.token * p.qn + 8 * hi;
        const unsigned short* gr = p.d_o + b * p.gb + hq * p.gh + (long long)row.token * p.gn + 8 * hi;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            qf[kk] = *(const u16x8*)(qr + kk * 16);
            gf[kk] = *(const u16x8*)(gr + kk * 16);
            const u16x8 of = *(const u16x8*)(p.o + orow + 8 * hi + kk * 16);
#pragma unroll
            for (int e = 0; e < 8; ++e) dsum += gg_elt_f<T>(gf[kk][e]) * gg_elt_f<T>(of[e]);
        }
    }
    dsum = gg_sum_xor32(dsum);
    const float lse = p.lse[at], a2 = p.scale * GGW_LOG2E;
    if (hi == 0 && rr < rows) p.dvec[at] = dsum;
    f32x16 dqt[DB];

    GgwRegs<D> rk, rv;
    unsigned char rkeep = 1;
    auto load = [&](int i) {
        const int j0 = ggw_tile_at(rg, i) * 64;
        rk = ggw_load_keys<D>(kb, p.kn, j0, rg, p.sinks, keep);
        rv = ggw_load_keys<D>(vb, p.vn, j0, rg, p.sinks, keep);
        if (keep && threadIdx.x < 64) rkeep = j0 + (int)threadIdx.x < len ? keep[j0 + threadIdx.x] : 0;
    };
    bool again = false;             // the second walk: a row that sees a key with a NaN or an infinity gets NaN, the others go without that key
    float nan = 0.f;
    auto store = [&](int buf) {
        if (again) {
            ggw_take_bad<T, D>(rk, sBad[buf], false);
            ggw_take_bad<T, D>(rv, sBad[buf], true);
        }
        ggw_store_tile<D>(rk, sK[buf]);
        ggw_store_tile<D>(rv, sV[buf]);
        if (keep && threadIdx.x < 64) sKeep[buf][threadIdx.x] = rkeep;
    };
walk:
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) dqt[db][r] = 0.f;
    if (rg.nt > 0) {
        load(0);
        store(0);
        if (rg.nt > 1) load(1);
    }
    if (threadIdx.x == 0) sAgain = 0;
    gg_sync();
    for (int i = 0, buf = 0; i < rg.nt; ++i, buf ^= 1) {
        if (i + 1 < rg.nt) {
            store(buf ^ 1);
            if (i + 2 < rg.nt) load(i + 2);
        }
        const int j0 = ggw_tile_at(rg, i) * 64;
        if (j0 <= whij && (j0 + 63 >= wlo - p.left || j0 < p.sinks) && wr0 < rows) {
            const bool masked = !(whole && !keep && j0 + 63 <= wlij && (j0 >= whi - p.left || j0 + 63 < p.sinks));
            unsigned long long bits = ~0ull;
            if (keep) bits = gg_ballot(sKeep[buf][lane] != 0);
            bits >>= 4 * hi;
#pragma unroll
            for (int jb = 0; jb < 2; ++jb) {
                f32x16 st, dp;
#pragma unroll
                for (int r = 0; r < 16; ++r) { st[r] = 0.f; dp[r] = -dsum; }
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    st = ggw_mfma<T>(ggw_frag<D>(sK[buf], jb * 32, kk, lane), qf[kk], st);
                    dp = ggw_mfma<T>(ggw_frag<D>(sV[buf], jb * 32, kk, lane), gf[kk], dp);
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) st[r] = gg_exp2f(gg_fmaf(st[r], a2, -lse)) * dp[r];
                if (masked)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int jr = jb * 32 + (r & 3) + 8 * (r >> 2), j = j0 + jr + 4 * hi;
                        const bool see = j <= hij && (j >= lo || j < p.sinks) && ((bits >> jr) & 1);
                        st[r] = see ? st[r] : 0.f;
                    }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const u16x8 sf = ggw_pack8<T>(st, c);
#pragma unroll
                    for (int db = 0; db < DB; ++db) dqt[db] = ggw_mfma<T>(ggw_frag_tr<D>(sK[buf], db * 32, jb * 32 + 16 * c, lane), sf, dqt[db]);
                }
            }
            if (again)
                for (int jr = 0; jr < 64; ++jr)
                    if (ggw_any_bad<D>(sBad[buf], jr)) {
                        const int j = j0 + jr;
                        if (j <= hij && (j >= lo || j < p.sinks) && (!keep || sKeep[buf][jr])) nan = __builtin_nanf("");
                    }
        }
        gg_sync();
    }
    if (!again) {
        if (ggw_not_finite<DB>(dqt)) sAgain = 1;
        gg_sync();
        if (sAgain) {
            again = true;
            gg_sync();
            goto walk;
        }
    }
    if (rr >= rows) return;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int gq = 0; gq < 4; ++gq) {
            u16x4 o4;
#pragma unroll
            for (int e = 0; e < 4; ++e) o4[e] = gg_elt<T>(dqt[db][4 * gq + e] * p.scale + nan);
            *(u16x4*)(p.dq + orow + db * 32 + 8 * gq + 4 * hi) = o4;
        }
}

// ---- backward, part 2: dk, dv -----------------------------------------------------------------------------------------
// workgroup: 4 waves x 32 keys, row tiles of 64 (Q and dO, each read as rows and transposed). The key tiles that hold sinks are seen by
// every later row: their rows are cut into p.sink_chunks chunks, each a workgroup of its own that leaves fp32 sums for
// gg_win_sink_kernel.  part_o: [B*hk][sink_tiles][chunks][2][128][D].
template <int T, int D>
GG_KERNEL GG_LAUNCH_BOUNDS(256) void gg_win_dkv_kernel(GgWinParams p) {
    constexpr int KK = D / 16, DB = D / 32;
    GG_SHARED __attribute__((aligned(16))) char sQ[GgwTile<D>::BYTES];
    GG_SHARED __attribute__((aligned(16))) char sG[GgwTile<D>::BYTES];
    GG_SHARED __attribute__((aligned(16))) float sLse[64];
    GG_SHARED __attribute__((aligned(16))) float sD[64];
    GG_SHARED __attribute__((aligned(16))) int sPos[64];
    GG_SHARED __attribute__((aligned(16))) unsigned char sBad[64 * (D / 8)];
    GG_SHARED int sAgain;

    const int lane = threadIdx.x & 63, wave = gg_uniform(threadIdx.x >> 6), hi = lane >> 5;
    const int per = p.sink_tiles * p.sink_chunks + p.row_tiles - p.sink_tiles;
    const int item = ggw_item();
    const int bkv = item / per;
    int tile = item - bkv * per, chunk = 0;
    const bool chunked = p.sink_chunks > 1 && tile < p.sink_tiles * p.sink_chunks;
    if (tile < p.sink_tiles * p.sink_chunks) { chunk = tile % p.sink_chunks; tile /= p.sink_chunks; }
    else tile -= p.sink_tiles * (p.sink_chunks - 1);
    const int b = bkv / p.hk, kvh = bkv - b * p.hk;
    const int rows = p.n * p.g;
    const int len = ggw_len(p, b), shift = len - p.n;
    const int k0 = tile * 128;
    const unsigned char* keep = p.keep ? p.keep + b * p.keep_b : nullptr;

    // the rows that see some key of the tile
    const int klast = (k0 + 127 < len - 1 ? k0 + 127 : len - 1);
    long long ra = 0, rb = -1;
    if (klast >= k0) {
        int tlo = k0 - p.right - shift, thi = klast + p.left - shift;
        if (k0 < p.sinks || thi > p.n - 1) thi = p.n - 1;
        if (tlo < -shift) tlo = -shift;
        if (tlo < 0) tlo = 0;
        ra = (long long)tlo * p.g;
        rb = (long long)thi * p.g + p.g - 1;
    }
    if (tile < p.sink_tiles && rb >= ra) {
        const long long nt = (rb - ra + 64) / 64, c0 = nt * chunk / p.sink_chunks, c1 = nt * (chunk + 1) / p.sink_chunks;
        const long long a = ra + c0 * 64, z = ra + c1 * 64 - 1;
        ra = a;
        rb = z < rb ? z : rb;
    }

    const int kj0 = k0 + wave * 32, kj = kj0 + (lane & 31), kjc = kj < p.m ? kj : p.m - 1;
    const bool kept = kj < len && (!keep || keep[kj]);
    const bool whole = kj0 + 31 < len && !keep;             // (wave-uniform)
    const int wlast = kj0 + 31;
    u16x8 kf[KK], vf[KK];
    {
        const unsigned short* kr = p.k + b * p.kb + kvh * p.kh + (long long)kjc * p.kn + 8 * hi;
        const unsigned short* vr = p.v + b * p.vb + kvh * p.vh + (long long)kjc * p.vn + 8 * hi;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) { kf[kk] = *(const u16x8*)(kr + kk * 16); vf[kk] = *(const u16x8*)(vr + kk * 16); }
    }
    const float a2 = p.scale * GGW_LOG2E;
    f32x16 acc[2 * DB];                     // dk, dv
    f32x16 *dkt = acc, *dvt = acc + DB;

    const unsigned short* qb = p.q + b * p.qb + (long long)kvh * p.g * p.qh;
    const unsigned short* gb = p.d_o + b * p.gb + (long long)kvh * p.g * p.gh;
    GgwRegs<D> rq, rg;
    float r_lse = 0.f, r_d = 0.f;
    int r_pos = 0;
    auto load = [&](int i0) {
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            const int v = threadIdx.x + 256 * s, c8 = v % (D / 8);
            int r = i0 + v / (D / 8);
            r = r <= (int)rb ? r : (int)rb;
            const int tok = (int)((unsigned)r / (unsigned)p.g), hd = r - tok * p.g;
            rq.v[s] = rg.v[s] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
            if (p.lse[(long long)bkv * rows + r] < __builtin_inff()) {          // (a row that sees nothing: zeros, whatever lies there)
                rq.v[s] = *(const u16x8*)(qb + hd * p.qh + (long long)tok * p.qn + c8 * 8);
                rg.v[s] = *(const u16x8*)(gb + hd * p.gh + (long long)tok * p.gn + c8 * 8);
            }
        }
        if (threadIdx.x < 64) {
            const int r = i0 + (int)threadIdx.x, rc = r <= (int)rb ? r : (int)rb;
            r_lse = r <= (int)rb ? p.lse[(long long)bkv * rows + rc] : __builtin_inff();
            r_d = p.dvec[(long long)bkv * rows + rc];
            r_pos = r <= (int)rb ? (int)((unsigned)r / (unsigned)p.g) + shift : -2 * GGW_NONE;
        }
    };
    bool again = false;             // the second walk: a key that a row with a NaN or an infinity sees gets NaN, the others go without that row
    float nan = 0.f;
walk:
#pragma unroll
    for (int i = 0; i < 2 * DB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
    if (threadIdx.x == 0) sAgain = 0;
    if (ra <= rb) load((int)ra);
    for (int i0 = (int)ra; i0 <= (int)rb; i0 += 64) {
        gg_sync();
        if (again) {
            ggw_take_bad<T, D>(rq, sBad, false);
            ggw_take_bad<T, D>(rg, sBad, true);
        }
        ggw_store_tile<D>(rq, sQ);
        ggw_store_tile<D>(rg, sG);
        if (threadIdx.x < 64) { sLse[threadIdx.x] = r_lse; sD[threadIdx.x] = r_d; sPos[threadIdx.x] = r_pos; }
        gg_sync();
        if (i0 + 64 <= (int)rb) load(i0 + 64);
#pragma unroll
        for (int ib = 0; ib < 2; ++ib) {
            // the 32 rows' positions: all there, and the wave's 32 keys all seen by all of them?
            const int r1 = i0 + ib * 32 + 31;
            if (i0 + ib * 32 > (int)rb) break;
            const int plo = (i0 + ib * 32) / p.g + shift, phi = (r1 <= (int)rb ? r1 : (int)rb) / p.g + shift;
            if (kj0 > phi + p.right || (wlast < plo - p.left && kj0 >= p.sinks) || kj0 >= len) continue;
            const bool full = whole && r1 <= (int)rb && wlast <= plo + p.right && (kj0 >= phi - p.left || wlast < p.sinks);
            f32x16 st, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) { st[r] = 0.f; dp[r] = 0.f; }
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                st = ggw_mfma<T>(ggw_frag<D>(sQ, ib * 32, kk, lane), kf[kk], st);
                dp = ggw_mfma<T>(ggw_frag<D>(sG, ib * 32, kk, lane), vf[kk], dp);
            }
#pragma unroll
            for (int gq = 0; gq < 4; ++gq) {
                const int at = ib * 32 + 8 * gq + 4 * hi;
                const f32x4 ls = *(const f32x4*)&sLse[at], dd = *(const f32x4*)&sD[at];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 4 * gq + e;
                    st[r] = gg_exp2f(gg_fmaf(st[r], a2, -ls[e]));
                    dp[r] = st[r] * (dp[r] - dd[e]);
                }
                if (!full)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 4 * gq + e, pos = sPos[at + e];
                        const bool see = kept && kj <= pos + p.right && (kj >= pos - p.left || kj < p.sinks);
                        st[r] = see ? st[r] : 0.f;
                        dp[r] = see ? dp[r] : 0.f;
                    }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const u16x8 pf = ggw_pack8<T>(st, c), sf = ggw_pack8<T>(dp, c);
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    dvt[db] = ggw_mfma<T>(ggw_frag_tr<D>(sG, db * 32, ib * 32 + 16 * c, lane), pf, dvt[db]);
                    dkt[db] = ggw_mfma<T>(ggw_frag_tr<D>(sQ, db * 32, ib * 32 + 16 * c, lane), sf, dkt[db]);
                }
            }
            if (again)
                for (int ir = ib * 32; ir < ib * 32 + 32; ++ir)
                    if (ggw_any_bad<D>(sBad, ir)) {
                        const int pos = sPos[ir];
                        if (kept && kj <= pos + p.right && (kj >= pos - p.left || kj < p.sinks)) nan = __builtin_nanf("");
                    }
        }
    }
    if (!again) {
        gg_sync();
        if (ggw_not_finite<2 * DB>(acc)) sAgain = 1;
        gg_sync();
        if (sAgain) {
            again = true;
            gg_sync();
            goto walk;
        }
    }
    if (chunked) {
        float* po = p.part_o + ((((long long)bkv * p.sink_tiles + tile) * p.sink_chunks + chunk) * 2 * 128 + wave * 32 + (lane & 31)) * D;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int gq = 0; gq < 4; ++gq) {
                const int d = db * 32 + 8 * gq + 4 * hi;
                *(f32x4*)(po + d) = f32x4{dkt[db][4 * gq] + nan, dkt[db][4 * gq + 1] + nan, dkt[db][4 * gq + 2] + nan, dkt[db][4 * gq + 3] + nan};
                *(f32x4*)(po + 128 * D + d) = f32x4{dvt[db][4 * gq] + nan, dvt[db][4 * gq + 1] + nan, dvt[db][4 * gq + 2] + nan, dvt[db][4 * gq + 3] + nan};
            }
        return;
    }
    if (kj >= p.m) return;
    const long long krow = (((long long)b * p.m + kj) * p.hk + kvh) * D;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int gq = 0; gq < 4; ++gq) {
            u16x4 k4, v4;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                k4[e] = gg_elt<T>(dkt[db][4 * gq + e] * p.scale + nan);
                v4[e] = gg_elt<T>(dvt[db][4 * gq + e] + nan);
            }
            *(u16x4*)(p.dk + krow + db * 32 + 8 * gq + 4 * hi) = k4;
            *(u16x4*)(p.dv + krow + db * 32 + 8 * gq + 4 * hi) = v4;
        }
}

// the row chunks of the sink tiles added in order: four features of one key's dk and dv a thread
template <int T, int D>
GG_KERNEL GG_LAUNCH_BOUNDS(256) void gg_win_sink_kernel(GgWinParams p) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const int d = (int)(i % (D / 4)) * 4;
    const long long key = i / (D / 4);                       // (b, kvh, key of the sink tiles)
    const int span = p.sink_tiles * 128;
    const int bkv = (int)(key / span), j = (int)(key - (long long)bkv * span);
    if (bkv >= p.B * p.hk || j >= p.m) return;
    const float* po = p.part_o + (((long long)bkv * p.sink_tiles + j / 128) * p.sink_chunks * 2 * 128 + j % 128) * D + d;
    f32x4 sk = {0.f, 0.f, 0.f, 0.f}, sv = sk;
    for (int c = 0; c < p.sink_chunks; ++c) {
        sk += *(const f32x4*)(po + (long long)c * 2 * 128 * D);
        sv += *(const f32x4*)(po + ((long long)c * 2 + 1) * 128 * D);
    }
    const int b = bkv / p.hk, kvh = bkv - b * p.hk;
    const long long at = (((long long)b * p.m + j) * p.hk + kvh) * D + d;
    u16x4 k4, v4;
#pragma unroll
    for (int e = 0; e < 4; ++e) { k4[e] = gg_elt<T>(sk[e] * p.scale); v4[e] = gg_elt<T>(sv[e]); }
    *(u16x4*)(p.dk + at) = k4;
    *(u16x4*)(p.dv + at) = v4;
}

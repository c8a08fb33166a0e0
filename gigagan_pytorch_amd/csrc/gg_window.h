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
// Keys behind the sequence's end are staged as zeros. For the rest every kernel looks at its own result once, at the end: if something in
// it is not finite, the tiles are walked a second time with every non-finite vector taken out of the tile and accounted for by itself,
// key by key, for the rows that see it. Finite inputs never take the second walk.
#pragma once
#include "gg_element.h"

#define GGW_NONE 0x20000000          // "no bound" of a window side, and (negated, doubled) the position of a row that is not there
#define GGW_SPAN 0xf0000000u         // buffer length behind a row tile's first token; an offset of this size reads zeros
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
// A tile is 64 rows of D features as the LDS-DMA deposits them: wave instruction after wave instruction of 64 x 16 bytes, rows back to
// back. No padding is possible, so the 16-byte vectors of a row are permuted instead: vector c lies at position c ^ ggw_swz(row) (the
// DMA's source addresses are permuted, its LDS addresses cannot be). The LDS serves 256 bytes, all 64 banks, at a time: a ds_read_b128 in
// four groups of sixteen lanes (0-3, 12-15, 20-27 | 4-11, 16-19, 28-31 | the same + 32: measured pair by pair), a transpose read in two
// halves of the wave. The permutation gives sixteen such rows sixteen different positions of one vector, and four consecutive rows four
// different 64-byte spans: neither kind of read waits for a bank (a two-way conflict halves its rate, 5.7 for 2.9 cycles a read).
template <int D> struct GgwTile { static constexpr int BYTES = 64 * D * 2; };
template <int D>
GG_DEVICE int ggw_swz(int row) {
    const int q = (row >> 2) & 3;
    if constexpr (D == 32) return q;                        // (four rows span the banks)
    else if constexpr (D == 64) return ((row & 2) << 1) | q;        // (two rows)
    else return ((row & 3) << 2) | q;
}

// A operand, rows as they lie: lane l -> row row0 + (l & 31), features kk*16 + 8(l >> 5) + 0..7
template <int D>
GG_DEVICE u16x8 ggw_frag(const char* tile, int row0, int kk, int lane) {
    const int row = lane & 31;                              // (row0 is a multiple of 32: it does not change the permutation)
    return *(const u16x8*)(tile + row0 * D * 2 + ((row * D * 2 + (((lane >> 5) ^ ggw_swz<D>(row)) << 4)) ^ (kk << 5)));
}
// A operand of the tile's transpose: lane l -> feature d0 + (l & 31), slots (hi, e) <-> rows rb + 4hi + (e & 3) + 8(e >> 2)
template <int D>
GG_DEVICE u16x8 ggw_frag_tr(const char* tile, int d0, int rb, int lane) {
    const int i = lane & 15, gq = lane >> 4;
    const int row = 4 * (gq >> 1) + (i >> 2), c = 2 * (gq & 1) + ((i & 3) >> 1);
    // (rb is a multiple of 16 and does not change the permutation; eight rows further on it differs by 2)
    const int at = (row * D * 2 + ((c ^ ggw_swz<D>(row)) << 4) + 8 * (i & 1)) ^ (d0 << 1);
    const u16x4 a = gg_lds_read_tr16((const bf16_t*)(tile + rb * D * 2 + at));
    const u16x4 b = gg_lds_read_tr16((const bf16_t*)(tile + (rb + 8) * D * 2 + (at ^ 32)));
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
// a key that some row of the range sees (key mask apart)
GG_DEVICE bool ggw_in_range(const GgwRange& r, int sinks, int j) { return j <= r.khi && (j >= r.klo || j < sinks); }

// One 64-row tile from memory to LDS by DMA: NW waves, D / (8 NW) instructions each. `base` points at the tile's first row, `rows` of it
// exist (the rest is deposited as zeros by the buffer's bounds check). voff[] = ggw_dma_offsets.
template <int D, int NW> struct GgwDma { static constexpr int N = D / (8 * NW) < 1 ? 1 : D / (8 * NW); };
template <int D, int NW>
GG_DEVICE void ggw_dma_offsets(unsigned* voff, long long stride) {
#pragma unroll
    for (int i = 0; i < GgwDma<D, NW>::N; ++i) {
        const int v = threadIdx.x + 64 * NW * i, row = v / (D / 8), c = v % (D / 8);
        voff[i] = (unsigned)(row * stride * 2) + ((c ^ ggw_swz<D>(row)) << 4);
    }
}
template <int D, int NW>
GG_DEVICE void ggw_dma(const unsigned short* base, int rows, long long stride, const unsigned* voff, char* tile, int wave) {
    if (GgwDma<D, NW>::N * 8 * NW > D && wave >= D / 8) return;             // (D 32, eight waves: four of them have nothing to fetch)
    const unsigned long long bytes = rows <= 0 ? 0 : ((unsigned long long)(rows < 64 ? rows - 1 : 63) * stride + D) * 2;
    const GgBufS buf = gg_make_bufs(base, bytes);
#pragma unroll
    for (int i = 0; i < GgwDma<D, NW>::N; ++i) gg_bufs_load_lds16(buf, voff[i], 0, tile + (wave + NW * i) * 1024);
}

// The second walk's tile, through registers: rows that `want` names, the others zeros; vectors with a NaN or an infinity are taken out
// and marked, bad[row][vector] (add: on top of what is marked there; bad null: all stay).
template <int T, int D, int NW, class Row>
GG_DEVICE void ggw_stage_clean(char* tile, unsigned char* bad, bool add, Row row_at) {
    for (int v = threadIdx.x; v < 64 * (D / 8); v += 64 * NW) {
        const int row = v / (D / 8), c = v % (D / 8);
        const unsigned short* src = row_at(row);            // null: nobody sees it
        u16x8 x = {0, 0, 0, 0, 0, 0, 0, 0};
        if (src) x = *(const u16x8*)(src + c * 8);
        if (bad) {
            const bool b = ggw_bad8<T>(x);
            if (b) x = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
            bad[v] = (unsigned char)((add ? bad[v] : 0) | b);
        }
        *(u16x8*)(tile + row * D * 2 + ((c ^ ggw_swz<D>(row)) << 4)) = x;
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
        const float pj = see(j) ? gg_exp2f(gg_fmaf(s, a2, -m)) : 0.f;
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
            if (bad[jr * (D / 8) + c]) {
                const u16x4 v4 = *(const u16x4*)(vb + (long long)j * vn + c * 8 + 4 * hi);
#pragma unroll
                for (int e = 0; e < 4; ++e) ot[c / 4][4 * (c % 4) + e] += pj > 0.f ? pj * gg_elt_f<T>(v4[e]) : 0.f;
            }
    }
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

// the rows of one wave, lane by lane, and what its 32 rows see between them
struct GgwWave {
    GgwRow row;
    int r0, r;              // the wave's first row, this lane's
    int lo, hi;             // this lane: window keys lo .. hi (hi = -1: nothing)
    int lo_any, hi_any;     // (wave-uniform) window keys that some / all of the wave's rows see
    int lo_all, hi_all;
    bool there;             // some row exists
};
GG_DEVICE GgwWave ggw_wave(const GgWinParams& p, int r0, int len, bool masked) {
    GgwWave w;
    const int rows = p.n * p.g, lane = threadIdx.x & 63, shift = len - p.n;
    w.r0 = r0;
    w.r = r0 + (lane & 31);
    w.row = ggw_row(p, w.r, len);
    w.there = r0 < rows;
    const int last = r0 + 31 < rows ? r0 + 31 : rows - 1;
    const int plo = r0 / p.g + shift, phi = last / p.g + shift;
    w.lo = w.row.pos - p.left;
    w.hi = w.row.in ? (w.row.pos + p.right < len - 1 ? w.row.pos + p.right : len - 1) : -1;
    w.lo_any = plo - p.left;
    w.hi_any = w.there ? (phi + p.right < len - 1 ? phi + p.right : len - 1) : -1;
    w.lo_all = phi - p.left;
    // rows that are missing or padding see nothing, and a key mask may take any key away: no tile is whole then
    w.hi_all = r0 + 31 < rows && plo >= 0 && !masked ? (plo + p.right < len - 1 ? plo + p.right : len - 1) : -1;
    return w;
}
GG_DEVICE bool ggw_some(const GgwWave& w, int sinks, int j0, int j1) { return j0 <= w.hi_any && (j1 >= w.lo_any || j0 < sinks); }
GG_DEVICE bool ggw_whole(const GgwWave& w, int sinks, int j0, int j1) { return j1 <= w.hi_all && (j0 >= w.lo_all || j1 < sinks); }
GG_DEVICE bool ggw_sees(const GgwWave& w, int sinks, int j) { return j <= w.hi && (j >= w.lo || j < sinks); }

// ---- forward -------------------------------------------------------------------------------------------------------
// workgroup: NW waves x 32 rows, key tiles of 64 fetched once for all of them by LDS-DMA, double buffered: one barrier a tile, behind
// which the next tile's transfers start and run under this tile's arithmetic.
// SPLIT: the tiles are dealt out to p.splits workgroups, which leave (m, l, O) for gg_win_join_kernel.
template <int T, int D, int NW, bool SPLIT>
GG_KERNEL GG_LAUNCH_BOUNDS2(64 * NW, 2) void gg_win_fwd_kernel(GgWinParams p) {
    constexpr int KK = D / 16, DB = D / 32;
    GG_SHARED __attribute__((aligned(1024))) char sK[2][GgwTile<D>::BYTES];
    GG_SHARED __attribute__((aligned(1024))) char sV[2][GgwTile<D>::BYTES];
    GG_SHARED __attribute__((aligned(16))) unsigned char sBad[64 * (D / 8)];
    GG_SHARED int sAgain;

    const int lane = threadIdx.x & 63, wave = gg_uniform(threadIdx.x >> 6), hi = lane >> 5;
    int item = ggw_item();
    int split = 0;
    if (SPLIT) { split = item % p.splits; item /= p.splits; }
    const int bkv = item / p.row_tiles, tile = item - bkv * p.row_tiles;
    const int b = bkv / p.hk, kvh = bkv - b * p.hk;
    const int rows = p.n * p.g;
    const int len = ggw_len(p, b);
    const int r0 = tile * (32 * NW), rl = r0 + 32 * NW - 1 < rows - 1 ? r0 + 32 * NW - 1 : rows - 1;
    const GgwRange rg = ggw_range<64>(p, len, r0 / p.g, rl / p.g);
    const int ta = SPLIT ? (int)((long long)rg.nt * split / p.splits) : 0, tb = SPLIT ? (int)((long long)rg.nt * (split + 1) / p.splits) : rg.nt;

    const unsigned char* keep = p.keep ? p.keep + b * p.keep_b : nullptr;
    const GgwWave w = ggw_wave(p, r0 + wave * 32, len, keep != nullptr);
    const unsigned short* kb = p.k + b * p.kb + kvh * p.kh;
    const unsigned short* vb = p.v + b * p.vb + kvh * p.vh;
    u16x8 qf[KK];
    {
        const unsigned short* qr = p.q + b * p.qb + (long long)(kvh * p.g + w.row.head) * p.qh + (long long)w.row.token * p.qn + 8 * hi;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) qf[kk] = *(const u16x8*)(qr + kk * 16);
    }
    unsigned ko[GgwDma<D, NW>::N], vo[GgwDma<D, NW>::N];
    ggw_dma_offsets<D, NW>(ko, p.kn);
    ggw_dma_offsets<D, NW>(vo, p.vn);
    auto fetch = [&](int i, int buf) {
        const int j0 = ggw_tile_at(rg, i) * 64;
        ggw_dma<D, NW>(kb + (long long)j0 * p.kn, len - j0, p.kn, ko, sK[buf], wave);
        ggw_dma<D, NW>(vb + (long long)j0 * p.vn, len - j0, p.vn, vo, sV[buf], wave);
    };
    const float a2 = p.scale * GGW_LOG2E;
    float m, l;
    f32x16 ot[DB];
    bool again = false;             // the second walk (workgroup-uniform)
walk:
    m = -1.0e30f;
    l = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) ot[db][r] = 0.f;
    if (threadIdx.x == 0) sAgain = 0;
    if (!again && ta < tb) fetch(ta, 0);
    for (int i = ta, buf = 0; i < tb; ++i, buf ^= 1) {
        const int j0 = ggw_tile_at(rg, i) * 64;
        if (!again) {
            gg_wait_vm<0>();
            gg_barrier_lds();       // this tile is there for everyone, and everyone is through with the last one: its buffer is free
            if (i + 1 < tb) fetch(i + 1, buf ^ 1);
        } else {
            gg_sync();
            auto in = [&](int j) { return ggw_in_range(rg, p.sinks, j) && (!keep || keep[j]); };
            ggw_stage_clean<T, D, NW>(sK[buf], nullptr, false, [&](int row) { return in(j0 + row) ? kb + (long long)(j0 + row) * p.kn : nullptr; });
            ggw_stage_clean<T, D, NW>(sV[buf], sBad, false, [&](int row) { return in(j0 + row) ? vb + (long long)(j0 + row) * p.vn : nullptr; });
            gg_sync();
        }
        if (!ggw_some(w, p.sinks, j0, j0 + 63)) continue;
        f32x16 st[2];
#pragma unroll
        for (int jb = 0; jb < 2; ++jb) {
#pragma unroll
            for (int r = 0; r < 16; ++r) st[jb][r] = 0.f;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) st[jb] = ggw_mfma<T>(ggw_frag<D>(sK[buf], jb * 32, kk, lane), qf[kk], st[jb]);
        }
        if (!ggw_whole(w, p.sinks, j0, j0 + 63)) {
            unsigned long long bits = ~0ull;
            if (keep) bits = gg_ballot(j0 + lane < len && keep[j0 + lane]);
            bits >>= 4 * hi;
#pragma unroll
            for (int jb = 0; jb < 2; ++jb)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int jr = jb * 32 + (r & 3) + 8 * (r >> 2);
                    const bool see = ggw_sees(w, p.sinks, j0 + jr + 4 * hi) && ((bits >> jr) & 1);
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
            ggw_add_bad<T, D>(ot, sBad, 64, j0, kb, p.kn, vb, p.vn, qf, a2, m, hi, [&](int j) { return ggw_sees(w, p.sinks, j) && (!keep || keep[j]); });
    }
    if (!again) {
        gg_sync();
        if (ggw_not_finite<DB>(ot)) sAgain = 1;
        gg_sync();
        if (sAgain) {
            again = true;
            gg_sync();
            goto walk;
        }
    }
    l = gg_sum_xor32(l);
    if (w.r >= rows) return;
    const long long at = (long long)bkv * rows + w.r;
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
    unsigned short* orow = p.o + (((long long)b * p.n + w.row.token) * p.h + kvh * p.g + w.row.head) * D;
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
    constexpr int KK = D / 16, DB = D / 32;
    GG_SHARED __attribute__((aligned(16))) char sV[4][32 * D * 2];
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
            const int vrow = v / (D / 8);
            *(u16x8*)(sV[wave] + vrow * D * 2 + (((v % (D / 8)) ^ ggw_swz<D>(vrow)) << 4)) = vr[s];
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
            ggw_add_bad<T, D>(ot, sBad[wave], 32, j0, kb, p.kn, vb, p.vn, qf, a2, m, hi, [&](int j) { return j <= hij && (j >= lo || j < p.sinks) && (!keep || keep[j]); });
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
// the forward's mapping and transfers; K is read as rows (scores) and transposed (dq), V as rows (dP)
template <int T, int D, int NW>
GG_KERNEL GG_LAUNCH_BOUNDS2(64 * NW, 2) void gg_win_dq_kernel(GgWinParams p) {
    constexpr int KK = D / 16, DB = D / 32;
    GG_SHARED __attribute__((aligned(1024))) char sK[2][GgwTile<D>::BYTES];
    GG_SHARED __attribute__((aligned(1024))) char sV[2][GgwTile<D>::BYTES];
    GG_SHARED __attribute__((aligned(16))) unsigned char sBad[64 * (D / 8)];
    GG_SHARED int sAgain;

    const int lane = threadIdx.x & 63, wave = gg_uniform(threadIdx.x >> 6), hi = lane >> 5;
    const int item = ggw_item();
    const int bkv = item / p.row_tiles, tile = item - bkv * p.row_tiles;
    const int b = bkv / p.hk, kvh = bkv - b * p.hk;
    const int rows = p.n * p.g;
    const int len = ggw_len(p, b);
    const int r0 = tile * (32 * NW), rl = r0 + 32 * NW - 1 < rows - 1 ? r0 + 32 * NW - 1 : rows - 1;
    const GgwRange rg = ggw_range<64>(p, len, r0 / p.g, rl / p.g);
    const unsigned char* keep = p.keep ? p.keep + b * p.keep_b : nullptr;
    const GgwWave w = ggw_wave(p, r0 + wave * 32, len, keep != nullptr);
    const unsigned short* kb = p.k + b * p.kb + kvh * p.kh;
    const unsigned short* vb = p.v + b * p.vb + kvh * p.vh;
    const int hq = kvh * p.g + w.row.head;
    const long long orow = (((long long)b * p.n + w.row.token) * p.h + hq) * D;
    const long long at = (long long)bkv * rows + (w.r < rows ? w.r : rows - 1);
    u16x8 qf[KK], gf[KK];
    float dsum = 0.f;
    {
        const unsigned short* qr = p.q + b * p.qb + hq * p.qh + (long long)w.row.token * p.qn + 8 * hi;
        const unsigned short* gr = p.d_o + b * p.gb + hq * p.gh + (long long)w.row.token * p.gn + 8 * hi;
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
    if (hi == 0 && w.r < rows) p.dvec[at] = dsum;
    unsigned ko[GgwDma<D, NW>::N], vo[GgwDma<D, NW>::N];
    ggw_dma_offsets<D, NW>(ko, p.kn);
    ggw_dma_offsets<D, NW>(vo, p.vn);
    auto fetch = [&](int i, int buf) {
        const int j0 = ggw_tile_at(rg, i) * 64;
        ggw_dma<D, NW>(kb + (long long)j0 * p.kn, len - j0, p.kn, ko, sK[buf], wave);
        ggw_dma<D, NW>(vb + (long long)j0 * p.vn, len - j0, p.vn, vo, sV[buf], wave);
    };
    f32x16 dqt[DB];
    bool again = false;             // the second walk: a row that sees a key with a NaN or an infinity gets NaN, the others go without that key
    float nan = 0.f;
walk:
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) dqt[db][r] = 0.f;
    if (threadIdx.x == 0) sAgain = 0;
    if (!again && rg.nt > 0) {
        gg_wait_vm<0>();            // (the rows above: the transfers' count starts at zero)
        fetch(0, 0);
    }
    for (int i = 0, buf = 0; i < rg.nt; ++i, buf ^= 1) {
        const int j0 = ggw_tile_at(rg, i) * 64;
        if (!again) {
            gg_wait_vm<0>();
            gg_barrier_lds();
            if (i + 1 < rg.nt) fetch(i + 1, buf ^ 1);
        } else {
            gg_sync();
            auto in = [&](int j) { return ggw_in_range(rg, p.sinks, j) && (!keep || keep[j]); };
            ggw_stage_clean<T, D, NW>(sK[buf], sBad, false, [&](int row) { return in(j0 + row) ? kb + (long long)(j0 + row) * p.kn : nullptr; });
            ggw_stage_clean<T, D, NW>(sV[buf], sBad, true, [&](int row) { return in(j0 + row) ? vb + (long long)(j0 + row) * p.vn : nullptr; });
            gg_sync();
        }
        if (!ggw_some(w, p.sinks, j0, j0 + 63)) continue;
        const bool masked = !ggw_whole(w, p.sinks, j0, j0 + 63);
        unsigned long long bits = ~0ull;
        if (keep) bits = gg_ballot(j0 + lane < len && keep[j0 + lane]);
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
            if (masked) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int jr = jb * 32 + (r & 3) + 8 * (r >> 2);
                    const bool see = ggw_sees(w, p.sinks, j0 + jr + 4 * hi) && ((bits >> jr) & 1);
                    st[r] = see ? st[r] : 0.f;
                }
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
                if (ggw_any_bad<D>(sBad, jr) && ggw_sees(w, p.sinks, j0 + jr) && (!keep || keep[j0 + jr])) nan = __builtin_nanf("");
    }
    if (!again) {
        gg_sync();
        if (ggw_not_finite<DB>(dqt)) sAgain = 1;
        gg_sync();
        if (sAgain) {
            again = true;
            gg_sync();
            goto walk;
        }
    }
    if (w.r >= rows) return;
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
// workgroup: 4 waves x 32 keys, row tiles of 64 (Q and dO by LDS-DMA, double buffered, each read as rows and transposed). The key tiles that hold sinks are seen by
// every later row: their rows are cut into p.sink_chunks chunks, each a workgroup of its own that leaves fp32 sums for
// gg_win_sink_kernel.  part_o: [B*hk][sink_tiles][chunks][2][128][D].
template <int T, int D>
GG_KERNEL GG_LAUNCH_BOUNDS2(256, 2) void gg_win_dkv_kernel(GgWinParams p) {
    constexpr int KK = D / 16, DB = D / 32;
    GG_SHARED __attribute__((aligned(1024))) char sQ[2][GgwTile<D>::BYTES];
    GG_SHARED __attribute__((aligned(1024))) char sG[2][GgwTile<D>::BYTES];
    GG_SHARED __attribute__((aligned(16))) float sLse[2][64];
    GG_SHARED __attribute__((aligned(16))) float sD[2][64];
    GG_SHARED __attribute__((aligned(16))) int sPos[2][64];
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
    // this thread's vectors of a row tile: row index -> (token, head) kept up from tile to tile, addresses relative to the tile's first
    // token (host: they fit 32 bits)
    constexpr int NV = D / 32;
    const int step_t = 64 / p.g, step_h = 64 - step_t * p.g;
    int vt[NV], vh[NV];
    int rt = 0, rh = 0;                     // the row whose statistics this thread fetches (threads 0 .. 63)
    auto start = [&](int i0) {
#pragma unroll
        for (int s = 0; s < NV; ++s) {
            const int r = i0 + (int)(threadIdx.x + 256 * s) / (D / 8);
            vt[s] = (int)((unsigned)r / (unsigned)p.g);
            vh[s] = r - vt[s] * p.g;
        }
        const int r = i0 + (int)(threadIdx.x & 63);
        rt = (int)((unsigned)r / (unsigned)p.g);
        rh = r - rt * p.g;
    };
    float r_lse = 0.f, r_d = 0.f;
    int r_pos = 0;
    auto fetch = [&](int i0, int buf) {
        const int t0 = (int)((unsigned)i0 / (unsigned)p.g);
        const GgBufS bq = gg_make_bufs(qb + (long long)t0 * p.qn, GGW_SPAN), bg = gg_make_bufs(gb + (long long)t0 * p.gn, GGW_SPAN);
#pragma unroll
        for (int s = 0; s < NV; ++s) {
            const int v = threadIdx.x + 256 * s, row = v / (D / 8), c = (v % (D / 8)) ^ ggw_swz<D>(row);
            // (rows behind the last one: an offset that the buffer's bounds check turns into zeros)
            const bool in = i0 + row <= (int)rb;
            const unsigned oq = in ? (unsigned)(((long long)(vt[s] - t0) * p.qn + (long long)vh[s] * p.qh) * 2) + (c << 4) : GGW_SPAN;
            const unsigned og = in ? (unsigned)(((long long)(vt[s] - t0) * p.gn + (long long)vh[s] * p.gh) * 2) + (c << 4) : GGW_SPAN;
            gg_bufs_load_lds16(bq, oq, 0, sQ[buf] + (wave + 4 * s) * 1024);
            gg_bufs_load_lds16(bg, og, 0, sG[buf] + (wave + 4 * s) * 1024);
            vt[s] += step_t;
            vh[s] += step_h;
            if (vh[s] >= p.g) { vh[s] -= p.g; ++vt[s]; }
        }
    };
    auto stats = [&](int i0) {              // lse = +inf: a row that is not there or sees nothing
        const int r = i0 + (int)(threadIdx.x & 63);
        const bool in = r <= (int)rb;
        const long long at = (long long)bkv * rows + (in ? r : (int)rb);
        r_lse = in ? p.lse[at] : __builtin_inff();
        r_d = in ? p.dvec[at] : 0.f;
        r_pos = in ? rt + shift : -2 * GGW_NONE;
        rt += step_t;
        rh += step_h;
        if (rh >= p.g) { rh -= p.g; ++rt; }
    };
    bool again = false;             // the second walk: a key that a row with a NaN or an infinity sees gets NaN, the others go without that row
    float nan = 0.f;
walk:
#pragma unroll
    for (int i = 0; i < 2 * DB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
    if (threadIdx.x == 0) sAgain = 0;
    if (ra <= rb) {
        start((int)ra);
        stats((int)ra);
        if (!again) fetch((int)ra, 0);
    }
    for (int i0 = (int)ra, buf = 0; i0 <= (int)rb; i0 += 64, buf ^= 1) {
        if (threadIdx.x < 64) { sLse[buf][threadIdx.x] = r_lse; sD[buf][threadIdx.x] = r_d; sPos[buf][threadIdx.x] = r_pos; }
        if (!again) {
            gg_wait_vm<0>();
            gg_barrier_lds();
            if (i0 + 64 <= (int)rb) {
                stats(i0 + 64);
                fetch(i0 + 64, buf ^ 1);
            }
        } else {
            gg_sync();
            auto at = [&](const unsigned short* base, long long hs, long long ns, int row) -> const unsigned short* {
                const int r = i0 + row, tok = (int)((unsigned)r / (unsigned)p.g);
                if (r > (int)rb || !(sLse[buf][row] < __builtin_inff())) return nullptr;
                return base + (long long)tok * ns + (long long)(r - tok * p.g) * hs;
            };
            ggw_stage_clean<T, D, 4>(sQ[buf], sBad, false, [&](int row) { return at(qb, p.qh, p.qn, row); });
            ggw_stage_clean<T, D, 4>(sG[buf], sBad, true, [&](int row) { return at(gb, p.gh, p.gn, row); });
            if (i0 + 64 <= (int)rb) stats(i0 + 64);
            gg_sync();
        }
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
                st = ggw_mfma<T>(ggw_frag<D>(sQ[buf], ib * 32, kk, lane), kf[kk], st);
                dp = ggw_mfma<T>(ggw_frag<D>(sG[buf], ib * 32, kk, lane), vf[kk], dp);
            }
#pragma unroll
            for (int gq = 0; gq < 4; ++gq) {
                const int at = ib * 32 + 8 * gq + 4 * hi;
                const f32x4 ls = *(const f32x4*)&sLse[buf][at], dd = *(const f32x4*)&sD[buf][at];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 4 * gq + e;
                    st[r] = gg_exp2f(gg_fmaf(st[r], a2, -ls[e]));
                    dp[r] = st[r] * (dp[r] - dd[e]);
                }
                if (!full)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 4 * gq + e, pos = sPos[buf][at + e];
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
                    dvt[db] = ggw_mfma<T>(ggw_frag_tr<D>(sG[buf], db * 32, ib * 32 + 16 * c, lane), pf, dvt[db]);
                    dkt[db] = ggw_mfma<T>(ggw_frag_tr<D>(sQ[buf], db * 32, ib * 32 + 16 * c, lane), sf, dkt[db]);
                }
            }
            if (again)
                for (int ir = ib * 32; ir < ib * 32 + 32; ++ir)
                    if (ggw_any_bad<D>(sBad, ir)) {
                        const int pos = sPos[buf][ir];
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

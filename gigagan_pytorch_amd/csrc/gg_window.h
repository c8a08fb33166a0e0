// gg_window.h — attention with a sliding window and sinks, forward, backward and its few-query form.
//
// Query i of batch item b sits at position p = len_b - n + i (the queries are the last n of the sequence's len_b <= m keys) and sees
//     key j   when   j < len_b,   j <= p + right,   j >= p - left or j < sinks,   keep[b][j]
// (a query at a negative position is padding and sees nothing).
//     o_i = sum_j P_ij v_j,   P = softmax over the seen keys of scale q_i.k_j;   a query that sees no key gets zeros and no gradient.
//     (a query that sees keys of score -inf alone: 0 / 0, NaN, as in any softmax; scale log2e s beyond fp32 counts as infinite)
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
// Keys behind the sequence's end are staged as zeros. For the rest every wave looks at its own result once, at the end: rows (dk / dv:
// keys) whose result is not finite are computed again one by one, from memory and from what they see alone (ggw_fix_*). Finite inputs
// come there only with far scores.
//
// Far scores. P is exp2(fma(s, scale log2e, -m)): the rounding of m moves it by a factor of 2^(m 2^-24), and a log-sum-exp of 32 bits
// forgets log2 of the sum beside a large m. From |m| = GGW_FAR on, where that is 2^(1/16), a row is computed again as well, with the
// product rounded before the difference. Its log-sum-exp is m alone; dq finds log2 of the sum anew and leaves it for dk and dv.
#pragma once
#include "gg_element.h"

#define GGW_NONE 0x20000000          // "no bound" of a window side, and (negated, doubled) the position of a row that is not there
#define GGW_SPAN 0xf0000000u         // buffer length behind a row tile's first token; an offset of this size reads zeros
#define GGW_LOG2E 1.4426950408889634f
#define GGW_FAR 1048576.0f           // (see above)
#define GGW_LOW (-3.402823466e38f)   // where the running maximum starts: any finite score is above it, or is it
// What P is taken relative to ("the running maximum") moves when a score exceeds it by TAU (in log2): fewer rescales of the output. It
// moves to LEAD below the largest score: the largest P is 2^LEAD .. 2^TAU. IEEE half, whose least number is 2^-24, has 2^15 to spare
// above one; bf16 has fp32's range.
template <int T> struct GgwExp { static constexpr float LEAD = T == GG_ELT_F16 ? 7.f : 0.f, TAU = LEAD + 8.f; };

struct GgWinParams {
    const unsigned short *q, *k, *v, *d_o;
    unsigned short *o, *o_lo, *dq, *dk, *dv;        // dense: o, o_lo, dq [B][n][h][D]; dk, dv [B][m][hk][D]
    float* lse;                             // [B*hk][n*g]: log2 of the row's sum of 2^(scale log2e s); +inf for a row that sees nothing, NaN for 0 / 0
    float* dvec;                            // [2][B*hk][n*g]: D_i; of far rows log2 of the sum that lse does not hold
    long long qb, qh, kb, kh, vb, vh, gb, gh;       // element strides of q, k, v, dO: batch, head ...
    unsigned qn, kn, vn, gn;                        // ... and token (below 2^24)
    const int* lengths;                     // [B] or null (= m)
    const unsigned char* keep;              // [B][m], batch stride keep_b, or null
    long long keep_b;
    float* part_o;                          // key splits: [split][B*hk][n*g][D] and [split][B*hk][n*g][2] (m, l)
    float* part_ml;
    int B, n, m, h, hk, g;
    int left, right, sinks;
    float scale;
    int splits, join;                       // ... and the thread groups that join a row's splits
    int row_tiles;                          // row (dk / dv: key) tiles per (batch, key head)
    int sink_tiles, sink_chunks;            // dk / dv: the first key tiles (those that hold sinks; all, where there are few), each in row chunks
};

// ---- shared pieces -----------------------------------------------------------------------------------------------

template <int T>
GG_DEVICE f32x16 ggw_mfma(u16x8 a, u16x8 b, f32x16 c) {
    if constexpr (T == GG_ELT_BF16) return gg_mfma_32x32x16_bf16(a, b, c);
    else return gg_mfma_32x32x16_f16(a, b, c);
}
// registers 8c .. 8c + 7 of a result, rounded to 16 bits: the B operand of the follow-up contraction. P and dS are rounded to the operands'
// type because the matrix pipe takes both operands in one type, and an fp32 product runs at a sixteenth of its rate; their sums stay
// fp32. Each rounding is half a step of the type relative to the value (32 captions of 78 tokens, bf16: o and gradients are 0.0022 -
// 0.0025 from 64 bits in the mean, 0.0016 - 0.0017 with P and dS in fp32).
template <int T>
GG_DEVICE u16x8 ggw_pack8(const f32x16& v, int c) {
    u16x8 f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = gg_elt<T>(v[8 * c + e]);
    return f;
}
// dS in IEEE half. P (dP - D) of small gradients lies below half's least number, so a lane keeps a power of two for its row (dk / dv: its
// key) that dS is multiplied with before it is rounded, and its sums with it: 2^e, lowered where a larger dS would leave the range,
// so that the largest so far is 2^8 .. 2^15 (what is rounded to half's least number is 2^-32 of it, or less). bf16 needs none. A training
// pass of 8 x 4096 tokens, 8 heads, window 512 both sides: 430 us without and 455 with it at 64 features, 278 and 310 at 32.
struct GgwScale { int e; };
GG_DEVICE float ggw_pow2(int e) { return __builtin_bit_cast(float, (unsigned)(127 + e) << 23); }       // -126 <= e <= 127
template <int N>
GG_DEVICE void ggw_rescale(GgwScale& s, f32x16& ds, f32x16* sums) {
    float mx = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, fabsf(ds[r]));
    mx = gg_max_xor32(mx);
    if (!gg_wave_any(mx >= 32768.f)) return;
    const bool move = mx >= 32768.f && mx < __builtin_inff();          // (what is infinite is computed again at the end)
    const int k = move ? (int)(__builtin_bit_cast(unsigned, mx) >> 23) - 127 - 8 : 0;
    const float f = ggw_pow2(-k);
    s.e -= k;
#pragma unroll
    for (int r = 0; r < 16; ++r) ds[r] *= f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) sums[i][r] *= f;
}
// which of the wave's 32 rows (columns of the transposed results) hold something that is not finite, as bits
template <int N>
GG_DEVICE unsigned ggw_not_finite(const f32x16* v) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s = gg_fmaf(v[i][r], 0.f, s);
    s = gg_sum_xor32(s);
    return (unsigned)gg_ballot(s != s);
}
// a condition of either lane of a row, as bits of the wave's 32 rows
GG_DEVICE unsigned ggw_rows32(bool x) {
    const unsigned long long b = gg_ballot(x);
    return (unsigned)b | (unsigned)(b >> 32);
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

// This lane's offsets inside a tile, for the two kinds of reads. The vector's index (features 16 kk.., d0..) enters by exclusive or, one
// instruction at the read: kept opaque per tile, or the compiler hoists two dozen addresses out of the loop and runs out of registers.
struct GgwLane { unsigned rows, cols; };
template <int D>
GG_DEVICE GgwLane ggw_lane() {
    const int lane = threadIdx.x & 63, row = lane & 31;
    const int i = lane & 15, gq = lane >> 4, trow = 4 * (gq >> 1) + (i >> 2), c = 2 * (gq & 1) + ((i & 3) >> 1);
    GgwLane o = {(unsigned)(row * D * 2 + (((lane >> 5) ^ ggw_swz<D>(row)) << 4)), (unsigned)(trow * D * 2 + ((c ^ ggw_swz<D>(trow)) << 4) + 8 * (i & 1))};
    return o;
}
GG_DEVICE GgwLane ggw_here(GgwLane o) {
    gg_opaque(o.rows);
    gg_opaque(o.cols);
    return o;
}
// A operand, rows as they lie: lane l -> row row0 + (l & 31), features kk*16 + 8(l >> 5) + 0..7 (row0 a multiple of 32)
template <int D>
GG_DEVICE u16x8 ggw_frag(const char* tile, int row0, int kk, const GgwLane& o) {
    return *(const u16x8*)(tile + row0 * D * 2 + (o.rows ^ (unsigned)(kk << 5)));
}
// A operand of the tile's transpose: lane l -> feature d0 + (l & 31), slots (hi, e) <-> rows rb + 4hi + (e & 3) + 8(e >> 2) (rb a multiple
// of 16; eight rows further on the permutation differs by 2)
template <int D>
GG_DEVICE u16x8 ggw_frag_tr(const char* tile, int d0, int rb, const GgwLane& o) {
    const unsigned at = o.cols ^ (unsigned)(d0 << 1);
    const u16x4 a = gg_lds_read_tr16((const bf16_t*)(tile + rb * D * 2 + at));
    const u16x4 b = gg_lds_read_tr16((const bf16_t*)(tile + (rb + 8) * D * 2 + (at ^ 32)));
    return u16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// N products whose A operands come from the LDS, AHEAD operands read ahead of their use and the order kept (2, 4, 6, 8 ahead: forward at
// head 64 106, 101, 108, 109 us; four, and two where the accumulators leave no registers)
template <int N, int AHEAD = 4, class Read, class Use>
GG_DEVICE void ggw_pipe(Read read, Use use) {
    constexpr int A = AHEAD < N ? AHEAD : N;
    u16x8 f[A];
#pragma unroll
    for (int s = 0; s < A; ++s) f[s] = read(s);
    gg_sched_fence();
#pragma unroll
    for (int s = 0; s < N; ++s) {
        use(s, f[s % A]);
        if (s + A < N) f[s % A] = read(s + A);
        gg_sched_fence();
    }
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

// Keys j0 .. j0 + 63 from memory to LDS by DMA: four waves, D / 32 instructions each. Rows from `len` on are deposited as zeros by the
// buffer's bounds check. voff[] = ggw_dma_offsets.
template <int D>
GG_DEVICE void ggw_dma_offsets(unsigned* voff, unsigned stride) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const int v = threadIdx.x + 256 * i, row = v / (D / 8), c = v % (D / 8);
        voff[i] = row * stride * 2 + ((c ^ ggw_swz<D>(row)) << 4);
    }
}
template <int D>
GG_DEVICE void ggw_dma(const unsigned short* base, int j0, int len, unsigned stride, const unsigned* voff, char* tile, int wave) {
    const int last = len - 1 - j0 < 63 ? len - 1 - j0 : 63;                 // the tile's last row that exists
    const GgBufS buf = gg_make_bufs(base + (unsigned long long)(unsigned)j0 * stride, last < 0 ? 0u : (last * stride + D) * 2);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) gg_bufs_load_lds16(buf, voff[i], 0, tile + (wave + 4 * i) * 1024);
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

// keys j0 .. j0 + 63 that this lane's row sees, key mask apart, as bits
GG_DEVICE unsigned long long ggw_view(const GgwWave& w, int sinks, int j0) {
    const int hi = w.hi - j0 < 63 ? w.hi - j0 : 63, lo = w.lo - j0, s = sinks - j0;
    if (hi < 0) return 0;
    const unsigned long long up = ~0ull >> (63 - hi);
    return up & ((lo <= 0 ? ~0ull : lo > 63 ? 0ull : ~0ull << lo) | (s <= 0 ? 0ull : s > 63 ? ~0ull : (1ull << s) - 1));
}
// scores that their row does not see become -inf; keep: this item's key mask or null. saw: the row saw a key. Without a key mask every row
// that is there sees the key at its own position; with one no tile is whole, and this looks.
GG_DEVICE void ggw_mask(f32x16* st, int blocks, const GgwWave& w, int sinks, int j0, int len, const unsigned char* keep, bool& saw) {
    const int lane = threadIdx.x & 63, hi = lane >> 5;
    unsigned long long bits = ~0ull;
    if (keep) {
        bits = gg_ballot(j0 + lane < len && keep[j0 + lane]);
        saw |= (bits & ggw_view(w, sinks, j0)) != 0;
    }
    bits >>= 4 * hi;
#pragma unroll
    for (int jb = 0; jb < 2; ++jb)
        if (jb < blocks) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int jr = jb * 32 + (r & 3) + 8 * (r >> 2);
                const bool see = ggw_sees(w, sinks, j0 + jr + 4 * hi) && ((bits >> jr) & 1);
                st[jb][r] = see ? st[jb][r] : -__builtin_inff();
            }
        }
}
// one softmax step over N 32-key blocks of scores: running maximum m (log2 domain), this lane's part of the row's sum l, the probabilities
// packed as the next product's operands. The maximum moves (and O with it) only when a score exceeds it by TAU.
template <int T, int DB, int N>
GG_DEVICE void ggw_softmax(f32x16* st, u16x8* pf, f32x16* ot, float& m, float& l, float a2) {
    float mx = -__builtin_inff();
#pragma unroll
    for (int jb = 0; jb < N; ++jb)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[jb][r]);
    mx = gg_max_xor32(mx) * a2;
    if (gg_wave_any(mx > m + GgwExp<T>::TAU)) {
        const float mn = fmaxf(m, mx - GgwExp<T>::LEAD), corr = gg_exp2f(m - mn);
        l *= corr;
        m = mn;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) ot[db][r] *= corr;
    }
    float sum = 0.f;
#pragma unroll
    for (int jb = 0; jb < N; ++jb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            st[jb][r] = gg_exp2f(gg_fmaf(st[jb][r], a2, -m));
            sum += st[jb][r];
        }
    l += sum;
#pragma unroll
    for (int jc = 0; jc < 2 * N; ++jc) pf[jc] = ggw_pack8<T>(st[jc >> 1], jc & 1);
}
// four features of o; o_lo (training): what the rounding took off, for D (a row of few keys has dP close to D, and half a step of o in
// D is then as large as their difference)
template <int T>
GG_DEVICE void ggw_store_o(const GgWinParams& p, long long at, f32x4 x) {
    u16x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        // (what is stored and what is taken off are one conversion: left to itself the compiler rounds the product with 1 / l to half twice,
        // fused for the store and from fp32 for the difference, and near a tie the two are a unit in the last place apart)
        unsigned h = gg_elt<T>(x[e]);
        gg_opaque(h);
        hi[e] = (unsigned short)h;
        lo[e] = gg_elt<T>(x[e] - gg_elt_f<T>((unsigned short)h));
    }
    *(u16x4*)(p.o + at) = hi;
    if (p.o_lo) *(u16x4*)(p.o_lo + at) = lo;
}
// A row that saw no key: zeros, and +inf for its log-sum-exp (its P is zero everywhere in the backward). A row that saw keys and has
// l = 0 saw scores of -inf alone: NaN. Where a row's parts are joined, one that saw no key has the maximum -inf in all of them, any other
// GGW_LOW or more in some.
GG_DEVICE float ggw_inverse(float l, bool saw) { return l == 0.f ? (saw ? __builtin_nanf("") : 0.f) : 1.f / l; }
GG_DEVICE bool ggw_far(float m) { return fabsf(m) >= GGW_FAR && fabsf(m) < __builtin_inff(); }
GG_DEVICE float ggw_lse(float m, float l, bool saw) {
    if (l == 0.f) return saw ? __builtin_nanf("") : __builtin_inff();
    return l == l && ggw_far(m) ? m : m + log2f(l);
}
// the wave's 32 rows: o and the log-sum-exp, or (SPLIT) what gg_win_join_kernel takes
template <int T, int D, bool SPLIT>
GG_DEVICE void ggw_write_rows(const GgWinParams& p, const GgwWave& w, int bkv, int split, const f32x16* ot, float m, float l, bool saw) {
    const int hi = (threadIdx.x & 63) >> 5, rows = p.n * p.g;
    l = gg_sum_xor32(l);
    if (w.r >= rows) return;
    const long long at = (long long)bkv * rows + w.r;
    if (SPLIT) {
        const long long sp = (long long)split * p.B * p.hk * rows + at;
        float* po = p.part_o + sp * D;
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int gq = 0; gq < 4; ++gq)
                *(f32x4*)(po + db * 32 + 8 * gq + 4 * hi) = f32x4{ot[db][4 * gq], ot[db][4 * gq + 1], ot[db][4 * gq + 2], ot[db][4 * gq + 3]};
        if (hi == 0) { p.part_ml[2 * sp] = saw ? m : -__builtin_inff(); p.part_ml[2 * sp + 1] = l; }
        return;
    }
    const int b = bkv / p.hk, kvh = bkv - b * p.hk;
    const float inv = ggw_inverse(l, saw);
    const long long orow = (((long long)b * p.n + w.row.token) * p.h + kvh * p.g + w.row.head) * D;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int gq = 0; gq < 4; ++gq)
            ggw_store_o<T>(p, orow + db * 32 + 8 * gq + 4 * hi, f32x4{ot[db][4 * gq] * inv, ot[db][4 * gq + 1] * inv, ot[db][4 * gq + 2] * inv, ot[db][4 * gq + 3] * inv});
    if (hi == 0 && p.lse) p.lse[at] = ggw_lse(m, l, saw);
}
template <int KK>
GG_DEVICE void ggw_load_row(u16x8* f, const unsigned short* base, long long head_stride, unsigned token_stride, int head, int token) {
    const unsigned short* r = base + (long long)head * head_stride + (long long)token * token_stride + 8 * ((threadIdx.x & 63) >> 5);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) f[kk] = *(const u16x8*)(r + kk * 16);
}

template <int T, int D>
GG_DEVICE float ggw_dot(const unsigned short* x, const unsigned short* y) {
    float s = 0.f;
    for (int c = 0; c < D; c += 8) {
        const u16x8 a = *(const u16x8*)(x + c), b = *(const u16x8*)(y + c);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = gg_fmaf(gg_elt_f<T>(a[e]), gg_elt_f<T>(b[e]), s);
    }
    return s;
}
// a score in log2 units, rounded before anything is taken from it (the same bits for a pair wherever it is computed again)
template <int T, int D>
GG_DEVICE float ggw_score(const unsigned short* q, const unsigned short* k, float a2) {
#pragma clang fp contract(off)
    const float s = ggw_dot<T, D>(q, k);
    return s * a2;
}
// One row again, by one wave, from the keys it sees alone: tiles i0, i0 + step .. of TK keys, a key a lane for the scores, a feature a lane
// for the output. fix[D] = sum of p v, relative to the maximum m, l the sum of p.
template <int T, int D, int TK>
GG_DEVICE void ggw_fix_row(const GgWinParams& p, const GgwRange& rg, int len, const unsigned char* keep, const unsigned short* q,
                           const unsigned short* kb, const unsigned short* vb, int pos, int i0, int i1, int step, float* fix, float& m, float& l) {
    constexpr int C = (D + 63) / 64;
    const int lane = threadIdx.x & 63;
    const float a2 = p.scale * GGW_LOG2E;
    float acc[C];
    m = GGW_LOW;
    l = 0.f;
    for (int c = 0; c < C; ++c) acc[c] = 0.f;
    for (int i = i0; i < i1; i += step) {
        const int j0 = ggw_tile_at(rg, i) * TK, j = j0 + lane;
        const bool see = lane < TK && j < len && j <= pos + p.right && (j >= pos - p.left || j < p.sinks) && (!keep || keep[j]);
        const float x = see ? ggw_score<T, D>(q, kb + (long long)j * p.kn, a2) : -__builtin_inff();
        float mx = x;
        for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, gg_shfl_xor(mx, o));
        const float mn = fmaxf(m, mx), corr = gg_exp2f(m - mn), pj = see ? gg_exp2f(x - mn) : 0.f;
        l = l * corr + gg_wave_sum_all(pj);
        m = mn;
        for (int c = 0; c < C; ++c) acc[c] *= corr;
        const unsigned long long bits = gg_ballot(see);         // (not where p > 0: a NaN value counts where its probability underflows too)
        for (int k = 0; k < TK; ++k) {
            const float pk = gg_readlane(pj, k);
            if (!((bits >> k) & 1)) continue;
            for (int c = 0; c < C; ++c)
                if (lane + 64 * c < D) acc[c] += pk * gg_elt_f<T>(vb[(long long)(j0 + k) * p.vn + lane + 64 * c]);
        }
    }
    for (int c = 0; c < C; ++c)
        if (lane + 64 * c < D) fix[lane + 64 * c] = acc[c];
}
// its values into the registers of the lanes that own the row
template <int DB>
GG_DEVICE void ggw_take_fix(f32x16* v, const float* fix, bool mine) {
    const int hi = (threadIdx.x & 63) >> 5;
    gg_wave_sync();
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float x = fix[db * 32 + (r & 3) + 8 * (r >> 2) + 4 * hi];
            v[db][r] = mine ? x : v[db][r];
        }
    gg_wave_sync();
}
template <int T, int D, int TK>
GG_DEVICE void ggw_fix_rows(const GgWinParams& p, const GgwWave& w, const GgwRange& rg, int len, int b, int kvh, const unsigned char* keep, int i0,
                            int i1, int step, unsigned bad, float* fix, f32x16* ot, float& m, float& l) {
    const int lane = threadIdx.x & 63, rows = p.n * p.g;
    for (int k = 0; k < 32; ++k) {
        if (!((bad >> k) & 1) || w.r0 + k >= rows) continue;
        const int token = (w.r0 + k) / p.g, head = w.r0 + k - token * p.g, pos = token + len - p.n;
        float fm, fl;
        ggw_fix_row<T, D, TK>(p, rg, len, keep, p.q + b * p.qb + (long long)(kvh * p.g + head) * p.qh + (long long)token * p.qn,
                              p.k + b * p.kb + kvh * p.kh, p.v + b * p.vb + kvh * p.vh, pos < 0 ? -2 * GGW_NONE : pos, i0, i1, step, fix, fm, fl);
        const bool mine = (lane & 31) == k;
        ggw_take_fix<D / 32>(ot, fix, mine);
        if (mine) {
            m = fm;
            l = lane < 32 ? fl : 0.f;
        }
    }
}

// workgroup: 4 waves x 32 rows; key tiles of 64 fetched once for all of them by LDS-DMA, double buffered: one barrier a tile, behind
// which the next tile's transfers start and run under this tile's arithmetic. No unit bounds it alone (32768 tokens, window 4096, 32 heads
// on 8 of 128: matrix pipe busy 54 % of the time, vector ALU 52 %, two waves a SIMD; without the operand reads from the LDS - a kilobyte
// a product - 1515 of 2145 us, without the softmax 1751, without the transfers 1875); at 64 features the softmax leads (vector ALU
// 62 %, matrix pipe 32 %). Measured and
// not kept: two 32-row blocks a wave for each operand read (half the reads, but one wave a SIMD: 2604 against 2010 in the same run),
// eight waves a tile in two groups half a tile apart (2334 against 2114), wave priorities (no change).
// SPLIT: the tiles are dealt out to p.splits workgroups, which leave (m, l, O) for gg_win_join_kernel.
template <int T, int D, bool SPLIT>
GG_KERNEL GG_LAUNCH_BOUNDS2(256, D == 128 ? 2 : 3) void gg_win_fwd_kernel(GgWinParams p) {
    constexpr int KK = D / 16, DB = D / 32;
    GG_SHARED __attribute__((aligned(1024))) char sK[2][GgwTile<D>::BYTES];
    GG_SHARED __attribute__((aligned(1024))) char sV[2][GgwTile<D>::BYTES];
    GG_SHARED float sFix[4][D];

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

    const unsigned char* keep = p.keep ? p.keep + b * p.keep_b : nullptr;
    const GgwWave w = ggw_wave(p, r0 + wave * 32, len, keep != nullptr);
    const unsigned short* kb = p.k + b * p.kb + kvh * p.kh;
    const unsigned short* vb = p.v + b * p.vb + kvh * p.vh;
    u16x8 qf[KK];
    ggw_load_row<KK>(qf, p.q + b * p.qb, p.qh, p.qn, kvh * p.g + w.row.head, w.row.token);
    unsigned ko[D / 32], vo[D / 32];
    ggw_dma_offsets<D>(ko, p.kn);
    ggw_dma_offsets<D>(vo, p.vn);
    auto fetch = [&](int i, int buf) {
        const int j0 = ggw_tile_at(rg, i) * 64;
        ggw_dma<D>(kb, j0, len, p.kn, ko, sK[buf], wave);
        ggw_dma<D>(vb, j0, len, p.vn, vo, sV[buf], wave);
    };
    const float a2 = p.scale * GGW_LOG2E;
    float m = GGW_LOW, l = 0.f;
    bool saw = w.row.in && !keep;
    f32x16 ot[DB], st[2];
    u16x8 pf[4];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) ot[db][r] = 0.f;
    const GgwLane lanes = ggw_lane<D>();
    gg_wait_vm<0>();                // (the rows above: the transfers' count starts at zero)
    if (ta < tb) fetch(ta, 0);
    for (int i = ta, buf = 0; i < tb; ++i, buf ^= 1) {
        const int j0 = ggw_tile_at(rg, i) * 64;
        gg_wait_vm<0>();
        gg_barrier_lds();           // this tile is there for everyone, and everyone is through with the last one: its buffer is free
        if (i + 1 < tb) fetch(i + 1, buf ^ 1);
        if (!ggw_some(w, p.sinks, j0, j0 + 63)) continue;
        const GgwLane lo = ggw_here(lanes);
#pragma unroll
        for (int r = 0; r < 16; ++r) st[0][r] = st[1][r] = 0.f;
        ggw_pipe<2 * KK>([&](int s) { return ggw_frag<D>(sK[buf], (s & 1) * 32, s >> 1, lo); },
                         [&](int s, u16x8 x) { st[s & 1] = ggw_mfma<T>(x, qf[s >> 1], st[s & 1]); });
        if (!ggw_whole(w, p.sinks, j0, j0 + 63)) ggw_mask(st, 2, w, p.sinks, j0, len, keep, saw);
        ggw_softmax<T, DB, 2>(st, pf, ot, m, l, a2);
        ggw_pipe<4 * DB>([&](int s) { return ggw_frag_tr<D>(sV[buf], (s % DB) * 32, 16 * (s / DB), lo); },
                         [&](int s, u16x8 x) { ot[s % DB] = ggw_mfma<T>(x, pf[s / DB], ot[s % DB]); });
    }
    const unsigned bad = ggw_not_finite<DB>(ot) | ggw_rows32(saw && ggw_far(m));
    if (__builtin_expect(bad != 0, 0)) ggw_fix_rows<T, D, 64>(p, w, rg, len, b, kvh, keep, ta, tb, 1, bad, sFix[wave], ot, m, l);
    ggw_write_rows<T, D, SPLIT>(p, w, bkv, split, ot, m, l, saw);
}

// ---- forward with few rows ------------------------------------------------------------------------------------------
// One new token: a handful of rows against a long cache - bound by reading K and V once. The four waves share the 32 rows and take key
// tiles of 32 in turn, each on its own: K goes from memory straight into the score product's operand registers, V through a wave-private
// LDS tile (the transpose read), no barrier in the loop; the waves' (m, l, O) are joined in LDS at the end, the splits' by
// gg_win_join_kernel. 64 sequences, 8 key heads of 128, window 4096: 199 us (5.2 TB/s).
template <int T, int D>
GG_KERNEL GG_LAUNCH_BOUNDS2(256, 2) void gg_win_few_kernel(GgWinParams p) {
    constexpr int KK = D / 16, DB = D / 32;
    GG_SHARED __attribute__((aligned(16))) char sV[4][32 * D * 2];
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
    const unsigned char* keep = p.keep ? p.keep + b * p.keep_b : nullptr;
    const GgwWave w = ggw_wave(p, r0, len, keep != nullptr);
    const unsigned short* kb = p.k + b * p.kb + kvh * p.kh;
    const unsigned short* vb = p.v + b * p.vb + kvh * p.vh;
    u16x8 qf[KK], pf[2];
    ggw_load_row<KK>(qf, p.q + b * p.qb, p.qh, p.qn, kvh * p.g + w.row.head, w.row.token);
    const float a2 = p.scale * GGW_LOG2E;
    float m = GGW_LOW, l = 0.f;
    bool saw = w.row.in && !keep;
    f32x16 ot[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) ot[db][r] = 0.f;

    u16x8 kf[KK], vr[D / 16];
    auto load = [&](int i) {        // (0 <= khi < len: the clamped rows exist; what they hold meets a masked score)
        const int j0 = ggw_tile_at(rg, i) * 32, j = j0 + (lane & 31);
        ggw_load_row<KK>(kf, kb, 0, p.kn, 0, j <= rg.khi ? j : rg.khi);
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
            const int v = lane + 64 * s, jv = j0 + v / (D / 8), c8 = v % (D / 8);
            vr[s] = *(const u16x8*)(vb + (long long)(jv <= rg.khi ? jv : rg.khi) * p.vn + c8 * 8);
        }
    };
    const GgwLane lo = ggw_lane<D>();
    if (ta + wave < tb) load(ta + wave);
    for (int i = ta + wave; i < tb; i += 4) {
        const int j0 = ggw_tile_at(rg, i) * 32;
        gg_wave_sync();
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
            const int v = lane + 64 * s, vrow = v / (D / 8);
            *(u16x8*)(sV[wave] + vrow * D * 2 + (((v % (D / 8)) ^ ggw_swz<D>(vrow)) << 4)) = vr[s];
        }
        gg_wave_sync();
        f32x16 st;
#pragma unroll
        for (int r = 0; r < 16; ++r) st[r] = 0.f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) st = ggw_mfma<T>(kf[kk], qf[kk], st);
        if (i + 4 < tb) load(i + 4);
        if (!ggw_whole(w, p.sinks, j0, j0 + 31)) ggw_mask(&st, 1, w, p.sinks, j0, len, keep, saw);
        ggw_softmax<T, DB, 1>(&st, pf, ot, m, l, a2);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int db = 0; db < DB; ++db) ot[db] = ggw_mfma<T>(ggw_frag_tr<D>(sV[wave], db * 32, 16 * c, lo), pf[c], ot[db]);
    }
    const unsigned bad = ggw_not_finite<DB>(ot) | ggw_rows32(saw && ggw_far(m));
    if (__builtin_expect(bad != 0, 0)) {
        gg_wave_sync();             // (the wave's own tile is free)
        ggw_fix_rows<T, D, 32>(p, w, rg, len, b, kvh, keep, ta + wave, tb, 4, bad, (float*)sV[wave], ot, m, l);
    }
    l = gg_sum_xor32(l);
    if (hi == 0) { sM[wave][lane] = saw ? m : -__builtin_inff(); sL[wave][lane] = l; }
    gg_sync();
    const int q = lane & 31;
    float top = GGW_LOW;
    for (int w = 0; w < 4; ++w) top = fmaxf(top, sM[w][q]);
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
        const bool any = mt >= GGW_LOW;
        for (int w = 0; w < 4; ++w) lt += sL[w][rr] * gg_exp2f(sM[w][rr] - fmaxf(mt, GGW_LOW));
        const f32x4 x = *(const f32x4*)&sO[rr][d];
        const long long at = (long long)bkv * rows + r;
        if (p.splits > 1) {
            const long long sp = (long long)split * p.B * p.hk * rows + at;
            *(f32x4*)(p.part_o + sp * D + d) = x;
            if (d == 0) { p.part_ml[2 * sp] = mt; p.part_ml[2 * sp + 1] = lt; }
        } else {
            const float inv = ggw_inverse(lt, any);
            const int token = (int)((unsigned)r / (unsigned)p.g), head = r - token * p.g;
            ggw_store_o<T>(p, (((long long)b * p.n + token) * p.h + kvh * p.g + head) * D + d, x * inv);
            if (d == 0 && p.lse) p.lse[at] = ggw_lse(mt, lt, any);
        }
    }
}

// The splits' (m, l, O) of a row joined: four features a thread, p.join groups of threads a row that share its splits (few rows and many
// splits: a thread that walked them all would wait for memory a dozen times over), the groups' sums added in order in LDS.
template <int T, int D>
GG_KERNEL GG_LAUNCH_BOUNDS(256) void gg_win_join_kernel(GgWinParams p) {
    constexpr int Q = D / 4, R = 256 / Q;                   // threads a group, groups a workgroup
    GG_SHARED __attribute__((aligned(16))) float sO[R][D + 4];
    GG_SHARED float sM[R], sL[R];
    const int rows = p.n * p.g, grp = threadIdx.x / Q, d = threadIdx.x % Q * 4, share = grp % p.join;
    const long long all = (long long)p.B * p.hk * rows;
    const long long at0 = (long long)blockIdx.x * (R / p.join) + grp / p.join, at = at0 < all ? at0 : all - 1;
    float top = -__builtin_inff();
#pragma unroll 4
    for (int s = share; s < p.splits; s += p.join) top = fmaxf(top, p.part_ml[2 * (s * all + at)]);
    float base = fmaxf(top, GGW_LOW);
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
#pragma unroll 4
    for (int s = share; s < p.splits; s += p.join) {
        const float f = gg_exp2f(p.part_ml[2 * (s * all + at)] - base);
        l += f * p.part_ml[2 * (s * all + at) + 1];
        x += f * *(const f32x4*)(p.part_o + (s * all + at) * D + d);
    }
    if (p.join > 1) {
        *(f32x4*)&sO[grp][d] = x;
        if (d == 0) { sM[grp] = top; sL[grp] = l; }
        gg_sync();
        if (share) return;
        for (int k = 1; k < p.join; ++k) top = fmaxf(top, sM[grp + k]);
        base = fmaxf(top, GGW_LOW);
        x = f32x4{0.f, 0.f, 0.f, 0.f};
        l = 0.f;
        for (int k = 0; k < p.join; ++k) {
            const float f = gg_exp2f(sM[grp + k] - base);
            l += f * sL[grp + k];
            x += f * *(const f32x4*)&sO[grp + k][d];
        }
    }
    if (at0 >= all) return;
    const bool saw = top >= GGW_LOW;
    const float inv = ggw_inverse(l, saw);
    const int bkv = (int)(at / rows), r = (int)(at - (long long)bkv * rows);
    const int b = bkv / p.hk, kvh = bkv - b * p.hk, token = r / p.g, head = r - token * p.g;
    ggw_store_o<T>(p, (((long long)b * p.n + token) * p.h + kvh * p.g + head) * D + d, x * inv);
    if (d == 0 && p.lse) p.lse[at] = ggw_lse(top, l, saw);
}

// ---- backward, part 1: dq and D ---------------------------------------------------------------------------------------
// the forward's mapping and transfers; K is read as rows (scores) and transposed (dq), V as rows (dP)
template <int T, int D>
GG_DEVICE void ggw_write_dq(const GgWinParams& p, const GgwWave& w, int b, int hq, const f32x16* dqt) {
    if (w.r >= p.n * p.g) return;
    unsigned short* row = p.dq + (((long long)b * p.n + w.row.token) * p.h + hq) * D + 4 * ((threadIdx.x & 63) >> 5);
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int gq = 0; gq < 4; ++gq) {
            u16x4 o4;
#pragma unroll
            for (int e = 0; e < 4; ++e) o4[e] = gg_elt<T>(dqt[db][4 * gq + e] * p.scale);
            *(u16x4*)(row + db * 32 + 8 * gq) = o4;
        }
}
// dS (times 2^e where neg_lse = e - lse) of one 32-key block from its scores and dP - D, in the scores' place
GG_DEVICE void ggw_ds(f32x16& st, const f32x16& dp, float a2, float neg_lse, bool masked, const GgwWave& w, int sinks, int j, unsigned long long bits) {
#pragma unroll
    for (int r = 0; r < 16; ++r) st[r] = gg_exp2f(gg_fmaf(st[r], a2, neg_lse)) * dp[r];
    if (masked) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int jr = (r & 3) + 8 * (r >> 2);
            st[r] = ggw_sees(w, sinks, j + jr) && ((bits >> jr) & 1) ? st[r] : 0.f;
        }
    }
}

// one row's dq again, by one wave, from the keys it sees alone: fix[D] = sum of dS k. Of a far row (lse its largest score) log2 of the
// sum first, which is returned.
template <int T, int D>
GG_DEVICE float ggw_fix_dq(const GgWinParams& p, const GgwRange& rg, int len, const unsigned char* keep, const unsigned short* q,
                          const unsigned short* g, const unsigned short* kb, const unsigned short* vb, int pos, float lse, float dsum, float* fix) {
    constexpr int C = (D + 63) / 64;
    const int lane = threadIdx.x & 63;
    const float a2 = p.scale * GGW_LOG2E;
    float acc[C];
    for (int c = 0; c < C; ++c) acc[c] = 0.f;
    auto sees = [&](int j) { return j < len && j <= pos + p.right && (j >= pos - p.left || j < p.sinks) && (!keep || keep[j]); };
    float log_sum = 0.f;
    if (ggw_far(lse)) {
        for (int i = 0; i < rg.nt; ++i) {
            const int j = ggw_tile_at(rg, i) * 64 + lane;
            log_sum += gg_wave_sum_all(sees(j) ? gg_exp2f(ggw_score<T, D>(q, kb + (long long)j * p.kn, a2) - lse) : 0.f);
        }
        log_sum = log2f(log_sum);
    }
    for (int i = 0; i < rg.nt; ++i) {
        const int j0 = ggw_tile_at(rg, i) * 64, j = j0 + lane;
        const bool see = sees(j);
        float ds = 0.f;
        if (see) ds = gg_exp2f(ggw_score<T, D>(q, kb + (long long)j * p.kn, a2) - lse - log_sum) * (ggw_dot<T, D>(g, vb + (long long)j * p.vn) - dsum);
        const unsigned long long bits = gg_ballot(see);
        for (int k = 0; k < 64; ++k) {
            const float dk = gg_readlane(ds, k);
            if (!((bits >> k) & 1)) continue;
            for (int c = 0; c < C; ++c)
                if (lane + 64 * c < D) acc[c] += dk * gg_elt_f<T>(kb[(long long)(j0 + k) * p.kn + lane + 64 * c]);
        }
    }
    for (int c = 0; c < C; ++c)
        if (lane + 64 * c < D) fix[lane + 64 * c] = acc[c];
    return log_sum;
}

template <int T, int D>
GG_KERNEL GG_LAUNCH_BOUNDS2(256, 2) void gg_win_dq_kernel(GgWinParams p) {
    constexpr int KK = D / 16, DB = D / 32;
    GG_SHARED __attribute__((aligned(1024))) char sK[2][GgwTile<D>::BYTES];
    GG_SHARED __attribute__((aligned(1024))) char sV[2][GgwTile<D>::BYTES];
    GG_SHARED float sFix[4][D];

    const int lane = threadIdx.x & 63, wave = gg_uniform(threadIdx.x >> 6), hi = lane >> 5;
    const int item = ggw_item();
    const int bkv = item / p.row_tiles, tile = item - bkv * p.row_tiles;
    const int b = bkv / p.hk, kvh = bkv - b * p.hk;
    const int rows = p.n * p.g;
    const int len = ggw_len(p, b);
    const int r0 = tile * 128, rl = r0 + 127 < rows - 1 ? r0 + 127 : rows - 1;
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
    ggw_load_row<KK>(qf, p.q + b * p.qb, p.qh, p.qn, hq, w.row.token);
    ggw_load_row<KK>(gf, p.d_o + b * p.gb, p.gh, p.gn, hq, w.row.token);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
        const u16x8 of = *(const u16x8*)(p.o + orow + 8 * hi + kk * 16), ol = *(const u16x8*)(p.o_lo + orow + 8 * hi + kk * 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) dsum = gg_fmaf(gg_elt_f<T>(gf[kk][e]), gg_elt_f<T>(of[e]) + gg_elt_f<T>(ol[e]), dsum);
    }
    dsum = gg_sum_xor32(dsum);
    const float lse = p.lse[at], a2 = p.scale * GGW_LOG2E;
    if (hi == 0 && w.r < rows) p.dvec[at] = dsum;
    unsigned ko[D / 32], vo[D / 32];
    ggw_dma_offsets<D>(ko, p.kn);
    ggw_dma_offsets<D>(vo, p.vn);
    auto fetch = [&](int i, int buf) {
        const int j0 = ggw_tile_at(rg, i) * 64;
        ggw_dma<D>(kb, j0, len, p.kn, ko, sK[buf], wave);
        ggw_dma<D>(vb, j0, len, p.vn, vo, sV[buf], wave);
    };
    GgwScale sc = {64};
    f32x16 dqt[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) dqt[db][r] = 0.f;
    const GgwLane lanes = ggw_lane<D>();
    gg_wait_vm<0>();                // (the rows above: the transfers' count starts at zero)
    if (rg.nt > 0) fetch(0, 0);
    for (int i = 0, buf = 0; i < rg.nt; ++i, buf ^= 1) {
        const int j0 = ggw_tile_at(rg, i) * 64;
        gg_wait_vm<0>();
        gg_barrier_lds();           // this tile is there for everyone, and everyone is through with the last one: its buffer is free
        if (i + 1 < rg.nt) fetch(i + 1, buf ^ 1);
        if (!ggw_some(w, p.sinks, j0, j0 + 63)) continue;
        const bool masked = !ggw_whole(w, p.sinks, j0, j0 + 63);
        unsigned long long bits = ~0ull;
        if (keep) bits = gg_ballot(j0 + lane < len && keep[j0 + lane]);
        bits >>= 4 * hi;
#pragma unroll
        for (int jb = 0; jb < 2; ++jb) {
            f32x16 st, dp;
            const GgwLane lo = ggw_here(lanes);
            // scores and dP in turn, then dq: one stream of operands from the LDS each
            ggw_pipe<2 * KK>([&](int s) { return ggw_frag<D>(s & 1 ? sV[buf] : sK[buf], jb * 32, s >> 1, lo); },
                             [&](int s, u16x8 x) {
                                 if (s < 2) {
#pragma unroll
                                     for (int r = 0; r < 16; ++r) (s ? dp : st)[r] = s ? -dsum : 0.f;
                                 }
                                 if (s & 1) dp = ggw_mfma<T>(x, gf[s >> 1], dp);
                                 else st = ggw_mfma<T>(x, qf[s >> 1], st);
                             });
            ggw_ds(st, dp, a2, T == GG_ELT_F16 ? (float)sc.e - lse : -lse, masked, w, p.sinks, j0 + jb * 32 + 4 * hi, bits >> (jb * 32));
            if constexpr (T == GG_ELT_F16) ggw_rescale<DB>(sc, st, dqt);
            const u16x8 sf[2] = {ggw_pack8<T>(st, 0), ggw_pack8<T>(st, 1)};
            ggw_pipe<2 * DB>([&](int s) { return ggw_frag_tr<D>(sK[buf], (s % DB) * 32, jb * 32 + 16 * (s / DB), lo); },
                             [&](int s, u16x8 x) { dqt[s % DB] = ggw_mfma<T>(x, sf[s / DB], dqt[s % DB]); });
        }
    }
    if constexpr (T == GG_ELT_F16)
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) dqt[db][r] *= ggw_pow2(-sc.e);
    const unsigned bad = ggw_not_finite<DB>(dqt) | ggw_rows32(ggw_far(lse));
    if (__builtin_expect(bad != 0, 0))
        for (int k = 0; k < 32; ++k) {
            if (!((bad >> k) & 1) || w.r0 + k >= rows) continue;
            const int token = (w.r0 + k) / p.g, head = kvh * p.g + w.r0 + k - token * p.g, pos = token + len - p.n;
            const float log_sum = ggw_fix_dq<T, D>(
                             p, rg, len, keep, p.q + b * p.qb + head * p.qh + (long long)token * p.qn,
                             p.d_o + b * p.gb + head * p.gh + (long long)token * p.gn, kb, vb, pos < 0 ? -2 * GGW_NONE : pos, gg_readlane(lse, k),
                             gg_readlane(dsum, k), sFix[wave]);
            if (lane == 0) p.dvec[(long long)p.B * p.hk * rows + (long long)bkv * rows + w.r0 + k] = log_sum;
            ggw_take_fix<DB>(dqt, sFix[wave], (lane & 31) == k);
        }
    ggw_write_dq<T, D>(p, w, b, hq, dqt);
}

// ---- backward, part 2: dk, dv -----------------------------------------------------------------------------------------
// the rows ra .. rb that see some key of the 128-key tile at k0, or their part `chunk` of `chunks` (whole 64-row tiles); none: ra > rb.
// Compared as tokens before they become rows: keys far in front of every query are a token that, times g, 32 bits do not hold.
struct GgwRows { int ra, rb; };
GG_HOST_DEVICE GgwRows ggw_rows(const GgWinParams& p, int len, int k0, int chunk, int chunks) {
    GgwRows r = {0, -1};
    const int shift = len - p.n, klast = k0 + 127 < len - 1 ? k0 + 127 : len - 1;
    int tlo = k0 - p.right - shift, thi = klast + p.left - shift;
    if (k0 < p.sinks || thi > p.n - 1) thi = p.n - 1;
    if (tlo < -shift) tlo = -shift;
    if (tlo < 0) tlo = 0;
    if (klast < k0 || thi < tlo) return r;
    r.ra = tlo * p.g;
    r.rb = thi * p.g + p.g - 1;
    if (chunks > 1) {
        const long long nt = ((long long)r.rb - r.ra + 64) / 64, c0 = nt * chunk / chunks, c1 = nt * (chunk + 1) / chunks;
        const int z = r.ra + (int)(c1 * 64 - 1);
        r.ra += (int)(c0 * 64);
        r.rb = z < r.rb ? z : r.rb;
    }
    return r;
}
// one key's dk and dv again, by one wave, from the rows ra .. rb that see it alone: fix[2 D] = sum of dS q, sum of P dO
template <int T, int D>
GG_DEVICE void ggw_fix_dkv(const GgWinParams& p, const unsigned short* qb, const unsigned short* gb, const unsigned short* k, const unsigned short* v,
                           int j, int shift, long long stat, int ra, int rb, float* fix) {
    constexpr int C = (D + 63) / 64;
    const int lane = threadIdx.x & 63;
    const float a2 = p.scale * GGW_LOG2E;
    float dk[C], dv[C];
    for (int c = 0; c < C; ++c) dk[c] = dv[c] = 0.f;
    for (int i0 = ra; i0 <= rb; i0 += 64) {
        const int r = i0 + lane, rc = r <= rb ? r : rb, tok = rc / p.g, hd = rc - tok * p.g, pos = tok + shift;
        const float lse = p.lse[stat + rc];
        const bool see = r <= rb && lse < __builtin_inff() && j <= pos + p.right && (j >= pos - p.left || j < p.sinks);
        float pr = 0.f, ds = 0.f;
        if (see || (r <= rb && lse != lse)) {
            const long long qo = hd * p.qh + (long long)tok * p.qn, go = hd * p.gh + (long long)tok * p.gn;
            const float log_sum = ggw_far(lse) ? p.dvec[(long long)p.B * p.hk * p.n * p.g + stat + rc] : 0.f;
            pr = gg_exp2f(ggw_score<T, D>(qb + qo, k, a2) - lse - log_sum);
            ds = pr * (ggw_dot<T, D>(gb + go, v) - p.dvec[stat + rc]);
        }
        const unsigned long long bits = gg_ballot(r <= rb && !(lse == __builtin_inff()) && j <= pos + p.right && (j >= pos - p.left || j < p.sinks));
        for (int t = 0; t < 64; ++t) {
            const float st = gg_readlane(ds, t), pt = gg_readlane(pr, t);
            if (!((bits >> t) & 1)) continue;
            const int rt = i0 + t, tk = rt / p.g, h = rt - tk * p.g;
            const unsigned short* qr = qb + h * p.qh + (long long)tk * p.qn;
            const unsigned short* gr = gb + h * p.gh + (long long)tk * p.gn;
            for (int c = 0; c < C; ++c)
                if (lane + 64 * c < D) {
                    dk[c] += st * gg_elt_f<T>(qr[lane + 64 * c]);
                    dv[c] += pt * gg_elt_f<T>(gr[lane + 64 * c]);
                }
        }
    }
    for (int c = 0; c < C; ++c)
        if (lane + 64 * c < D) {
            fix[lane + 64 * c] = dk[c];
            fix[D + lane + 64 * c] = dv[c];
        }
}

// workgroup: 4 waves x 32 keys, row tiles of 64 (Q and dO by LDS-DMA, double buffered, each read as rows and transposed). The key tiles
// that hold sinks are seen by every later row: where the chip needs it their rows are cut into p.sink_chunks chunks, each a workgroup of
// its own that leaves fp32 sums for gg_win_sink_kernel; where there are few key tiles, every tile's are (gg_win_plan).
// part_o: [B*hk][sink_tiles][chunks][2][128][D].
template <int T, int D>
GG_KERNEL GG_LAUNCH_BOUNDS2(256, 2) void gg_win_dkv_kernel(GgWinParams p) {
    constexpr int KK = D / 16, DB = D / 32;
    GG_SHARED __attribute__((aligned(1024))) char sQ[2][GgwTile<D>::BYTES];
    GG_SHARED __attribute__((aligned(1024))) char sG[2][GgwTile<D>::BYTES];
    GG_SHARED __attribute__((aligned(16))) float sLse[2][64];
    GG_SHARED __attribute__((aligned(16))) float sD[2][64];
    GG_SHARED __attribute__((aligned(16))) int sPos[2][64];
    GG_SHARED float sFix[4][2 * D];

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

    const GgwRows rw = ggw_rows(p, len, k0, tile < p.sink_tiles ? chunk : 0, tile < p.sink_tiles ? p.sink_chunks : 1);
    const int ra = rw.ra, rb = rw.rb;

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
    // half: P for dv is 2^14 P (a constant does: P <= 1), dS = P (dP - D) 2^e
    constexpr int PE = T == GG_ELT_F16 ? 14 : 0;
    GgwScale sc = {64};

    const unsigned short* qb = p.q + b * p.qb + (long long)kvh * p.g * p.qh;
    const unsigned short* gb = p.d_o + b * p.gb + (long long)kvh * p.g * p.gh;
    // This thread's vectors of a row tile, as 32-bit offsets from the tile's first token (host: they fit). Where g divides 64 every tile
    // starts at a token's first head and the offsets stay what they are; else the vectors' (token, head) are kept up from tile to tile.
    constexpr int NV = D / 32;
    const int step_t = 64 / p.g, step_h = 64 - step_t * p.g;
    int vt[NV], vh[NV];
    unsigned oq[NV], og[NV];
    int ft = 0, fh = 0;                     // (uniform) the next tile's first row
    int rt = 0, rh = 0;                     // the row whose statistics this thread fetches (threads 0 .. 63)
    auto offsets = [&]() {
#pragma unroll
        for (int s = 0; s < NV; ++s) {
            const int v = threadIdx.x + 256 * s, c = (v % (D / 8)) ^ ggw_swz<D>(v / (D / 8));
            const unsigned dt = vt[s] - ft, dh = vh[s];
            oq[s] = (dt * p.qn + dh * (unsigned)p.qh) * 2 + (c << 4);
            og[s] = (dt * p.gn + dh * (unsigned)p.gh) * 2 + (c << 4);
            vt[s] += step_t;
            vh[s] += step_h;
            if (vh[s] >= p.g) { vh[s] -= p.g; ++vt[s]; }
        }
    };
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
        ft = (int)((unsigned)i0 / (unsigned)p.g);
        fh = i0 - ft * p.g;
        offsets();
    };
    const GgwLane lanes = ggw_lane<D>();
    float r_lse = 0.f, r_d = 0.f;
    int r_pos = 0;
    unsigned long long far = 0;             // (wave-uniform)
    auto fetch = [&](int i0, int buf) {
        const GgBufS bq = gg_make_bufs(qb + (unsigned long long)(unsigned)ft * p.qn, GGW_SPAN), bg = gg_make_bufs(gb + (unsigned long long)(unsigned)ft * p.gn, GGW_SPAN);
        const bool all = i0 + 63 <= rb;
#pragma unroll
        for (int s = 0; s < NV; ++s) {
            // (rows behind the last one: an offset that the buffer's bounds check turns into zeros)
            const bool in = all || i0 + (int)(threadIdx.x + 256 * s) / (D / 8) <= rb;
            gg_bufs_load_lds16(bq, in ? oq[s] : GGW_SPAN, 0, sQ[buf] + (wave + 4 * s) * 1024);
            gg_bufs_load_lds16(bg, in ? og[s] : GGW_SPAN, 0, sG[buf] + (wave + 4 * s) * 1024);
        }
        ft += step_t;
        fh += step_h;
        if (fh >= p.g) { fh -= p.g; ++ft; }
        if (step_t * p.g != 64) offsets();
    };
    const float *lse = p.lse + (long long)bkv * rows, *dvec = p.dvec + (long long)bkv * rows;
    auto stats = [&](int i0) {              // lse = +inf: a row that is not there or sees nothing
        const int r = i0 + (int)(threadIdx.x & 63);
        const bool in = r <= rb;
        const unsigned at = in ? r : rb;
        r_lse = in ? lse[at] : __builtin_inff();
        r_d = in ? dvec[at] : 0.f;
        r_pos = in ? rt + shift : -2 * GGW_NONE;
        rt += step_t;
        rh += step_h;
        if (rh >= p.g) { rh -= p.g; ++rt; }
    };
#pragma unroll
    for (int i = 0; i < 2 * DB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
    if (ra <= rb) {
        start(ra);
        stats(ra);
        gg_wait_vm<0>();            // (this wave's keys: the transfers' count starts at zero)
        fetch(ra, 0);
    }
    // a row's distance from its tile's first row to tokens: x / g for x < g + 64 by a reciprocal rounded up (exact: x g < 2^32, which the
    // host checks)
    const unsigned recip = p.g > 1 ? (unsigned)(0xffffffffu / (unsigned)p.g) + 1u : 0u;
    auto tokens = [&](int x) { return recip ? (int)(((unsigned long long)(unsigned)x * recip) >> 32) : x; };
    int ct = 0, ch = 0;
    if (ra <= rb) { ct = (int)((unsigned)ra / (unsigned)p.g); ch = ra - ct * p.g; }
    for (int i0 = ra, buf = 0; i0 <= rb; i0 += 64, buf ^= 1) {
        const int t0 = ct, h0 = ch;
        ct += step_t;
        ch += step_h;
        if (ch >= p.g) { ch -= p.g; ++ct; }
        far |= gg_ballot(ggw_far(r_lse));           // (not where it is loaded: nothing waits for it there)
        if (threadIdx.x < 64) { sLse[buf][threadIdx.x] = r_lse - (float)PE; sD[buf][threadIdx.x] = r_d; sPos[buf][threadIdx.x] = r_pos; }
        gg_wait_vm<0>();
        gg_barrier_lds();
        if (i0 + 64 <= rb) {
            stats(i0 + 64);
            fetch(i0 + 64, buf ^ 1);
        }
#pragma unroll
        for (int ib = 0; ib < 2; ++ib) {
            // the 32 rows' positions: all there, and the wave's 32 keys all seen by all of them?
            const int r1 = i0 + ib * 32 + 31;
            if (i0 + ib * 32 > rb) break;
            const int plo = t0 + tokens(h0 + ib * 32) + shift, phi = t0 + tokens(h0 + (r1 <= rb ? ib * 32 + 31 : rb - i0)) + shift;
            if (kj0 > phi + p.right || (wlast < plo - p.left && kj0 >= p.sinks) || kj0 >= len) continue;
            const bool full = whole && r1 <= rb && wlast <= plo + p.right && (kj0 >= phi - p.left || wlast < p.sinks);
            f32x16 st, dp;
            const GgwLane lo = ggw_here(lanes);
            ggw_pipe<2 * KK, D == 128 ? 2 : 4>([&](int s) { return ggw_frag<D>(s & 1 ? sG[buf] : sQ[buf], ib * 32, s >> 1, lo); },
                             [&](int s, u16x8 x) {
                                 if (s < 2) {
#pragma unroll
                                     for (int r = 0; r < 16; ++r) (s ? dp : st)[r] = 0.f;
                                 }
                                 if (s & 1) dp = ggw_mfma<T>(x, vf[s >> 1], dp);
                                 else st = ggw_mfma<T>(x, kf[s >> 1], st);
                             });
            const float ps = T == GG_ELT_F16 ? ggw_pow2(sc.e - PE) : 1.f;
#pragma unroll
            for (int gq = 0; gq < 4; ++gq) {
                const int at = ib * 32 + 8 * gq + 4 * hi;
                const f32x4 ls = *(const f32x4*)&sLse[buf][at], dd = *(const f32x4*)&sD[buf][at];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 4 * gq + e;
                    st[r] = gg_exp2f(gg_fmaf(st[r], a2, -ls[e]));
                    dp[r] = st[r] * (T == GG_ELT_F16 ? (dp[r] - dd[e]) * ps : dp[r] - dd[e]);
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
            if constexpr (T == GG_ELT_F16) ggw_rescale<DB>(sc, dp, dkt);
            const u16x8 pf[2] = {ggw_pack8<T>(st, 0), ggw_pack8<T>(st, 1)}, sf[2] = {ggw_pack8<T>(dp, 0), ggw_pack8<T>(dp, 1)};
            ggw_pipe<4 * DB, D == 128 ? 2 : 4>([&](int s) { return ggw_frag_tr<D>(s & 1 ? sQ[buf] : sG[buf], (s / 2 % DB) * 32, ib * 32 + 16 * (s / (2 * DB)), lo); },
                             [&](int s, u16x8 x) {
                                 const int db = s / 2 % DB, c = s / (2 * DB);
                                 if (s & 1) dkt[db] = ggw_mfma<T>(x, sf[c], dkt[db]);
                                 else dvt[db] = ggw_mfma<T>(x, pf[c], dvt[db]);
                             });
        }
    }
    if constexpr (T == GG_ELT_F16)
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                dkt[db][r] *= ggw_pow2(-sc.e);
                dvt[db][r] *= ggw_pow2(-PE);
            }
    const unsigned bad = far ? ~0u : ggw_not_finite<2 * DB>(acc);       // (a far row may have reached any key)
    if (__builtin_expect(bad != 0, 0))
        for (int k = 0; k < 32; ++k) {
            const int j = kj0 + k;
            if (!((bad >> k) & 1) || j >= len || (keep && !keep[j])) continue;          // (a key that nobody sees ends as zeros below)
            ggw_fix_dkv<T, D>(p, qb, gb, p.k + b * p.kb + kvh * p.kh + (long long)j * p.kn, p.v + b * p.vb + kvh * p.vh + (long long)j * p.vn, j, shift,
                              (long long)bkv * rows, ra, rb, sFix[wave]);
            ggw_take_fix<2 * DB>(acc, sFix[wave], (lane & 31) == k);
        }
    if (__builtin_expect(bad != 0, 0) && !kept) {
        for (int i = 0; i < 2 * DB; ++i)
            for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
    }
    if (chunked) {
        float* po = p.part_o + ((((long long)bkv * p.sink_tiles + tile) * p.sink_chunks + chunk) * 2 * 128 + wave * 32 + (lane & 31)) * D;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int gq = 0; gq < 4; ++gq) {
                const int d = db * 32 + 8 * gq + 4 * hi;
                *(f32x4*)(po + d) = f32x4{dkt[db][4 * gq], dkt[db][4 * gq + 1], dkt[db][4 * gq + 2], dkt[db][4 * gq + 3]};
                *(f32x4*)(po + 128 * D + d) = f32x4{dvt[db][4 * gq], dvt[db][4 * gq + 1], dvt[db][4 * gq + 2], dvt[db][4 * gq + 3]};
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
                k4[e] = gg_elt<T>(dkt[db][4 * gq + e] * p.scale);
                v4[e] = gg_elt<T>(dvt[db][4 * gq + e]);
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

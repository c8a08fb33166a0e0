// gg_transformer.hip — the C ABI of the transformer operators (declared in include/gigagan_amd.h): layer norm, rotary positions,
// attention with a sliding window and sinks. Argument validation and kernel launches; no allocation, no synchronisation.
#include "gg_device.h"
#include "gg_host.h"
#include "../../include/gigagan_amd.h"
#include "gg_layernorm.h"
#include "gg_rotary.h"
#include "gg_window.h"

#include <string.h>

// a launch holds fewer than 2^32 threads along an axis
static bool gg_grid_fits(long long blocks, int threads) { return blocks <= 0xffffffffll / threads; }

// ---- layer norm ------------------------------------------------------------------------------------------------

static int gg_ln_check(const char* who, const void* x, int64_t ldx, const float* w, int64_t rows, int32_t C, int32_t dtype) {
    if (!x || !w) return gg_fail(-1, "%s: null pointer", who);
    if (rows <= 0 || C <= 0 || C > GG_LAYERNORM_MAX_C) return gg_fail(-2, "%s: need rows > 0 and 0 < C <= %d (rows=%lld, C=%d)", who, GG_LAYERNORM_MAX_C, (long long)rows, C);
    if (ldx < 0) return gg_fail(-2, "%s: negative row pitch", who);
    if (dtype < 0 || dtype > 2) return gg_fail(-3, "%s: dtype must be bf16 (0), half (1) or fp32 (2)", who);
    return 0;
}

// threads per row and vectors per thread: the fewest threads that hold the row (gg_layernorm.h)
#define GG_LN_SHAPES(C, GO)                  \
    if ((C) <= 128) { GO(16, 1) }            \
    else if ((C) <= 512) { GO(64, 1) }       \
    else if ((C) <= 1024) { GO(64, 2) }      \
    else if ((C) <= 2048) { GO(64, 4) }      \
    else if ((C) <= 4096) { GO(256, 2) }     \
    else if ((C) <= 8192) { GO(256, 4) }     \
    else { GO(1024, 2) }

extern "C" int gg_layernorm_fwd(const void* x, int64_t ldx, const float* w, const float* b, void* y, float* mean, float* rstd,
                                int64_t rows, int32_t C, float eps, int32_t dtype, void* stream) {
    int rc = gg_ln_check("gg_layernorm_fwd", x, ldx, w, rows, C, dtype);
    if (rc) return rc;
    if (!y || ((mean == nullptr) != (rstd == nullptr))) return gg_fail(-1, "gg_layernorm_fwd: null pointer");
    GgLnParams p;
    memset(&p, 0, sizeof(p));
    p.x = x; p.ldx = ldx; p.w = w; p.b = b; p.y = y; p.mean = mean; p.rstd = rstd; p.rows = rows; p.C = C; p.eps = eps;
#define GG_LN_GO(TPR, NV)                                                                                                    \
    const long long rpb = TPR > 256 ? 1 : 256 / TPR, blocks = (rows - 1) / rpb + 1;                                          \
    if (!gg_grid_fits(blocks, TPR > 256 ? TPR : 256)) return gg_fail(-2, "gg_layernorm_fwd: too many rows");                  \
    const dim3 grid((unsigned)blocks), block(TPR > 256 ? TPR : 256);                                                         \
    if (dtype == GG_ELT_BF16) GG_LAUNCH((gg_layernorm_fwd_kernel<GG_ELT_BF16, TPR, NV>), grid, block, (hipStream_t)stream, p);     \
    else if (dtype == GG_ELT_F16) GG_LAUNCH((gg_layernorm_fwd_kernel<GG_ELT_F16, TPR, NV>), grid, block, (hipStream_t)stream, p);  \
    else GG_LAUNCH((gg_layernorm_fwd_kernel<GG_ELT_F32, TPR, NV>), grid, block, (hipStream_t)stream, p);
    GG_LN_SHAPES(C, GG_LN_GO)
#undef GG_LN_GO
    return gg_check_launch();
}

extern "C" int32_t gg_layernorm_blocks(int64_t rows, int32_t C) {
    const long long rpb = C <= 128 ? 16 : (C <= 2048 ? 4 : 1);
    const long long blocks = (rows - 1) / rpb + 1;
    return (int32_t)(blocks < 1 ? 1 : (blocks > 512 ? 512 : blocks));
}

extern "C" int gg_layernorm_bwd(const void* x, int64_t ldx, const void* dy, int64_t ldy, const float* w, const float* mean,
                                const float* rstd, void* dx, float* part, float* dw, float* db, int64_t rows, int32_t C, int32_t dtype,
                                void* stream) {
    int rc = gg_ln_check("gg_layernorm_bwd", x, ldx, w, rows, C, dtype);
    if (rc) return rc;
    if (!dy || !mean || !rstd || !dx || !part || !dw) return gg_fail(-1, "gg_layernorm_bwd: null pointer");
    if (ldy < 0) return gg_fail(-2, "gg_layernorm_bwd: negative row pitch");
    GgLnParams p;
    memset(&p, 0, sizeof(p));
    p.x = x; p.ldx = ldx; p.dy = dy; p.ldy = ldy; p.w = w; p.mean = (float*)mean; p.rstd = (float*)rstd; p.y = dx; p.part = part;
    p.rows = rows; p.C = C;
    const int blocks = gg_layernorm_blocks(rows, C);
#define GG_LN_GO(TPR, NV)                                                                                                    \
    const dim3 grid((unsigned)blocks), block(TPR > 256 ? TPR : 256);                                                         \
    if (dtype == GG_ELT_BF16) GG_LAUNCH((gg_layernorm_bwd_kernel<GG_ELT_BF16, TPR, NV>), grid, block, (hipStream_t)stream, p);     \
    else if (dtype == GG_ELT_F16) GG_LAUNCH((gg_layernorm_bwd_kernel<GG_ELT_F16, TPR, NV>), grid, block, (hipStream_t)stream, p);  \
    else GG_LAUNCH((gg_layernorm_bwd_kernel<GG_ELT_F32, TPR, NV>), grid, block, (hipStream_t)stream, p);
    GG_LN_SHAPES(C, GG_LN_GO)
#undef GG_LN_GO
    rc = gg_check_launch();
    if (rc) return rc;
    GG_LAUNCH(gg_layernorm_finish_kernel, dim3((unsigned)((2 * C + 31) / 32)), dim3(1024), (hipStream_t)stream, (const float*)part, dw, db, blocks, (int)C);
    return gg_check_launch();
}

// ---- rotary positions --------------------------------------------------------------------------------------------

extern "C" int gg_rotary(const gg_rotary_desc* d, void* stream) {
    if (!d || !d->q || !d->yq || !d->positions || !d->freqs || !d->axes) return gg_fail(-1, "gg_rotary: null pointer");
    if (d->hk < 0 || (d->hk > 0 && (!d->k || !d->yk))) return gg_fail(-1, "gg_rotary: %d key heads without keys", d->hk);
    if (d->B <= 0 || d->n <= 0 || d->hq <= 0) return gg_fail(-2, "gg_rotary: B, n and hq must be positive");
    if (d->pairs <= 0 || d->pairs > GG_ROT_MAX_PAIRS || d->d < 2 * d->pairs || d->d > GG_ROTARY_MAX_D)
        return gg_fail(-2, "gg_rotary: need 1 <= pairs <= %d and 2 pairs <= d <= %d (pairs=%d, d=%d)", GG_ROT_MAX_PAIRS, GG_ROTARY_MAX_D, d->pairs, d->d);
    if ((long long)d->hq + d->hk > 65536) return gg_fail(-2, "gg_rotary: more than 65536 heads");
    if (d->dtype < 0 || d->dtype > 2) return gg_fail(-3, "gg_rotary: dtype must be bf16 (0), half (1) or fp32 (2)");
    if (d->pos_type < 0 || d->pos_type > 2) return gg_fail(-3, "gg_rotary: positions must be int32 (0), int64 (1) or fp32 (2)");
    if (d->n_axes <= 0 || d->n_axes > 255) return gg_fail(-2, "gg_rotary: need 1 to 255 axes");
    GgRotParams p;
    memset(&p, 0, sizeof(p));
    p.x[0] = d->q; p.x[1] = d->k; p.y[0] = d->yq; p.y[1] = d->yk;
    for (int i = 0; i < 2; ++i) {
        const int64_t* s = i ? d->k_strides : d->q_strides;
        p.sb[i] = s[0]; p.sh[i] = s[1]; p.sn[i] = s[2];
    }
    p.h[0] = d->hq; p.h[1] = d->hk;
    p.pos = d->positions; p.pb = d->p_strides[0]; p.pn = d->p_strides[1]; p.pa = d->p_strides[2]; p.pos_type = d->pos_type;
    p.B = d->B; p.n = d->n; p.d = d->d; p.pairs = d->pairs; p.interleaved = d->interleaved != 0; p.inverse = d->inverse != 0;
    for (int i = 0; i < d->pairs; ++i) {
        if (d->axes[i] >= d->n_axes) return gg_fail(-2, "gg_rotary: pair %d names axis %d of %d", i, (int)d->axes[i], d->n_axes);
        p.axis[i] = d->axes[i];
        p.turns[i] = d->freqs[i] * 0.15915494309189533577;      // 1 / 2 pi
    }
    // tokens per workgroup: about four eight-pair items a thread, as far as the sines fit (one token always does)
    const int per = (d->pairs + 7) / 8 + (d->d - 2 * d->pairs + 7) / 8;
    long long tb = 1024 / ((long long)(d->hq + d->hk) * per);
    if (tb > GG_ROT_LDS_PAIRS / d->pairs) tb = GG_ROT_LDS_PAIRS / d->pairs;
    const long long fill = (long long)d->B * d->n / 1024;           // (few tokens: rather spread over the chip)
    if (tb > fill) tb = fill;
    p.tb = (int)(tb < 1 ? 1 : tb);
    const long long grid = (long long)d->B * ((d->n - 1) / p.tb + 1);
    if (!gg_grid_fits(grid, 256)) return gg_fail(-2, "gg_rotary: too many tokens");
    if (d->dtype == GG_ELT_BF16) GG_LAUNCH(gg_rotary_kernel<GG_ELT_BF16>, dim3((unsigned)grid), dim3(256), (hipStream_t)stream, p);
    else if (d->dtype == GG_ELT_F16) GG_LAUNCH(gg_rotary_kernel<GG_ELT_F16>, dim3((unsigned)grid), dim3(256), (hipStream_t)stream, p);
    else GG_LAUNCH(gg_rotary_kernel<GG_ELT_F32>, dim3((unsigned)grid), dim3(256), (hipStream_t)stream, p);
    return gg_check_launch();
}

// ---- attention with a sliding window and sinks ----------------------------------------------------------------------

// what a call launches: a function of the sizes alone, so that the workspace query and the call agree
struct GgWinPlan {
    bool few;                   // rows fit one 32-row tile: gg_win_few_kernel
    int row_tiles, splits, join;        // forward
    int key_tiles, sink_tiles, sink_chunks;     // dk / dv: the first sink_tiles have their rows cut into sink_chunks
    size_t fwd_bytes, bwd_bytes;
};

static int gg_win_bound(int32_t v) { return v < 0 || v > GGW_NONE ? GGW_NONE : v; }

static GgWinPlan gg_win_plan(const gg_window_desc* d) {
    GgWinPlan w;
    const long long g = d->h / d->hk, rows = (long long)d->n * g, heads = (long long)d->B * d->hk;
    const long long left = gg_win_bound(d->left), right = gg_win_bound(d->right), sinks = d->sinks < d->m ? d->sinks : d->m;
    w.few = rows <= 32;
    const int tr = w.few ? 32 : 128, tk = w.few ? 32 : 64;
    w.row_tiles = (int)((rows + tr - 1) / tr);
    // keys that one row tile visits at most, in tiles
    long long span = left + right + (rows < tr ? rows : tr) / g + 1 + sinks;
    if (span > d->m) span = d->m;
    const long long tiles = (span + tk - 1) / tk;
    // split the keys where the row tiles alone do not fill the 256 CUs twice over, down to two key tiles a wave (one token, 8192 keys, two
    // key heads: 7.4 us and 4.4 for the join)
    const long long blocks = heads * w.row_tiles, least = w.few ? 8 : 4;
    long long s = blocks >= 512 ? 1 : (512 + blocks - 1) / blocks;
    if (s > tiles / least) s = tiles / least;
    if (s > 64) s = 64;
    w.splits = (int)(s < 1 ? 1 : s);
    // thread groups a row in the join: each takes four splits or so
    w.join = 1;
    while (w.join * 4 < w.splits && w.join < 1024 / d->d) w.join *= 2;
    w.fwd_bytes = w.splits > 1 ? (size_t)w.splits * heads * rows * (d->d + 2) * sizeof(float) : 0;
    w.key_tiles = (d->m + 127) / 128;
    w.sink_tiles = (int)((sinks + 127) / 128);
    // dk / dv, first rule: the sinks' tiles, which every row sees, are cut into chunks no longer than an ordinary key tile's work (`seen`
    // rows) - but no shorter than a chip's share of all the work (512 workgroups at a time): many sink tiles fill the chip uncut, and
    // the chunks are 1024 at most, however many sinks there are
    long long seen = (left + right + 128) * g;
    if (seen > rows) seen = rows;
    const long long tiles_kv = heads * w.key_tiles, share = heads * (w.sink_tiles * rows + (w.key_tiles - w.sink_tiles) * seen) / 512 + 1;
    long long c = w.sink_tiles ? rows / (seen < 512 ? 512 : seen) : 1;
    if (c > (rows + share - 1) / share) c = (rows + share - 1) / share;
    if (c < 1) c = 1;
    if (c > 64) c = 64;
    // Second rule, where there are too few key tiles for the chip: every tile's rows are cut, down to two row tiles a workgroup (66 tiles of
    // 11 row tiles: 44 us whole, 28 and 4 us in five chunks and their sum; 32 of 64: causal training of 4096 tokens 246 -> 188 us a
    // pass), into 1024 chunks at most, unless the first rule's longest workgroup is no longer
    if (tiles_kv < 256) {
        const long long most = (seen + 127) / 128, want = (511 + tiles_kv) / tiles_kv, room = 1024 / tiles_kv;
        long long cut = want < most ? want : most;
        if (cut < c) cut = c < room ? c : room;
        const long long longest = w.sink_tiles == w.key_tiles || rows / c > seen ? rows / c : seen;
        if (cut > 1 && (w.sink_tiles ? rows : seen) / cut < (w.sink_tiles ? longest : seen)) {
            w.sink_tiles = w.key_tiles;
            c = cut;
        }
    }
    w.sink_chunks = (int)c;
    w.bwd_bytes = w.sink_chunks > 1 ? (size_t)heads * w.sink_tiles * w.sink_chunks * 2 * 128 * d->d * sizeof(float) : 0;
    return w;
}

// the sizes that gg_win_plan may be asked about: what it divides by is positive, what it multiplies stays in 64 bits
static int gg_win_sizes(const char* who, const gg_window_desc* d) {
    if (d->B <= 0 || d->n <= 0 || d->m <= 0 || d->h <= 0 || d->hk <= 0 || d->h % d->hk)
        return gg_fail(-2, "%s: B, n, m, h and hk must be positive and h a multiple of hk", who);
    if (d->d != 32 && d->d != 64 && d->d != 128) return gg_fail(-2, "%s: heads of 32, 64 or 128 features (got %d)", who, d->d);
    if (d->sinks < 0) return gg_fail(-3, "%s: negative sinks", who);
    if (d->m > (1 << 28) || (long long)d->n * (d->h / d->hk) > (1 << 30)) return gg_fail(-2, "%s: more than 2^28 keys or 2^30 rows a head", who);
    // (dk / dv divides by a group's heads with a 32-bit reciprocal: exact for quotients of x < g + 64 while x g < 2^32)
    if (d->h / d->hk > GG_WINDOW_MAX_GROUP) return gg_fail(-2, "%s: more than %d query heads a key head", who, GG_WINDOW_MAX_GROUP);
    if (!gg_grid_fits((long long)d->B * d->hk, 256)) return gg_fail(-2, "%s: too many rows", who);      // (a workgroup a key head at least)
    return 0;
}

static int gg_win_check(const char* who, const gg_window_desc* d, GgWinParams& p) {
    if (!d || !d->q || !d->k || !d->v || !d->o) return gg_fail(-1, "%s: null pointer", who);
    const int rc = gg_win_sizes(who, d);
    if (rc) return rc;
    if (d->dtype != GG_ELT_BF16 && d->dtype != GG_ELT_F16) return gg_fail(-3, "%s: dtype must be bf16 (0) or half (1)", who);
    if (!(d->scale > 0.f) || d->scale > 1.0e30f) return gg_fail(-3, "%s: scale must be positive and finite", who);
    const long long g = d->h / d->hk;
    const void* ptrs[] = {d->q, d->k, d->v, d->o, d->o_lo, d->d_o, d->dq, d->dk, d->dv};
    for (const void* x : ptrs)
        if ((unsigned long long)x & 15) return gg_fail(-4, "%s: operands must be 16-byte aligned", who);
    const int64_t* strides[] = {d->q_strides, d->k_strides, d->v_strides, d->d_o ? d->g_strides : d->q_strides};
    for (int w = 0; w < 4; ++w) {
        const int64_t* s = strides[w];
        for (int i = 0; i < 3; ++i)
            if (s[i] < 0 || (s[i] & 7)) return gg_fail(-4, "%s: strides must be multiples of 8 elements", who);
        // a tile of 64 rows is addressed by 32-bit offsets from its first token
        const bool query = w == 0 || w == 3;
        if (s[2] >= GG_WINDOW_MAX_STRIDE || (query && s[1] >= 64ll * GG_WINDOW_MAX_STRIDE / g))
            return gg_fail(-4, "%s: token strides must be below 2^24 elements and head strides of queries below 2^30 a group", who);
    }
    memset(&p, 0, sizeof(p));
    p.q = (const unsigned short*)d->q; p.k = (const unsigned short*)d->k; p.v = (const unsigned short*)d->v;
    p.d_o = (const unsigned short*)d->d_o;
    p.o = (unsigned short*)d->o; p.o_lo = (unsigned short*)d->o_lo; p.dq = (unsigned short*)d->dq; p.dk = (unsigned short*)d->dk; p.dv = (unsigned short*)d->dv;
    p.lse = d->lse; p.dvec = d->dvec;
    p.qb = d->q_strides[0]; p.qh = d->q_strides[1]; p.qn = (unsigned)d->q_strides[2];
    p.kb = d->k_strides[0]; p.kh = d->k_strides[1]; p.kn = (unsigned)d->k_strides[2];
    p.vb = d->v_strides[0]; p.vh = d->v_strides[1]; p.vn = (unsigned)d->v_strides[2];
    p.gb = d->g_strides[0]; p.gh = d->g_strides[1]; p.gn = (unsigned)d->g_strides[2];
    p.lengths = d->lengths; p.keep = (const unsigned char*)d->key_mask; p.keep_b = d->mask_stride;
    p.B = d->B; p.n = d->n; p.m = d->m; p.h = d->h; p.hk = d->hk; p.g = (int)g;
    p.left = gg_win_bound(d->left); p.right = gg_win_bound(d->right); p.sinks = d->sinks < d->m ? d->sinks : d->m;
    p.scale = d->scale;
    return 0;
}

extern "C" size_t gg_window_workspace_bytes(const gg_window_desc* d, int32_t backward) {
    if (!d || gg_win_sizes("gg_window_workspace_bytes", d)) return 0;
    const GgWinPlan w = gg_win_plan(d);
    return backward ? w.bwd_bytes : w.fwd_bytes;
}

#define GG_WIN_SHAPES(GO)                                                                              \
    if (d->dtype == GG_ELT_BF16) {                                                                     \
        if (d->d == 32) { GO(GG_ELT_BF16, 32) } else if (d->d == 64) { GO(GG_ELT_BF16, 64) } else { GO(GG_ELT_BF16, 128) }  \
    } else {                                                                                           \
        if (d->d == 32) { GO(GG_ELT_F16, 32) } else if (d->d == 64) { GO(GG_ELT_F16, 64) } else { GO(GG_ELT_F16, 128) }     \
    }

extern "C" int gg_window_fwd(const gg_window_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
    GgWinParams p;
    int rc = gg_win_check("gg_window_fwd", d, p);
    if (rc) return rc;
    const GgWinPlan w = gg_win_plan(d);
    if (w.fwd_bytes && (!workspace || workspace_bytes < w.fwd_bytes || ((unsigned long long)workspace & 15)))
        return gg_fail(-5, "gg_window_fwd: needs %zu workspace bytes, 16-byte aligned", w.fwd_bytes);
    p.splits = w.splits; p.join = w.join; p.row_tiles = w.row_tiles;
    const long long all = (long long)p.B * p.hk * p.n * p.g;
    if (w.splits > 1) {
        p.part_o = (float*)workspace;
        p.part_ml = p.part_o + (long long)w.splits * all * d->d;
    }
    const long long grid = (long long)p.B * p.hk * w.row_tiles * w.splits;
    if (!gg_grid_fits(grid, 256) || (w.splits > 1 && !gg_grid_fits(all * w.join / (1024 / d->d) + 1, 256))) return gg_fail(-2, "gg_window_fwd: too many rows");
    hipStream_t s = (hipStream_t)stream;
#define GG_WIN_GO(T, D)                                                                                                       \
    if (w.few) GG_LAUNCH((gg_win_few_kernel<T, D>), dim3((unsigned)grid), dim3(256), s, p);                                     \
    else if (w.splits > 1) GG_LAUNCH((gg_win_fwd_kernel<T, D, true>), dim3((unsigned)grid), dim3(256), s, p);                   \
    else GG_LAUNCH((gg_win_fwd_kernel<T, D, false>), dim3((unsigned)grid), dim3(256), s, p);                                    \
    rc = gg_check_launch();                                                                                                   \
    if (rc || w.splits == 1) return rc;                                                                                       \
    GG_LAUNCH((gg_win_join_kernel<T, D>), dim3((unsigned)((all * w.join + 1024 / D - 1) / (1024 / D))), dim3(256), s, p);
    GG_WIN_SHAPES(GG_WIN_GO)
#undef GG_WIN_GO
    return gg_check_launch();
}

extern "C" int gg_window_bwd(const gg_window_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
    GgWinParams p;
    int rc = gg_win_check("gg_window_bwd", d, p);
    if (rc) return rc;
    if (!d->o_lo || !d->d_o || !d->dq || !d->dk || !d->dv || !d->lse || !d->dvec) return gg_fail(-1, "gg_window_bwd: null pointer");
    const GgWinPlan w = gg_win_plan(d);
    if (w.bwd_bytes && (!workspace || workspace_bytes < w.bwd_bytes || ((unsigned long long)workspace & 15)))
        return gg_fail(-5, "gg_window_bwd: needs %zu workspace bytes, 16-byte aligned", w.bwd_bytes);
    const long long rows = (long long)p.n * p.g, heads = (long long)p.B * p.hk;
    const long long dq_tiles = (rows + 127) / 128, dq_grid = heads * dq_tiles;
    const long long kv_grid = heads * ((long long)w.sink_tiles * w.sink_chunks + w.key_tiles - w.sink_tiles);
    if (!gg_grid_fits(dq_grid, 256) || !gg_grid_fits(kv_grid, 256) 
        || (w.sink_chunks > 1 && !gg_grid_fits(heads * w.sink_tiles * (d->d / 8), 256))) return gg_fail(-2, "gg_window_bwd: too many rows");
    hipStream_t s = (hipStream_t)stream;
    p.part_o = (float*)workspace;
#define GG_WIN_GO(T, D)                                                                                                       \
    p.row_tiles = (int)dq_tiles;                                                                                              \
    GG_LAUNCH((gg_win_dq_kernel<T, D>), dim3((unsigned)dq_grid), dim3(256), s, p);                                              \
    rc = gg_check_launch();                                                                                                   \
    if (rc) return rc;                                                                                                        \
    p.row_tiles = w.key_tiles; p.sink_tiles = w.sink_tiles; p.sink_chunks = w.sink_chunks;                                    \
    GG_LAUNCH((gg_win_dkv_kernel<T, D>), dim3((unsigned)kv_grid), dim3(256), s, p);                                             \
    rc = gg_check_launch();                                                                                                   \
    if (rc || w.sink_chunks == 1) return rc;                                                                                  \
    GG_LAUNCH((gg_win_sink_kernel<T, D>), dim3((unsigned)((heads * w.sink_tiles * 128 * (D / 4) + 255) / 256)), dim3(256), s, p);
    GG_WIN_SHAPES(GG_WIN_GO)
#undef GG_WIN_GO
    return gg_check_launch();
}

#ifdef GG_HOST_EMULATION
// for the tests: the rows that the dk / dv of the key tile at k0 visit (a case whose tensors no test can hold)
extern "C" void gg_emu_window_rows(const gg_window_desc* d, int32_t len, int32_t k0, int32_t chunk, int32_t chunks, int32_t* rows) {
    GgWinParams p;
    if (gg_win_check("gg_emu_window_rows", d, p)) return;
    const GgwRows r = ggw_rows(p, len, k0, chunk, chunks);
    rows[0] = r.ra;
    rows[1] = r.rb;
}
#endif

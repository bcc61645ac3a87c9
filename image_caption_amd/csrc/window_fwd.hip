// Forward of attention under a sliding window with first keys that stay visible (the rule and the shared pieces:
// window_attn.h), for whole sequences, for the last rows of one, and for one token per sequence over a K/V cache.
//
// One pass over the visible keys with a running maximum and sum per row:
//     S^T = K Q^T,  P = exp(S - m),  O^T = V^T P,  l = sum P;    o = O / l,  lse = m + log l.
// The reference m is only moved when a row's maximum has grown past it by more than 8 / log2(e): probabilities then stay below
// 2^8 and the accumulators are rescaled a few times per row instead of once per tile.  Statistics and accumulators are f32.
//
// Two shapes of workgroup, both four waves:
//   QW = 4: 4 x 32 rows share tiles of 64 keys (f32: 32); the next tile is on its way in registers while the current one is
//           used, two LDS buffers, one barrier per tile; two workgroups per CU, one's exponentials under the other's products.
//   KW = 4: 32 rows, each wave its own 32 of the 128 keys of a tile, joined through LDS at the end: few rows (one token, the
//           scored rows of a caption) are a matter of reading K and V once, with all four waves' loads in flight.
// Where the row tiles alone do not fill the GPU, the visible tiles of a row tile are cut into nsplit parts that leave
// (O, m, l) in the workspace, joined by win_join_kernel.
//
// Measured (bf16, us): the scored rows of a captioning batch of 256 (32 of 229 rows, 8 heads of 96) 42 = 205 MB at 4.9 TB/s (49 a call); one token of
// 32 sequences of up to 32768 rows (32 heads on 8, 128 channels, window 8192) 197 = 1.08 GB at 5.5 TB/s: HBM bounds both.  A
// prompt of 2 x 8192 (32 heads on 8, 128 channels, window 1024) 334 = 770 TFLOP/s: the matrix cores are busy 37 % of it, the vector
// unit (32 exponentials a lane and tile above all) 41 %, one wave's products only partly under the other's
// exponentials; a tenth of both falls on keys that no row of the wave sees, a tile being left out only as a whole.  Left out in turn: exp -26, reads of V -25, of K -50, global loads -40, their way to LDS -20.  Three waves a SIMD,
// one key half at a time, and the next tile's scores before this one's products measured the same.
#include "window_attn.h"

namespace {

template <typename T, int HD, int QW, int KW, int NSUB, bool DROP>
__global__ __launch_bounds__(64 * QW * KW, sizeof(T) == 2 ? 2 : 1) void win_fwd_kernel(WinArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    using G = WinGeo<T, HD>;
    constexpr int NT = 64 * QW * KW, BK = 32 * KW * NSUB, NBUF = KW == 1 ? 2 : 1;
    constexpr int MAT = BK * G::PB;
    constexpr bool PRE = KW == 1 || HD < 128;          // the next tile's loads go out before this one's products, where the registers hold them
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const LaneAt<T, HD> at(lane);
    const int qw = KW == 1 ? wave : 0, kw = KW == 1 ? 0 : wave;
    const int id = win_xcd_id(blockIdx.x, gridDim.x);
    const int split = id % p.nsplit, rest = id / p.nsplit;
    const int tile = rest % p.tiles, bh = rest / p.tiles;
    const int b = bh / p.Hkv, hkv = bh - b * p.Hkv;
    const int n = win_len(p, b);
    const int q0 = p.last ? n - 1 : p.q_start;
    const int r_first = tile * 32 * QW, r_end = min(p.rows, r_first + 32 * QW);
    const int p_first = q0 + win_row_query(p, r_first), p_last = q0 + win_row_query(p, r_end - 1);
    const WinTiles tl = win_tiles<BK>(p, p_first, p_last, n);
    const int t_begin = p.nsplit == 1 ? 0 : (int)((long)tl.nt * split / p.nsplit);
    const int t_end = p.nsplit == 1 ? tl.nt : (int)((long)tl.nt * (split + 1) / p.nsplit);

    // this lane's row (rows past the end repeat the last one; nothing of them is stored)
    const int w_first = r_first + 32 * qw;
    const int r = w_first + (lane & 31), rc = min(r, p.rows - 1);
    const int irel = win_row_query(p, rc), head = hkv * p.G + rc - irel * p.G, pos = q0 + irel;
    const WinSpan sp = win_span(p, pos, n);
    // the same for the wave: what all of its rows see, and what any does
    const int wp0 = q0 + win_row_query(p, min(w_first, p.rows - 1)), wp1 = q0 + win_row_query(p, min(w_first + 31, p.rows - 1));
    const WinSpan s0 = win_span(p, wp0, n), s1 = win_span(p, wp1, n);
    const bool all_live = wp1 < n;
    const int any_a = max(s0.a, s1.a), any_hi = all_live ? s1.hi : (wp0 < n ? n : 0);
    const int any_a2 = p.open ? any_a : max(any_a, min(p.prefix, any_hi));
    const int any_end = w_first < p.rows ? max(any_a2, any_hi) : 0;      // (a wave past the last row has nothing to do)

    RowFrag<T, HD> qf;
    qf.load(reinterpret_cast<const T*>(p.q) + (long)b * p.q_bs + (long)head * p.q_hs + (long)irel * p.q_ss, lane);
    f32x16 acc[G::DT];
#pragma unroll
    for (int d = 0; d < G::DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[d][e] = 0.f;
    float m = -INFINITY, l = 0.f;

    const char* kbase = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.k) + (long)b * p.k_bs + (long)hkv * p.k_hs);
    const char* vbase = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.v) + (long)b * p.v_bs + (long)hkv * p.v_hs);
    const long kss = p.k_ss * (long)sizeof(T), vss = p.v_ss * (long)sizeof(T);
    const WinSpan any = win_union(p, p_first, p_last, n);
    TilePair<T, HD, BK, NT> tp;
    auto fetch = [&](int idx) {
        const int key0 = tl.at(idx) * BK;
        tp.fetch(kbase, kss, vbase, vss, key0, max(any.a, any.hi) - key0, tid);
    };
    auto commit = [&](int idx, char* lk, char* lv) {
        const int key0 = tl.at(idx) * BK;
        if (key0 < any.lo && key0 + BK > any.a) tp.drop(any.a - key0, any.lo - key0, tid);       // (keys between the prefix and the first window)
        tp.commit(lk, lv, tid);
    };
    auto compute = [&](int idx, const char* lk, const char* lv) {
        const int key0 = tl.at(idx) * BK + kw * 32 * NSUB;
        lk += kw * 32 * NSUB * G::PB;
        lv += kw * 32 * NSUB * G::PB;
        constexpr int NK = 32 * NSUB;
        if (key0 >= any_end || (key0 >= any_a2 && key0 + NK <= s0.lo)) return;
        f32x16 s[NSUB];
#pragma unroll
        for (int u = 0; u < NSUB; ++u) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[u][e] = 0.f;
            if constexpr (NSUB == 1) mma_rows<HD>(s[u], lk + u * 32 * G::PB, qf, at);
        }
        if constexpr (NSUB == 2) mma_rows2<HD>(s[0], lk, qf, s[1], lk + 32 * G::PB, qf, at);
        const bool whole = all_live && (key0 + NK <= s0.a || (key0 >= s1.lo && key0 + NK <= s0.hi));
        if (!whole) {
#pragma unroll
            for (int u = 0; u < NSUB; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    s[u][e] = win_sees(sp, key0 + 32 * u + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) ? s[u][e] : -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int u = 0; u < NSUB; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[u][e]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        if (__any(mx > m + 8.f / WIN_LOG2E)) {
            const float mn = fmaxf(m, mx);
            const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - mn) * WIN_LOG2E);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < G::DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[d][e] *= alpha;
        }
        const float mu = m == -INFINITY ? 0.f : m, mul = mu * WIN_LOG2E;
#pragma unroll
        for (int u = 0; u < NSUB; ++u) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                // f32: the difference is formed first, so that its rounding is small where the probability is not
                const float x = sizeof(T) == 2 ? fmaf(s[u][e], WIN_LOG2E, -mul) : (s[u][e] - mu) * WIN_LOG2E;
                s[u][e] = __builtin_amdgcn_exp2f(x);
                l += s[u][e];
            }
            if constexpr (DROP) {
                const uint32_t row = (uint32_t)((((long)b * p.H + head) * p.S + pos) * p.S4) + (uint32_t)(key0 + 32 * u + 4 * (lane >> 5));
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                    bool keep[4];
                    dropout_keep4(p.drop_k0, p.drop_k1, row + 8 * jj, p.drop_thr, keep);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[u][4 * jj + e] = keep[e] ? s[u][4 * jj + e] * p.drop_scale : 0.f;
                }
            }
            mma_cols<HD>(acc, lv + u * 32 * G::PB, s[u], at);
        }
    };

    if (t_begin < t_end) {
        fetch(t_begin);
        if constexpr (NBUF == 2) {
            commit(t_begin, smem, smem + MAT);
            __syncthreads();
            for (int idx = t_begin; idx < t_end; ++idx) {
                const int cur = (idx - t_begin) & 1;
                const bool more = idx + 1 < t_end;
                if (more) fetch(idx + 1);
                compute(idx, smem + 2 * cur * MAT, smem + (2 * cur + 1) * MAT);
                if (more) commit(idx + 1, smem + 2 * (cur ^ 1) * MAT, smem + (2 * (cur ^ 1) + 1) * MAT);
                __syncthreads();
            }
        } else {
            for (int idx = t_begin; idx < t_end; ++idx) {
                commit(idx, smem, smem + MAT);
                __syncthreads();
                if (PRE && idx + 1 < t_end) fetch(idx + 1);
                compute(idx, smem, smem + MAT);
                __syncthreads();
                if (!PRE && idx + 1 < t_end) fetch(idx + 1);
            }
        }
    }
    l += __shfl_xor(l, 32, 64);

    T* out = reinterpret_cast<T*>(p.o) + (long)b * p.o_bs + (long)head * p.o_hs + (long)irel * p.o_ss;
    const long part_row = ((long)split * p.B * p.Hkv + bh) * p.rows;
    if constexpr (KW == 1) {
        const bool ok = r < p.rows;
        if (p.nsplit == 1) {
            store_rows<HD>(acc, l != 0.f ? 1.f / l : 0.f, out, ok, lane);
            if (p.lse && ok && lane < 32) p.lse[((long)b * p.H + head) * p.nq + irel] = l != 0.f ? m + logf(l) : -INFINITY;
        } else {
            store_rows<HD>(acc, 1.f, p.part_o + (part_row + r) * HD, ok, lane);
            if (ok && lane < 32) { p.part_ml[2 * (part_row + r)] = m; p.part_ml[2 * (part_row + r) + 1] = l; }
        }
    } else {
        // join the four waves' shares of the keys: [wave][32 rows][HD + 4] f32, then [wave][32][m, l]
        constexpr int PJ = HD + 4;
        float* jo = reinterpret_cast<float*>(smem);
        float* jm = jo + KW * 32 * PJ;
        if (lane < 32) { jm[(kw * 32 + lane) * 2] = m; jm[(kw * 32 + lane) * 2 + 1] = l; }
        __syncthreads();
        float mj = -INFINITY;
#pragma unroll
        for (int w = 0; w < KW; ++w) mj = fmaxf(mj, jm[(w * 32 + (lane & 31)) * 2]);
        const float share = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mj) * WIN_LOG2E);
        store_rows<HD>(acc, share, jo + (kw * 32 + (lane & 31)) * PJ, true, lane);
        __syncthreads();
        for (int u = tid; u < 32 * HD / 4; u += NT) {
            const int row = u / (HD / 4), c = (u - row * (HD / 4)) * 4, rr = r_first + row;
            if (rr >= p.rows) break;
            float mm = -INFINITY, ll = 0.f;
#pragma unroll
            for (int w = 0; w < KW; ++w) mm = fmaxf(mm, jm[(w * 32 + row) * 2]);
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                const float mw = jm[(w * 32 + row) * 2];
                ll += mw == -INFINITY ? 0.f : jm[(w * 32 + row) * 2 + 1] * __builtin_amdgcn_exp2f((mw - mm) * WIN_LOG2E);
                v += *reinterpret_cast<const f32x4*>(jo + (w * 32 + row) * PJ + c);
            }
            if (p.nsplit > 1) {
                *reinterpret_cast<f32x4*>(p.part_o + (part_row + rr) * HD + c) = v;
                if (c == 0) { p.part_ml[2 * (part_row + rr)] = mm; p.part_ml[2 * (part_row + rr) + 1] = ll; }
                continue;
            }
            const int i = win_row_query(p, rr), h = hkv * p.G + rr - i * p.G;
            T* at = reinterpret_cast<T*>(p.o) + (long)b * p.o_bs + (long)h * p.o_hs + (long)i * p.o_ss + c;
            const float inv = ll != 0.f ? 1.f / ll : 0.f;
            if constexpr (sizeof(T) == 2) {
                bf16x4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = (bf16_t)(v[e] * inv);
                *reinterpret_cast<bf16x4*>(at) = w;
            } else {
                *reinterpret_cast<f32x4*>(at) = v * inv;
            }
            if (c == 0 && p.lse) p.lse[((long)b * p.H + h) * p.nq + i] = ll != 0.f ? mm + logf(ll) : -INFINITY;
        }
    }
}

// o and lse of every row from its nsplit parts: one workgroup per row
template <typename T, int HD>
__global__ __launch_bounds__(256) void win_join_kernel(WinArgs p) {
    const long row = blockIdx.x;
    const int bh = (int)(row / p.rows), r = (int)(row - (long)bh * p.rows);
    const int b = bh / p.Hkv, i = win_row_query(p, r), h = (bh - b * p.Hkv) * p.G + r - i * p.G;
    join_parts<T>(p.part_o, p.part_ml, (long)p.B * p.Hkv * p.rows, row, HD, p.nsplit,
                  reinterpret_cast<T*>(p.o) + (long)b * p.o_bs + (long)h * p.o_hs + (long)i * p.o_ss, p.lse ? p.lse + ((long)b * p.H + h) * p.nq + i : nullptr);
}

template <typename T, int HD, int QW, int KW, int NSUB, bool DROP>
int fwd_go(WinArgs& a, hipStream_t st) {
    using G = WinGeo<T, HD>;
    constexpr int BK = 32 * KW * NSUB, NBUF = KW == 1 ? 2 : 1;
    constexpr int tiles_bytes = NBUF * 2 * BK * G::PB, join_bytes = KW == 1 ? 0 : KW * 32 * (HD + 4 + 2) * 4;
    constexpr int lds = tiles_bytes > join_bytes ? tiles_bytes : join_bytes;
    auto kfn = win_fwd_kernel<T, HD, QW, KW, NSUB, DROP>;
    if (lds > 64 * 1024) ensure_dynamic_lds((const void*)kfn, lds);
    const long grid = (long)a.B * a.Hkv * a.tiles * a.nsplit;
    CAPDEC_CHECK(grid < (1L << 31), "attn_window: %ld workgroups", grid);
    hipLaunchKernelGGL(kfn, dim3((unsigned)grid), dim3(64 * QW * KW), lds, st, a);
    CAPDEC_LAUNCH_CHECK();
    if (a.nsplit > 1) {
        hipLaunchKernelGGL((win_join_kernel<T, HD>), dim3((unsigned)((long)a.B * a.Hkv * a.rows)), dim3(256), 0, st, a);
        CAPDEC_LAUNCH_CHECK();
    }
    return CAPDEC_OK;
}
template <typename T, int HD>
int fwd_hd(WinArgs& a, int kw, hipStream_t st) {
    constexpr int NS = sizeof(T) == 2 ? 2 : 1;
    if (a.drop_thr) return kw ? fwd_go<T, HD, 1, 4, 1, true>(a, st) : fwd_go<T, HD, 4, 1, NS, true>(a, st);
    return kw ? fwd_go<T, HD, 1, 4, 1, false>(a, st) : fwd_go<T, HD, 4, 1, NS, false>(a, st);
}
template <typename T>
int fwd_type(WinArgs& a, int hd, int kw, hipStream_t st) {
    switch (hd) {
        case 32: return fwd_hd<T, 32>(a, kw, st);
        case 64: return fwd_hd<T, 64>(a, kw, st);
        case 96: return fwd_hd<T, 96>(a, kw, st);
        default: return fwd_hd<T, 128>(a, kw, st);
    }
}

}  // namespace

// ------------------------------------------------------------------ host side
int win_fill(const capdec_attn_window_desc* d, WinArgs& a, const char* what) {
    CAPDEC_CHECK(d && d->q && d->k && d->v && d->o, "%s: null pointer", what);
    CAPDEC_CHECK(d->dtype == CAPDEC_BF16 || d->dtype == CAPDEC_F32, "%s: bad dtype", what);
    CAPDEC_CHECK(d->B > 0 && d->H > 0 && d->Hkv > 0 && d->H % d->Hkv == 0, "%s: B %d, H %d, Hkv %d (Hkv must divide H)", what, d->B, d->H, d->Hkv);
    CAPDEC_CHECK(d->hd == 32 || d->hd == 64 || d->hd == 96 || d->hd == 128, "%s: head dim %d (32, 64, 96 or 128)", what, d->hd);
    CAPDEC_CHECK(d->S > 0 && d->S < (1 << 28), "%s: %d keys", what, d->S);
    CAPDEC_CHECK(d->q_start >= 0 && d->nq > 0 && (long)d->q_start + d->nq <= d->S, "%s: queries %d..%ld outside %d positions", what, d->q_start,
                 (long)d->q_start + d->nq, d->S);
    CAPDEC_CHECK(d->window >= 0 && d->prefix_len >= 0, "%s: window %d, prefix %d", what, d->window, d->prefix_len);
    const int G = d->H / d->Hkv;
    CAPDEC_CHECK((double)d->nq * G * G < 2147483648.0 && (long)d->B * d->Hkv < (1L << 31), "%s: %d queries of %d heads to a K/V head", what, d->nq, G);
    const int e = d->dtype == CAPDEC_BF16 ? 2 : 4, per16 = 16 / e;
    CAPDEC_CHECK(aligned16(d->q) && aligned16(d->k) && aligned16(d->v) && aligned16(d->o), "%s: operands must be 16-byte aligned", what);
    const long st[] = {d->q_bs, d->q_hs, d->q_ss, d->k_bs, d->k_hs, d->k_ss, d->v_bs, d->v_hs, d->v_ss, d->o_bs, d->o_hs, d->o_ss};
    for (long s : st) CAPDEC_CHECK(s >= 0 && s % per16 == 0, "%s: stride %ld (must be a non-negative multiple of %d elements)", what, s, per16);
    // (a buffer's 64 rows are addressed by 31 bits; compared by division: a product with a stride of 2^58 wraps)
    CAPDEC_CHECK(d->k_ss < (1L << 25) / e && d->v_ss < (1L << 25) / e, "%s: key rows lie too far apart (%ld and %ld elements, 32 MiB or more)", what, d->k_ss, d->v_ss);
    memset(&a, 0, sizeof(a));
    a.q = d->q; a.k = d->k; a.v = d->v; a.o = d->o;
    a.q_bs = d->q_bs; a.q_hs = d->q_hs; a.q_ss = d->q_ss;
    a.k_bs = d->k_bs; a.k_hs = d->k_hs; a.k_ss = d->k_ss;
    a.v_bs = d->v_bs; a.v_hs = d->v_hs; a.v_ss = d->v_ss;
    a.o_bs = d->o_bs; a.o_hs = d->o_hs; a.o_ss = d->o_ss;
    a.B = d->B; a.H = d->H; a.Hkv = d->Hkv; a.G = G; a.S = d->S; a.nq = d->nq; a.q_start = d->q_start;
    a.g_magic = (unsigned)((1ULL << 32) / (unsigned)G + 1);
    a.rows = d->nq * G;
    a.window = d->window == 0 ? 1 << 30 : (d->window < (1 << 30) ? d->window : 1 << 30);
    a.prefix = d->prefix_len < d->S ? d->prefix_len : d->S;
    a.open = d->prefix_open != 0;
    a.lens = d->lens;
    a.lse = d->lse;
    a.S4 = (d->S + 3) & ~3;
    if (d->drop.p > 0.f) {
        CAPDEC_CHECK(d->drop.p < 1.f, "%s: dropout probability %f", what, d->drop.p);
        CAPDEC_CHECK((double)d->B * d->H * d->S * a.S4 < 4294967296.0, "%s: dropout index space exceeds 2^32", what);
        a.drop_thr = dropout_threshold(d->drop.p);
        a.drop_k0 = d->drop.key0; a.drop_k1 = d->drop.key1;
        a.drop_scale = 1.f / (1.f - d->drop.p);
    }
    return CAPDEC_OK;
}

WinFwdPlan win_fwd_plan(bool f32, int B, int H, int Hkv, int S, int nq, int hd, int window, int prefix) {
    WinFwdPlan pl;
    const int G = H / Hkv;
    const long rows = (long)nq * G;
    pl.kw = win_few_rows(f32, (long)B * Hkv, rows);
    const int R = pl.kw ? 32 : 128, BK = pl.kw ? 128 : 64;
    pl.tiles = (int)((rows + R - 1) / R);
    // key tiles that a row tile can see at most
    const long w = window == 0 ? S : (window < S ? window : S);
    const long band = w + (R + G - 1) / G < S ? w + (R + G - 1) / G : S;
    const long pre = prefix < S ? prefix : S;
    const long seen = pre + band < S ? pre + band : S;
    const long nt = seen / BK + 2;
    const long wgs = (long)B * Hkv * pl.tiles;
    long ns = 1;
    // Two workgroups per CU, each with at least four key tiles of its own.  Measured (one token, us): not cut | as here | aimed at 1024
    // workgroups | at least two tiles | eight:  8 x 1024 keys, hd 96: 13.5 | 12.5 | 12.6 | 10.1 | 13.5;  8 x 4096, hd 128: 50 | 13.8 | 13.8 | 11.7 | 19.5;
    // 32 x 4096: 58 | 19.8 | 20.1 | 19.6 | 24.6;  8 x 32768: 428 | 31.0 | 30.9 | 31.0 | 30.4;  64 x 32768: 610 | 204 | 198 | 197 | 199;
    // 8 x 131072: 2363 | 111 | 109 | 107 | 108.  (Two tiles would gain a third at small caches.)
    if (wgs < 512) {
        ns = (512 + wgs - 1) / wgs;
        if (ns > nt / 4) ns = nt / 4;
        if (ns > 1024) ns = 1024;
        if (ns < 1) ns = 1;
    }
    pl.nsplit = (int)ns;
    pl.part_floats = ns > 1 ? ns * (long)B * Hkv * rows * (hd + 2) : 0;
    return pl;
}

int win_fwd_launch(WinArgs& a, int dtype, int hd, void* workspace, long workspace_bytes, hipStream_t st) {
    const WinFwdPlan pl = win_fwd_plan(dtype == CAPDEC_F32, a.B, a.H, a.Hkv, a.S, a.nq, hd, a.window >= (1 << 30) ? 0 : a.window, a.prefix);
    a.tiles = pl.tiles;
    a.nsplit = 1;
    if (pl.nsplit > 1 && workspace) {
        if (workspace_bytes < pl.part_floats * 4) {
            capdec_set_error("attn_window: workspace %ld bytes < %ld", workspace_bytes, pl.part_floats * 4);
            return CAPDEC_ERR_WORKSPACE;
        }
        CAPDEC_CHECK(aligned16(workspace), "attn_window: workspace must be 16-byte aligned");
        a.nsplit = pl.nsplit;
        a.part_o = (float*)workspace;
        a.part_ml = a.part_o + (long)pl.nsplit * a.B * a.Hkv * a.rows * hd;
    }
    return dtype == CAPDEC_BF16 ? fwd_type<bf16_t>(a, hd, pl.kw, st) : fwd_type<float>(a, hd, pl.kw, st);
}

extern "C" long capdec_attn_window_fwd_workspace(int B, int H, int Hkv, int S, int nq, int hd, int window, int prefix_len) {
    if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || S <= 0 || nq <= 0 || hd <= 0 || window < 0 || prefix_len < 0) return 0;
    // (either type's: the rows up to which the keys are shared out differ)
    const long f32 = win_fwd_plan(true, B, H, Hkv, S, nq, hd, window, prefix_len).part_floats, bf16 = win_fwd_plan(false, B, H, Hkv, S, nq, hd, window, prefix_len).part_floats;
    return (f32 > bf16 ? f32 : bf16) * 4;
}

extern "C" int capdec_attn_window_fwd(const capdec_attn_window_desc* d, void* stream) {
    WinArgs a;
    const int rc = win_fill(d, a, "attn_window_fwd");
    if (rc != CAPDEC_OK) return rc;
    return win_fwd_launch(a, d->dtype, d->hd, d->workspace, d->workspace_bytes, (hipStream_t)stream);
}

extern "C" long capdec_attn_window_decode_workspace(int B, int H, int Hkv, int hd, int smax, int window, int prefix_len) {
    return capdec_attn_window_fwd_workspace(B, H, Hkv, smax, 1, hd, window, prefix_len);
}

extern "C" int capdec_attn_window_decode(const void* q, const void* kv_cache, void* o, int dtype, int B, int H, int Hkv, int hd, int smax, int len,
                                         const int32_t* lens, int window, int prefix_len, void* workspace, long workspace_bytes, void* stream) {
    CAPDEC_CHECK(smax > 0 && len > 0 && len <= smax, "attn_window_decode: length %d outside 1..%d", len, smax);
    CAPDEC_CHECK(kv_cache != nullptr, "attn_window_decode: null pointer");
    CAPDEC_CHECK(dtype == CAPDEC_BF16 || dtype == CAPDEC_F32, "attn_window_decode: bad dtype");
    capdec_attn_window_desc d;
    memset(&d, 0, sizeof(d));
    const long e = dtype == CAPDEC_BF16 ? 2 : 4;
    d.q = q; d.k = kv_cache; d.v = (const char*)kv_cache + (long)smax * hd * e; d.o = o;
    d.q_bs = (long)H * hd; d.q_hs = hd; d.q_ss = hd;
    d.o_bs = (long)H * hd; d.o_hs = hd; d.o_ss = hd;
    d.k_bs = d.v_bs = (long)Hkv * 2 * smax * hd; d.k_hs = d.v_hs = 2L * smax * hd; d.k_ss = d.v_ss = hd;
    d.dtype = dtype; d.B = B; d.H = H; d.Hkv = Hkv; d.S = len; d.hd = hd;      // (keys past len are never read, whatever lens says)
    d.q_start = len - 1; d.nq = 1;
    d.window = window; d.prefix_len = prefix_len; d.lens = lens;
    WinArgs a;
    const int rc = win_fill(&d, a, "attn_window_decode");
    if (rc != CAPDEC_OK) return rc;
    a.last = 1;
    return win_fwd_launch(a, dtype, hd, workspace, workspace_bytes, (hipStream_t)stream);
}

// Backward of attention under a sliding window with first keys that stay visible (rule and shared pieces: window_attn.h).
//
//     P = exp(S - lse),  delta = sum_d dO O,  dP = dO V^T,  dS = P (dP - delta),
//     dQ = dS K,   dK = dS^T Q,   dV = P^T dO            (q carries its scale; dq is multiplied by dq_scale)
//
// Two kernels, each recomputing P from the saved log-sum-exp: one owns query rows and walks the key tiles they see (dQ, and
// delta on its way), one owns 128 keys and walks the rows that see them (dK, dV; the heads that share a K/V head are
// neighbouring rows, so their sum needs nothing more).  Seven products where five would do, but no atomics: every sum is
// formed in a fixed order.
//
// Keys of the prefix are seen by every row, the others by window + 128 positions: a prefix tile's rows are cut into chunks
// that leave f32 partial sums in the workspace, added in order by a third kernel.  At most 256 keys: one kernel for all three.
//
// Roundings (bf16): P and dS once, to be operands (half a step of each term, as much as the inputs have); delta is an f32 sum over
// the bf16 o that the forward wrote, so it carries o's own rounding.  Both leave a row of dS with a sum that is not quite 0,
// and what the keys have in common is multiplied by that sum: with channel offsets of 2 and 8 times the keys' spread dQ was
// 0.009 and 0.035 of its size off.  In exact numbers the sum is 0 and any c may be taken out of the keys, so
//     dQ = sum_j dS_j K_j - (sum_j dS_j) c,     the sum over the rounded dS, c the common part of some of the visible keys
// (KeyMean below): one number a row, a 2-term dot product per two elements of dS.  dQ then lies 0.0024-0.0033 of its size from the exact one
// whatever the offset (0.004-0.005 as a mean over 5000-10000 keys), dK 0.0024-0.0029, dV 0.0023, against 0.0017 for their own rounding alone.  Cost: captioning stack 123.0 -> 127.6 us, 3 of
// them the dot products (sums by matrix instructions against ones: 128.3), 8192 positions 318 -> 321, 100 rows over 10000 keys 98 -> 109.
// What V's rows have in common reaches delta through o's rounding, stays in the formula and is left: 0.005 of dQ and dK for an offset of
// twice V's spread, 0.02 for eight times, and 0.005 of dQ where 9000 keys are averaged over an offset of a quarter.  An exact delta, 0.0023-0.0026,
// would take S and dP a second time, two products of seven.
//
// Measured (bf16, us): 8192 positions, 16 heads on 4 of 128 channels, window 1024: dQ 127, dK / dV 190, join 19, 313-327 in all = 500-520 TFLOP/s
// of the five products the formulas have (seven are made).  The matrix cores are busy a third of the time (0.35, 0.31): a step is one chain of
// LDS reads, products, exponentials, products, LDS writes and a barrier, and only two waves a SIMD are there to fill it (the
// accumulators of 64 + 64 registers and V's rows allow no third).  Left out in turn: dK and dV's products -52, LDS writes
// -37, S and dP's products -32, loads from L2 -9, exponentials -5.  Two key blocks a wave at one wave a SIMD: 425.
#include "window_attn.h"

namespace {

constexpr int KT = 128;              // keys of a dK / dV workgroup: four waves of 32
constexpr int RB = 32;               // rows per step

// The common part c of the keys, for dQ: the mean of m keys spread over the longer run of visible ones, in the channels where it stands out
// of the keys' own spread (six standard errors of that mean: what is below would only be the sample's
// noise, and of keys without a common part one channel in 10^6 or 10^7 passes by chance).  One key in sixteen,
// 64 at least and 1024 at most: what is left of c costs dQ less than its roundings do with 64 keys up to about a thousand,
// and dQ, a mean over n keys, shrinks like 1 / sqrt(n) against it (100 rows over 10000 keys, 0.0074 of dQ with 64).  Fewer than 32
// keys say nothing: c = 0.  Formed at the start of a workgroup; partial sums and squares meet in LDS.
template <int HD, int NT> struct KeyMean {
    static constexpr int N = 64, P = HD / 2, RG = NT >= 512 ? 8 : NT / P, U = (N + RG - 1) / RG;      // channel pairs of a row, rows at a time, rows of a thread in N
    static constexpr int PART = RG * HD * 8, BYTES = PART + HD * 4;
    unsigned x[U];
    int key0, step, m;
    f32x4 s;                                                                 // sum and squares of either channel
    __device__ __forceinline__ void pick(const WinSpan& any) {
        const bool one = any.lo <= any.a, band = !one && any.hi - any.lo >= any.a;
        const int first = band ? any.lo : 0, len = one ? max(any.a, any.hi) : band ? any.hi - any.lo : any.a;
        m = min(len, max(N, min(1024, len >> 4)));
        step = m > 0 ? len / m : 1;
        key0 = first + (len - 1 - (m - 1) * step) / 2;
        s = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // keys base.. of the sample
    __device__ __forceinline__ void load(const bf16_t* k, long ss, int base, int tid) {
        const int row = tid / P, pair = tid - row * P;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int i = base + row + j * RG;
            x[j] = 0;
            if (row + j * RG < N && row < RG && i < m) x[j] = *reinterpret_cast<const unsigned*>(k + (long)(key0 + i * step) * ss + 2 * pair);
        }
    }
    // from K's rows in LDS (row 0 is key 0), of at most N keys
    __device__ __forceinline__ void load(const char* lk, int tid) {
        const int row = tid / P, pair = tid - row * P;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            x[j] = *reinterpret_cast<const unsigned*>(lk + WinGeo<bf16_t, HD>::at(max(0, key0 + min(row + j * RG, m - 1) * step), pair >> 2) + 4 * (pair & 3));
            x[j] = row + j * RG < m ? x[j] : 0u;
        }
    }
    __device__ __forceinline__ void add() {
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const float lo = __uint_as_float(x[j] << 16), hi = __uint_as_float(x[j] & 0xFFFF0000u);
            s = f32x4{s[0] + lo, fmaf(lo, lo, s[1]), s[2] + hi, fmaf(hi, hi, s[3])};
        }
    }
    __device__ __forceinline__ void partial(char* lds, int tid) const {
        const int row = tid / P, pair = tid - row * P;
        if (row < RG) *reinterpret_cast<f32x4*>(lds + (row * HD + 2 * pair) * 8) = s;
    }
    // (after a barrier; c may be read after another one)
    __device__ __forceinline__ void finish(char* lds, int tid) const {
        if (tid >= HD) return;
        float s = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < RG; ++j) {
            const f32x2 y = *reinterpret_cast<const f32x2*>(lds + (j * HD + tid) * 8);
            s += y[0];
            s2 += y[1];
        }
        const float inv = 1.f / (float)max(m, 1), mean = s * inv, var = fmaxf(fmaf(-mean, mean, s2 * inv), 0.f);
        *reinterpret_cast<float*>(lds + PART + 4 * tid) = m >= 32 && (float)m * mean * mean > 36.f * var ? mean : 0.f;
    }
    static __device__ __forceinline__ f32x4 at(const char* lds, int channel) { return *reinterpret_cast<const f32x4*>(lds + PART + 4 * channel); }
};

// ------------------------------------------------------------------ dQ (and delta)
// LDS of dQ's kernel: its tiles (KW: also the join of the four waves' shares), then the common part of the keys
template <typename T, int HD, int QW, int KW> struct DqLds {
    using G = WinGeo<T, HD>;
    static constexpr int BK = 32 * KW * (KW == 1 && sizeof(T) == 2 ? 2 : 1);
    static constexpr int STAGE = (KW == 1 ? 2 : 1) * 2 * BK * G::PB, JOIN = KW == 1 ? 0 : KW * 32 * (HD + 4) * 4;
    static constexpr int TILES = STAGE > JOIN ? STAGE : JOIN;
    static constexpr int BYTES = TILES + (sizeof(T) == 2 ? KeyMean<HD, 64 * QW * KW>::BYTES : 0);
};
template <typename T, int HD, int QW, int KW, bool DROP>
__global__ __launch_bounds__(64 * QW * KW, sizeof(T) == 2 ? 2 : 1) void win_dq_kernel(WinArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    using G = WinGeo<T, HD>;
    constexpr int NSUB = KW == 1 && sizeof(T) == 2 ? 2 : 1;
    constexpr int NT = 64 * QW * KW, BK = 32 * KW * NSUB, NBUF = KW == 1 ? 2 : 1;
    constexpr int MAT = BK * G::PB;
    constexpr bool PRE = KW == 1 || HD < 128;          // the next tile's loads go out before this one's products, where the registers hold them
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const LaneAt<T, HD> at0(lane);
    const int qw = KW == 1 ? wave : 0, kw = KW == 1 ? 0 : wave;
    const int id = win_xcd_id(blockIdx.x, gridDim.x);
    const int tile = id % p.tiles, bh = id / p.tiles;
    const int b = bh / p.Hkv, hkv = bh - b * p.Hkv;
    const int n = win_len(p, b), q0 = p.q_start;
    const int r_first = tile * 32 * QW, r_end = min(p.rows, r_first + 32 * QW);
    const WinTiles tl = win_tiles<BK>(p, q0 + win_row_query(p, r_first), q0 + win_row_query(p, r_end - 1), n);

    const int w_first = r_first + 32 * qw;
    const int r = w_first + (lane & 31), rc = min(r, p.rows - 1);
    const int irel = win_row_query(p, rc), head = hkv * p.G + rc - irel * p.G, pos = q0 + irel;
    const WinSpan sp = win_span(p, pos, n);
    const int wp0 = q0 + win_row_query(p, min(w_first, p.rows - 1)), wp1 = q0 + win_row_query(p, min(w_first + 31, p.rows - 1));
    const WinSpan s0 = win_span(p, wp0, n), s1 = win_span(p, wp1, n);
    const bool all_live = wp1 < n;
    const int any_hi = all_live ? s1.hi : (wp0 < n ? n : 0);
    const int any_a = p.open ? max(s0.a, s1.a) : min(p.prefix, any_hi);
    const int any_end = w_first < p.rows ? max(any_a, any_hi) : 0;

    RowFrag<T, HD> qf, df, of;
    const long stat = ((long)b * p.H + head) * p.nq + irel;
    float lse = INFINITY;
    qf.zero();
    df.zero();
    of.zero();
    if (pos < n) {                     // (a row past its sequence's end holds nothing that may be read into a sum)
        qf.load(reinterpret_cast<const T*>(p.q) + (long)b * p.q_bs + (long)head * p.q_hs + (long)irel * p.q_ss, lane);
        df.load(reinterpret_cast<const T*>(p.dout) + (long)b * p.do_bs + (long)head * p.do_hs + (long)irel * p.do_ss, lane);
        of.load(reinterpret_cast<const T*>(p.o) + (long)b * p.o_bs + (long)head * p.o_hs + (long)irel * p.o_ss, lane);
        lse = p.lse[stat];
    }
    const char* kbase = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.k) + (long)b * p.k_bs + (long)hkv * p.k_hs);
    const char* vbase = reinterpret_cast<const char*>(reinterpret_cast<const T*>(p.v) + (long)b * p.v_bs + (long)hkv * p.v_hs);
    const long kss = p.k_ss * (long)sizeof(T), vss = p.v_ss * (long)sizeof(T);
    const WinSpan any = win_union(p, q0 + win_row_query(p, r_first), q0 + win_row_query(p, r_end - 1), n);
    constexpr bool CENTRE = sizeof(T) == 2;
    char* lmean = smem + DqLds<T, HD, QW, KW>::TILES;
    [[maybe_unused]] KeyMean<HD, NT> mean;
    [[maybe_unused]] float rsum = 0.f;                 // of this lane's half of its row of dS
    TilePair<T, HD, BK, NT, true> tp;
    auto fetch = [&](int idx) {
        const int key0 = tl.at(idx) * BK;
        tp.fetch(kbase, kss, vbase, vss, key0, max(any.a, any.hi) - key0, tid);
    };
    auto commit = [&](int idx, char* lk, char* lv) {
        const int key0 = tl.at(idx) * BK;
        if (key0 < any.lo && key0 + BK > any.a) tp.drop(any.a - key0, any.lo - key0, tid);       // (keys between the prefix and the first window)
        tp.commit(lk, lv, tid);
    };
    if (tl.nt > 0) {                   // (on its way before the rows are waited for)
        fetch(0);
        if constexpr (CENTRE) {
            mean.pick(any);
            mean.load(reinterpret_cast<const T*>(kbase), p.k_ss, 0, tid);
        }
    }
    if (lse == -INFINITY) lse = INFINITY;              // a row that sees nothing: every probability is 0
    float delta = df.dot(of);
    delta += __shfl_xor(delta, 32, 64);
    if (kw == 0 && r < p.rows && lane < 32) p.delta[stat] = delta;

    f32x16 acc[G::DT];
#pragma unroll
    for (int d = 0; d < G::DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[d][e] = 0.f;

    const float lsel = lse * WIN_LOG2E;
    auto compute = [&](int idx, const char* lk0, const char* lv0) {
        const LaneAt<T, HD> at = at0.fresh();
#pragma unroll
        for (int u = 0; u < NSUB; ++u) {
            const int off = kw * 32 * NSUB + 32 * u, key0 = tl.at(idx) * BK + off;
            if (key0 >= any_end || (key0 >= any_a && key0 + 32 <= s0.lo)) continue;
            const char* lk = lk0 + off * G::PB;
            const char* lv = lv0 + off * G::PB;
            f32x16 s, dp;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = dp[e] = 0.f;
            mma_rows2<HD>(s, lk, qf, dp, lv, df, at);
            const bool whole = all_live && (key0 + 32 <= s0.a || (key0 >= s1.lo && key0 + 32 <= s0.hi));
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float x = sizeof(T) == 2 ? fmaf(s[e], WIN_LOG2E, -lsel) : (s[e] - lse) * WIN_LOG2E;
                s[e] = __builtin_amdgcn_exp2f(x);
            }
            if (!whole) {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = win_sees(sp, key0 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) ? s[e] : 0.f;
            }
            if constexpr (DROP) {
                const uint32_t row = (uint32_t)((((long)b * p.H + head) * p.S + pos) * p.S4) + (uint32_t)(key0 + 4 * (lane >> 5));
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                    bool keep[4];
                    dropout_keep4(p.drop_k0, p.drop_k1, row + 8 * jj, p.drop_thr, keep);
#pragma unroll
                    for (int e = 0; e < 4; ++e) dp[4 * jj + e] = keep[e] ? dp[4 * jj + e] * p.drop_scale : 0.f;
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] *= dp[e] - delta;
            if constexpr (CENTRE) mma_cols<HD, true>(acc, lk, s, at, &rsum);
            else mma_cols<HD>(acc, lk, s, at);
        }
    };
    auto sample = [&] {
        if constexpr (CENTRE) {
            mean.add();
            for (int base = mean.N; base < mean.m; base += mean.N) {
                mean.load(reinterpret_cast<const T*>(kbase), p.k_ss, base, tid);
                mean.add();
            }
            mean.partial(lmean, tid);
        }
    };
    if (tl.nt > 0) {
        if constexpr (NBUF == 2) {
            commit(0, smem, smem + MAT);
            sample();
            __syncthreads();
            if constexpr (CENTRE) mean.finish(lmean, tid);
            for (int idx = 0; idx < tl.nt; ++idx) {
                const int cur = idx & 1;
                const bool more = idx + 1 < tl.nt;
                if (more) fetch(idx + 1);
                compute(idx, smem + 2 * cur * MAT, smem + (2 * cur + 1) * MAT);
                if (more) commit(idx + 1, smem + 2 * (cur ^ 1) * MAT, smem + (2 * (cur ^ 1) + 1) * MAT);
                __syncthreads();
            }
        } else {
            sample();
            if constexpr (CENTRE) {
                __syncthreads();
                mean.finish(lmean, tid);
            }
            for (int idx = 0; idx < tl.nt; ++idx) {
                commit(idx, smem, smem + MAT);
                __syncthreads();
                if (PRE && idx + 1 < tl.nt) fetch(idx + 1);
                compute(idx, smem, smem + MAT);
                __syncthreads();
                if (!PRE && idx + 1 < tl.nt) fetch(idx + 1);
            }
        }
        if constexpr (CENTRE) {
            rsum += __shfl_xor(rsum, 32, 64);
#pragma unroll
            for (int d = 0; d < G::DT; ++d)
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                    const f32x4 c = mean.at(lmean, 32 * d + 8 * jj + 4 * (lane >> 5));
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[d][4 * jj + e] = fmaf(-rsum, c[e], acc[d][4 * jj + e]);
                }
        }
    }
    const float scale = !DROP && r < win_single_rows(p, n) ? 0.f : p.dq_scale;
    if constexpr (KW == 1) {
        T* out = reinterpret_cast<T*>(p.dq) + (long)b * p.dq_bs + (long)head * p.dq_hs + (long)irel * p.dq_ss;
        store_rows<HD>(acc, scale, out, r < p.rows, lane);
    } else {
        constexpr int PJ = HD + 4;
        float* jo = reinterpret_cast<float*>(smem);
        store_rows<HD>(acc, scale, jo + (kw * 32 + (lane & 31)) * PJ, true, lane);
        __syncthreads();
        for (int u = tid; u < 32 * HD / 4; u += NT) {
            const int row = u / (HD / 4), c = (u - row * (HD / 4)) * 4, rr = r_first + row;
            if (rr >= p.rows) break;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < KW; ++w) v += *reinterpret_cast<const f32x4*>(jo + (w * 32 + row) * PJ + c);
            const int i = win_row_query(p, rr), h = hkv * p.G + rr - i * p.G;
            T* at = reinterpret_cast<T*>(p.dq) + (long)b * p.dq_bs + (long)h * p.dq_hs + (long)i * p.dq_ss + c;
            if constexpr (sizeof(T) == 2) {
                bf16x4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = (bf16_t)v[e];
                *reinterpret_cast<bf16x4*>(at) = w;
            } else {
                *reinterpret_cast<f32x4*>(at) = v;
            }
        }
    }
}

// ------------------------------------------------------------------ dK, dV
// rows (relative to the packed axis) that see a key of tile k0..k0+KT-1: blocks of RB rows [first, first + count)
struct RowBlocks { int first, count; };
__device__ __forceinline__ RowBlocks win_row_blocks(const WinArgs& p, int k0, int n) {
    if (k0 >= n) return {0, 0};
    const bool pre = k0 < p.prefix;
    const int lo = pre && p.open ? 0 : k0;
    const long far = (long)k0 + KT - 1 + p.window;                                  // first position past the window of the tile's last key
    const int hi = pre ? n : (int)min((long)n, far);
    const int i0 = max(0, lo - p.q_start), i1 = min(p.nq, hi - p.q_start);
    if (i1 <= i0) return {0, 0};
    const int first = i0 * p.G / RB;
    return {first, (i1 * p.G + RB - 1) / RB - first};
}

// The two pairs of products of a step, S = Q K^T and dP = dO V^T (s, dp), then dV += P^T dO and dK += dS^T Q, with the reads of
// LDS AH instructions ahead of the matrix instruction that takes them.  (Left to itself the compiler reads every fragment into
// the same registers and waits for it before each instruction: an LDS latency each, 4 HD / 16 times a step.  2, 3, 4 ahead are
// alike; the long case 324 -> 313 us, the captioning stack 140 -> 135 us.)
template <int HD>
__device__ __forceinline__ void step_rows(f32x16& s, f32x16& dp, const char* q, const char* d, const char* lkw, const RowFrag<bf16_t, HD>& vf, const LaneAt<bf16_t, HD>& at) {
    constexpr int N = HD / 16;
    bf16x8 a[2 * N], k[N];
    auto read = [&](int i) {
        a[i] = *reinterpret_cast<const bf16x8*>((i < N ? q : d) + at.row(i % N));
        if (i < N) k[i] = *reinterpret_cast<const bf16x8*>(lkw + at.row(i));
    };
#pragma unroll
    for (int i = 0; i < AH; ++i) read(i);
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
        if (i + AH < 2 * N) read(i + AH);
        __builtin_amdgcn_sched_barrier(0x6);                                // (the vector and scalar units' instructions may pass)
        if (i < N) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], k[i % N], s, 0, 0, 0);
        else dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], vf.f[i % N], dp, 0, 0, 0);
    }
}
template <int HD>
__device__ __forceinline__ void step_cols(f32x16 (&dv)[HD / 32], f32x16 (&dk)[HD / 32], const f32x16& pd, const f32x16& ds, const char* d, const char* q,
                                          const LaneAt<bf16_t, HD>& at) {
    constexpr int DT = HD / 32, N = 2 * DT, PB = WinGeo<bf16_t, HD>::PB;
    bf16x8 a[2 * N], b[4];
    auto read = [&](int i) {
        const char* from = (i < N ? d : q) + 16 * (i / DT % 2) * PB;
        const bf16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, from + at.col(i % DT)));
        const bf16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, from + at.col8(i % DT)));
        a[i] = __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
    };
#pragma unroll
    for (int i = 0; i < AH; ++i) read(i);
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
        if (i + AH < 2 * N) read(i + AH);
        if (i % DT == 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) b[i / DT][e] = (bf16_t)(i < N ? pd : ds)[8 * (i / DT % 2) + e];
        }
        __builtin_amdgcn_sched_barrier(0x6);
        f32x16& acc = (i < N ? dv : dk)[i % DT];
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[i / DT], acc, 0, 0, 0);
    }
}

// One step of a wave: RB rows (Q, dO, lse, delta, positions in buf) against its 32 keys (K's rows at lkw, V's in vf): adds to dK and
// dV and leaves dS [row 8 (e >> 2) + 4 (lane >> 5) + (e & 3)][key lane & 31] in s.  False: none of the rows sees any of the keys.
template <typename T, int HD, bool DROP>
__device__ __forceinline__ bool dkv_step(const WinArgs& p, const LaneAt<T, HD>& at0, int blk, const char* buf, const char* lkw, const RowFrag<T, HD>& vf, int b,
                                         int hkv, int n, int kw0, int lane, f32x16 (&dk)[HD / 32], f32x16 (&dv)[HD / 32], f32x16& s) {
    constexpr int MAT = RB * WinGeo<T, HD>::PB;
    const int key = kw0 + (lane & 31);
    const LaneAt<T, HD> at = at0.fresh();
    const int ra = blk * RB, rz = min(p.rows, ra + RB) - 1;
    const int pf = p.q_start + win_row_query(p, ra), pl = p.q_start + win_row_query(p, rz);
    const bool pre = kw0 < p.prefix;
    const bool band = pl >= kw0 && pf - p.window < kw0 + 31;
    if (kw0 >= n || !(band || (pre && (p.open || pl >= kw0)))) return false;
    f32x16 dp;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = dp[e] = 0.f;
    if constexpr (sizeof(T) == 2) {
        step_rows<HD>(s, dp, buf, buf + MAT, lkw, vf, at);
    } else {
        mma_rows_lds<HD>(s, buf, lkw, at);
        mma_rows<HD>(dp, buf + MAT, vf, at);
    }
    const float* st = reinterpret_cast<const float*>(buf + 2 * MAT) + 4 * (lane >> 5);
    const bool whole = kw0 + 32 <= n && ((pf >= kw0 + 31 && pl - p.window < kw0) || (kw0 + 32 <= p.prefix && (p.open || pf >= kw0 + 31)));
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
        const f32x4 lse = *reinterpret_cast<const f32x4*>(st + 8 * jj);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float x = sizeof(T) == 2 ? fmaf(s[4 * jj + e], WIN_LOG2E, -lse[e]) : (s[4 * jj + e] - lse[e]) * WIN_LOG2E;
            s[4 * jj + e] = __builtin_amdgcn_exp2f(x);
        }
    }
    if (!whole) {
        const int* ps0 = reinterpret_cast<const int*>(st) + 2 * RB;
        // key <= pos and pos < far, or (a key of the prefix) pos >= near: two intervals of positions per lane
        const int far = key < n ? key + p.window : 0;                                  // (window <= 2^30, key < 2^28)
        const int near = key < min(p.prefix, n) ? (p.open ? 0 : key) : 0x7FFFFFFF;
#pragma unroll
        for (int jj = 0; jj < 4; ++jj)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int pos = ps0[8 * jj + e];
                s[4 * jj + e] = ((pos >= near) | ((pos >= key) & (pos < far))) ? s[4 * jj + e] : 0.f;
            }
    }
    f32x16 pd = s;                                // what multiplies dO: the probabilities after dropout
    if constexpr (DROP) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int r = min(ra + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3), p.rows - 1);
            const int i = win_row_query(p, r), h = hkv * p.G + r - i * p.G;
            const uint32_t idx = (uint32_t)((((long)b * p.H + h) * p.S + p.q_start + i) * p.S4) + (uint32_t)key;
            const float f = dropout_keep(p.drop_k0, p.drop_k1, idx, p.drop_thr) ? p.drop_scale : 0.f;
            pd[e] *= f;
            dp[e] *= f;
        }
    }
#pragma unroll
    for (int jj = 0; jj < 4; ++jj) {
        const f32x4 delta = *reinterpret_cast<const f32x4*>(st + RB + 8 * jj);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[4 * jj + e] *= dp[4 * jj + e] - delta[e];
    }
    if constexpr (sizeof(T) == 2) {
        step_cols<HD>(dv, dk, pd, s, buf + MAT, buf, at);
    } else {
        mma_cols<HD>(dv, buf + MAT, pd, at);
        mma_cols<HD>(dk, buf, s, at);
    }
    return true;
}

template <typename T, int HD, bool DROP>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void win_dkv_kernel(WinArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    using G = WinGeo<T, HD>;
    constexpr int CPR = G::CPR, U = (RB * CPR + 255) / 256;
    constexpr int MAT = RB * G::PB;
    // [2 buffers] { Q, dO, 32 lse, 32 delta, 32 positions }
    constexpr int BUF = 2 * MAT + 3 * RB * 4;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const LaneAt<T, HD> at(lane);
    // the tiles past the prefix come first, the prefix' chunks (shorter, as a rule) fill up behind them; each kind is spread over
    // the XCDs by itself (in one order over both, one XCD had all the short ones of a head and the other half as many long
    // ones again as places: 8192 positions 128 wide, 144 steps one after the other where 88 do)
    const int bhs = p.B * p.Hkv, n_band = bhs * (p.ktiles - p.kp) * p.ncn;
    int bh, tile, chunk, nc, slot;
    if ((int)blockIdx.x < n_band) {
        const int id = win_xcd_id(blockIdx.x, n_band), per = (p.ktiles - p.kp) * p.ncn;
        bh = id / per;
        const int x = id - bh * per;
        tile = p.kp + x / p.ncn; chunk = x % p.ncn; nc = p.ncn;
        slot = (p.ncp > 1 ? p.kp * p.ncp : 0) + x;
    } else {
        const int id = win_xcd_id(blockIdx.x - n_band, bhs * p.kp * p.ncp), per = p.kp * p.ncp;
        bh = id / per;
        slot = id - bh * per;
        tile = slot / p.ncp; chunk = slot - tile * p.ncp; nc = p.ncp;
    }
    const int b = bh / p.Hkv, hkv = bh - b * p.Hkv;
    const int n = win_len(p, b);
    const int k0 = tile * KT, kw0 = k0 + 32 * wave, key = kw0 + (lane & 31);
    const RowBlocks rb = win_row_blocks(p, k0, n);
    const int b_begin = rb.first + (int)((long)rb.count * chunk / nc), b_end = rb.first + (int)((long)rb.count * (chunk + 1) / nc);

    // the next block's rows on their way: loaded whatever they hold (rows past the end repeat the last one), and what may not
    // be used -- rows at or past the sequence's end -- put to zero when they reach LDS, so that nothing here waits for a load
    u32x4 fq[U], fd[U];
    float f_lse = 0.f, f_delta = 0.f;
    const T* qb = reinterpret_cast<const T*>(p.q) + (long)b * p.q_bs + (long)(hkv * p.G) * p.q_hs;
    const T* db = reinterpret_cast<const T*>(p.dout) + (long)b * p.do_bs + (long)(hkv * p.G) * p.do_hs;
    const long stat0 = ((long)b * p.H + hkv * p.G) * p.nq;
    auto fetch = [&](int blk) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int u = tid + 256 * j, row = u / CPR, ch = u - row * CPR;
            const int r = min(blk * RB + row, p.rows - 1), i = win_row_query(p, r), g = r - i * p.G;
            fq[j] = *reinterpret_cast<const u32x4*>(qb + (long)g * p.q_hs + (long)i * p.q_ss + ch * (16 / (int)sizeof(T)));
            fd[j] = *reinterpret_cast<const u32x4*>(db + (long)g * p.do_hs + (long)i * p.do_ss + ch * (16 / (int)sizeof(T)));
        }
        if (tid < RB) {
            const int r = min(blk * RB + tid, p.rows - 1), i = win_row_query(p, r), g = r - i * p.G;
            f_lse = p.lse[stat0 + (long)g * p.nq + i];
            f_delta = p.delta[stat0 + (long)g * p.nq + i];
        }
    };
    const WinSpan any = win_union(p, p.q_start, p.q_start + p.nq - 1, n);
    // K's rows stay in LDS and V's in registers: with both in registers the accumulators no longer fit beside them
    char* lk = smem + 2 * BUF;
    RowFrag<T, HD> vf;
    vf.zero();
    {
        u32x4 z[KT * CPR / 256];
#pragma unroll
        for (int j = 0; j < KT * CPR / 256; ++j) {
            const int u = tid + 256 * j, row = u / CPR, ch = u - row * CPR;
            z[j] = u32x4{0, 0, 0, 0};
            if (win_sees(any, k0 + row))
                z[j] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const T*>(p.k) + (long)b * p.k_bs + (long)hkv * p.k_hs + (long)(k0 + row) * p.k_ss + ch * (16 / (int)sizeof(T)));
        }
        if (win_sees(any, key)) vf.load(reinterpret_cast<const T*>(p.v) + (long)b * p.v_bs + (long)hkv * p.v_hs + (long)key * p.v_ss, lane);
        if (b_begin < b_end) fetch(b_begin);
#pragma unroll
        for (int j = 0; j < KT * CPR / 256; ++j) {
            const int u = tid + 256 * j, row = u / CPR, ch = u - row * CPR;
            *reinterpret_cast<u32x4*>(lk + G::at(row, ch)) = z[j];
        }
    }
    vf.landed();
    const char* lkw = lk + 32 * wave * G::PB;
    f32x16 dk[G::DT], dv[G::DT];
#pragma unroll
    for (int d = 0; d < G::DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[d][e] = dv[d][e] = 0.f;

    const int single = DROP ? 0 : win_single_rows(p, n);          // (with dropout o is V scaled and rounded: delta is the formula's with that o)
    auto commit = [&](int blk, char* buf) {
        // rows of a block are in the order of their positions: those before the sequence's end come first
        // (queries are counted before they are multiplied by the heads: (S - q_start) * G may pass 32 bits, rows = nq * G does not)
        const int live = min(p.nq, max(0, n - p.q_start)) * p.G - blk * RB;
        const int alone = single - blk * RB;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int u = tid + 256 * j, row = u / CPR, ch = u - row * CPR;
            if (RB * CPR % 256 == 0 || row < RB) {
                const u32x4 z = {0, 0, 0, 0};
                *reinterpret_cast<u32x4*>(buf + G::at(row, ch)) = (row < live) & (row >= alone) ? fq[j] : z;
                *reinterpret_cast<u32x4*>(buf + MAT + G::at(row, ch)) = row < live ? fd[j] : z;
            }
        }
        if (tid < RB) {
            float* st = reinterpret_cast<float*>(buf + 2 * MAT);
            // rows that are not there, and rows that see nothing: probability 0.  (bf16: in units of the exponent of 2)
            // rows that see one key: probability 1 from a score of 0, and nothing for dK
            st[tid] = tid >= live || f_lse == -INFINITY ? INFINITY : tid < alone ? 0.f : (sizeof(T) == 2 ? f_lse * WIN_LOG2E : f_lse);
            st[RB + tid] = tid >= live ? 0.f : f_delta;
            reinterpret_cast<int*>(st)[2 * RB + tid] = p.q_start + win_row_query(p, min(blk * RB + tid, p.rows - 1));
        }
    };
    auto compute = [&](int blk, const char* buf) {
        f32x16 ds;
        dkv_step<T, HD, DROP>(p, at, blk, buf, lkw, vf, b, hkv, n, kw0, lane, dk, dv, ds);
    };
    if (b_begin < b_end) {
        commit(b_begin, smem);
        __syncthreads();
        for (int blk = b_begin; blk < b_end; ++blk) {
            const int cur = (blk - b_begin) & 1;
            const bool more = blk + 1 < b_end;
            if (more) fetch(blk + 1);
            compute(blk, smem + cur * BUF);
            if (more) commit(blk + 1, smem + (cur ^ 1) * BUF);
            __syncthreads();
        }
    }
    if (nc == 1) {
        const bool ok = key < p.S;
        store_rows<HD>(dk, 1.f, reinterpret_cast<T*>(p.dk) + (long)b * p.dk_bs + (long)hkv * p.dk_hs + (long)min(key, p.S - 1) * p.dk_ss, ok, lane);
        store_rows<HD>(dv, 1.f, reinterpret_cast<T*>(p.dv) + (long)b * p.dv_bs + (long)hkv * p.dv_hs + (long)min(key, p.S - 1) * p.dv_ss, ok, lane);
    } else {
        const long slots = (p.ncp > 1 ? p.kp * p.ncp : 0) + (p.ncn > 1 ? (p.ktiles - p.kp) * p.ncn : 0);
        float* at = p.part + ((bh * slots + slot) * 2L * KT + 32 * wave + (lane & 31)) * HD;
        store_rows<HD>(dk, 1.f, at, true, lane);
        store_rows<HD>(dv, 1.f, at + (long)KT * HD, true, lane);
    }
}

// dK and dV of the tiles that were cut into chunks: the partial sums in chunk order.  Grid: (column pieces of a tile, cut tiles, B * Hkv)
template <typename T, int HD>
__global__ __launch_bounds__(256) void win_dkv_join_kernel(WinArgs p) {
    const int x = blockIdx.y, bh = blockIdx.z;
    const int np = p.ncp > 1 ? p.kp : 0;
    const int tile = x < np ? x : p.kp + (x - np), nc = x < np ? p.ncp : p.ncn;
    const long slots = (p.ncp > 1 ? p.kp * p.ncp : 0) + (p.ncn > 1 ? (p.ktiles - p.kp) * p.ncn : 0);
    const long slot0 = x < np ? (long)x * p.ncp : (long)np * p.ncp + (long)(x - np) * p.ncn;
    const int u = blockIdx.x * 256 + threadIdx.x;                         // four columns of dK (first half) or dV
    const int which = u / (KT * HD / 4), c4 = u - which * (KT * HD / 4);
    const int row = c4 / (HD / 4), c = (c4 - row * (HD / 4)) * 4, key = tile * KT + row;
    if (which > 1 || key >= p.S) return;
    const float* at = p.part + ((bh * slots + slot0) * 2 + which) * (long)KT * HD + (long)row * HD + c;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    int s = 0;
    for (; s + 16 <= nc; s += 16) {                                       // sixteen loads at a time, added in order
        f32x4 x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = *reinterpret_cast<const f32x4*>(at + (long)(s + e) * 2 * KT * HD);
#pragma unroll
        for (int e = 0; e < 16; ++e) v += x[e];
    }
    for (; s < nc; ++s) v += *reinterpret_cast<const f32x4*>(at + (long)s * 2 * KT * HD);
    const int b = bh / p.Hkv, hkv = bh - b * p.Hkv;
    T* out = which == 0 ? reinterpret_cast<T*>(p.dk) + (long)b * p.dk_bs + (long)hkv * p.dk_hs + (long)key * p.dk_ss + c
                        : reinterpret_cast<T*>(p.dv) + (long)b * p.dv_bs + (long)hkv * p.dv_hs + (long)key * p.dv_ss + c;
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = from_f32<T>(v[e]);
}

// ------------------------------------------------------------------ all three of short sequences
// At most 256 keys: one workgroup has them all, eight waves of 32, and goes over the rows once.  A step is dkv_step's; its dS
// (bf16, as both products take it) also goes to LDS as [key][row], and after every four steps each wave multiplies half of the
// channels of one of the four blocks' dQ out of it: dQ^T = K^T dS^T with both operands read by columns.  Five products instead of
// seven, q, k, v and dO read once instead of twice, and delta formed where dO passes by.  1024 heads of 229 rows of 96 channels:
// 126-130 us against 147 for the two kernels; the 360 MB alone take 77, the rest is the phases of a CU's one workgroup (147 KB of
// LDS, eight waves of 217 registers) following each other: K and V 26, the last stores 21, dQ 20.  One workgroup per CU that
// loads its next head's K and V during dQ measured the same, and so did dQ's reads a block ahead.
constexpr int SK = 256;
template <int HD> struct ShortGeo {
    using G = WinGeo<bf16_t, HD>;
    static constexpr int MAT = RB * G::PB, BUF = 2 * MAT + 3 * RB * 4, KB = SK * G::PB, DS = SK * RB * 2;
    static constexpr int LDS = 2 * BUF + KB + 4 * DS + KeyMean<HD, 512>::BYTES;
};
template <int HD, bool DROP>
__global__ __launch_bounds__(512, 2) void win_bwd_short_kernel(WinArgs p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    using T = bf16_t;
    using G = WinGeo<T, HD>;
    using L = ShortGeo<HD>;
    using D = WinGeo<T, RB>;
    constexpr int CPR = G::CPR, NZ = SK * CPR / 512, NT = HD / 32;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const LaneAt<T, HD> at(lane);
    const int bh = win_xcd_id(blockIdx.x, gridDim.x);
    const int b = bh / p.Hkv, hkv = bh - b * p.Hkv;
    const int n = win_len(p, b);
    const int kw0 = 32 * wave, key = kw0 + (lane & 31);
    char* lk = smem + 2 * L::BUF;
    char* lds_ds = lk + L::KB;
    char* lmean = lds_ds + 4 * L::DS;
    KeyMean<HD, 512> mean;
    const int nblk = (p.rows + RB - 1) / RB;

    // rows on their way: sixteen lanes to a row (of which CPR load), four rows to a wave
    const int srow = 4 * wave + (lane >> 4), ch = lane & 15;
    const bool loads = ch < CPR;
    const int che = (loads ? ch : 0) * 8;
    u32x4 fq, fd, fo;
    float f_lse;
    const int single = DROP ? 0 : win_single_rows(p, n);
    auto fetch = [&](int blk) {
        const int r = min(blk * RB + srow, p.rows - 1), i = win_row_query(p, r), h = hkv * p.G + r - i * p.G;
        fq = *reinterpret_cast<const u32x4*>(reinterpret_cast<const T*>(p.q) + (long)b * p.q_bs + (long)h * p.q_hs + (long)i * p.q_ss + che);
        fd = *reinterpret_cast<const u32x4*>(reinterpret_cast<const T*>(p.dout) + (long)b * p.do_bs + (long)h * p.do_hs + (long)i * p.do_ss + che);
        fo = *reinterpret_cast<const u32x4*>(reinterpret_cast<const T*>(p.o) + (long)b * p.o_bs + (long)h * p.o_hs + (long)i * p.o_ss + che);
        f_lse = p.lse[((long)b * p.H + h) * p.nq + i];
    };
    auto commit = [&](int blk, char* buf) {
        const bool live = srow < min(p.nq, max(0, n - p.q_start)) * p.G - blk * RB;
        const bool alone = srow < single - blk * RB;
        const u32x4 z = {0, 0, 0, 0};
        fd = live ? fd : z;
        fo = live ? fo : z;
        if (loads) {
            *reinterpret_cast<u32x4*>(buf + G::at(srow, ch)) = live & !alone ? fq : z;
            *reinterpret_cast<u32x4*>(buf + L::MAT + G::at(srow, ch)) = fd;
        }
        const bf16x8 x = __builtin_bit_cast(bf16x8, fd), y = __builtin_bit_cast(bf16x8, fo);
        float delta = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf((float)x[e], (float)y[e], delta);
        delta = sum16(loads ? delta : 0.f);
        if (ch == 0) {
            float* st = reinterpret_cast<float*>(buf + 2 * L::MAT);
            st[srow] = !live || f_lse == -INFINITY ? INFINITY : alone ? 0.f : f_lse * WIN_LOG2E;
            st[RB + srow] = delta;
            reinterpret_cast<int*>(st)[2 * RB + srow] = p.q_start + win_row_query(p, min(blk * RB + srow, p.rows - 1));
        }
    };

    const WinSpan any = win_union(p, p.q_start, p.q_start + p.nq - 1, n);
    RowFrag<T, HD> vf;
    vf.zero();
    {
        u32x4 z[NZ];
#pragma unroll
        for (int j = 0; j < NZ; ++j) {
            const int u = tid + 512 * j, row = u / CPR, c = u - row * CPR;
            z[j] = u32x4{0, 0, 0, 0};
            if (win_sees(any, row)) z[j] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const T*>(p.k) + (long)b * p.k_bs + (long)hkv * p.k_hs + (long)row * p.k_ss + c * 8);
        }
        if (win_sees(any, key)) vf.load(reinterpret_cast<const T*>(p.v) + (long)b * p.v_bs + (long)hkv * p.v_hs + (long)key * p.v_ss, lane);
        fetch(0);
#pragma unroll
        for (int j = 0; j < NZ; ++j) {
            const int u = tid + 512 * j, row = u / CPR, c = u - row * CPR;
            *reinterpret_cast<u32x4*>(lk + G::at(row, c)) = z[j];
        }
    }
    vf.landed();
    f32x16 dk[G::DT], dv[G::DT];
#pragma unroll
    for (int d = 0; d < G::DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[d][e] = dv[d][e] = 0.f;

    commit(0, smem);
    __syncthreads();
    mean.pick(any);
    mean.load(lk, tid);                                                     // (read from memory once more: 2048 heads of 48 rows of 64 channels 97 -> 107 us)
    mean.add();
    mean.partial(lmean, tid);
    for (int blk0 = 0; blk0 < nblk; blk0 += 4) {
        for (int blk = blk0; blk < min(blk0 + 4, nblk); ++blk) {
            const bool more = blk + 1 < nblk;
            if (more) fetch(blk + 1);
            f32x16 ds;
            if (!dkv_step<T, HD, DROP>(p, at, blk, smem + (blk & 1) * L::BUF, lk + kw0 * G::PB, vf, b, hkv, n, kw0, lane, dk, dv, ds)) {
#pragma unroll
                for (int e = 0; e < 16; ++e) ds[e] = 0.f;
            }
            char* to = lds_ds + (blk & 3) * L::DS;
#pragma unroll
            for (int jj = 0; jj < 4; ++jj)
                *reinterpret_cast<u32x2*>(to + D::at(key, jj) + 8 * (lane >> 5)) =
                    u32x2{win_pack(ds[4 * jj], ds[4 * jj + 1]), win_pack(ds[4 * jj + 2], ds[4 * jj + 3])};
            if (more) commit(blk + 1, smem + ((blk + 1) & 1) * L::BUF);
            __syncthreads();
            if (blk == 0) {                                                 // (read after the next step's barrier)
                mean.finish(lmean, tid);
                if (!more) __syncthreads();
            }
        }
        // 16x16x32 products: lane l holds column l & 15 of either operand and the keys 4 (l >> 4) + 0..3 and 16 + 4 (l >> 4) + 0..3
        const int rb = wave & 3, half = wave >> 2;
        if (blk0 + rb < nblk) {
            const int g = lane >> 4, i16 = lane & 15, krow = 4 * g + (i16 >> 2), sub = (i16 & 3) >> 1, byte = 8 * (i16 & 1);
            int koff[NT], doff[2];
#pragma unroll
            for (int t = 0; t < NT; ++t) koff[t] = G::at(krow, half * (CPR / 2) + 2 * t + sub) + byte;
#pragma unroll
            for (int rh = 0; rh < 2; ++rh) doff[rh] = D::at(krow, 2 * rh + sub) + byte;
            f32x4 acc[2][NT];
            float rsum[2] = {0.f, 0.f};
#pragma unroll
            for (int rh = 0; rh < 2; ++rh)
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[rh][t] = f32x4{0.f, 0.f, 0.f, 0.f};
            auto col = [](const char* at0, int pb) {
                const bf16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, at0));
                const bf16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, at0 + 16 * pb));
                return __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
            };
            const int kb_end = min(8, (n + 31) >> 5);                        // (keys past the end are zero in both)
            for (int kb = 0; kb < kb_end; ++kb) {
                bf16x8 x[2];
#pragma unroll
                for (int rh = 0; rh < 2; ++rh) {
                    x[rh] = col(lds_ds + rb * L::DS + kb * 32 * D::PB + doff[rh], D::PB);
                    rsum[rh] = win_sum8(x[rh], rsum[rh]);
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const bf16x8 kc = col(lk + kb * 32 * G::PB + koff[t], G::PB);
#pragma unroll
                    for (int rh = 0; rh < 2; ++rh) acc[rh][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kc, x[rh], acc[rh][t], 0, 0, 0);
                }
            }
#pragma unroll
            for (int rh = 0; rh < 2; ++rh) {
                rsum[rh] += __shfl_xor(rsum[rh], 16, 64);
                rsum[rh] += __shfl_xor(rsum[rh], 32, 64);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const f32x4 c = mean.at(lmean, half * (HD / 2) + 16 * t + 4 * g);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[rh][t][e] = fmaf(-rsum[rh], c[e], acc[rh][t][e]);
                }
                const int r = (blk0 + rb) * RB + 16 * rh + i16;
                if (r >= p.rows) continue;
                const int i = win_row_query(p, r), h = hkv * p.G + r - i * p.G;
                T* out = reinterpret_cast<T*>(p.dq) + (long)b * p.dq_bs + (long)h * p.dq_hs + (long)i * p.dq_ss + half * (HD / 2) + 4 * g;
                const float scale = r < single ? 0.f : p.dq_scale;
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    *reinterpret_cast<u32x2*>(out + 16 * t) = u32x2{win_pack(acc[rh][t][0] * scale, acc[rh][t][1] * scale),
                                                                    win_pack(acc[rh][t][2] * scale, acc[rh][t][3] * scale)};
            }
        }
        if (blk0 + 4 < nblk) __syncthreads();                               // the next step writes dS where this one was read
    }
    const bool ok = key < p.S;
    const int ks = min(key, p.S - 1);
    store_rows<HD>(dk, 1.f, reinterpret_cast<T*>(p.dk) + (long)b * p.dk_bs + (long)hkv * p.dk_hs + (long)ks * p.dk_ss, ok, lane);
    store_rows<HD>(dv, 1.f, reinterpret_cast<T*>(p.dv) + (long)b * p.dv_bs + (long)hkv * p.dv_hs + (long)ks * p.dv_ss, ok, lane);
}

// ------------------------------------------------------------------ launch
struct BwdPlan { int ktiles, kp, ncp, ncn; long part_floats; };
BwdPlan bwd_plan(int B, int H, int Hkv, int S, int nq, int hd, int window, int prefix) {
    BwdPlan pl;
    const int G = H / Hkv;
    const long bh = (long)B * Hkv, rows = (long)nq * G;
    pl.ktiles = (S + KT - 1) / KT;
    const int pre = prefix < S ? prefix : S;
    const long w = window == 0 || window > S ? S : window;
    pl.kp = (pre + KT - 1) / KT;
    const long all = (rows + RB - 1) / RB;                                 // row blocks a prefix tile sees
    long band = ((w + KT) * G + RB - 1) / RB;                              // and another one
    if (band > all) band = all;
    // enough workgroups for two per CU; a chunk's partial sums cost about what two steps do, so none has fewer than 16 steps
    // -- unless the tiles do not even give every other CU a workgroup, where latency counts: two.  Measured (us), not cut | aimed at
    // 256 | 512 | 1024 workgroups, then 512 of at least 2 | 8 | 16 | 32 steps:
    //   1 x 8192, 16 heads on 4 of 128, window 1024 + 4: 1780 | 333 | 309 | 332,  324 | 324 | 309 | 330
    //   8 x 1024, 16 on 4 of 128, causal:                 266 | 266 | 227 | 213,  227 | 227 | 227 | 227
    //   1 x 2048, 4 on 2 of 64, causal:                   158 |  56 |  52 |  61,   52 |  51 |  56 |  68
    //   1 x 4100, 4 on 2 of 32, window 70 + 4:            407 |  37 |  36 |  36,   36 |  37 |  43 |  68
    //   2 x 500, 8 on 2 of 128, causal:                   111 |  44 |  50 |  49,   49 |  47 |  61 | 113
    //   3 x 333, 4 on 2 of 64, window 50, f32:             88 |  42 |  42 |  42,   42 |  88 |  88 |  88
    const long least = bh * pl.ktiles < 128 ? 2 : 16;
    auto chunks = [least](long wgs, long steps) {
        long c = wgs > 0 ? (512 + wgs - 1) / wgs : 1;
        if (c > steps / least) c = steps / least;
        return (int)(c < 1 ? 1 : c);
    };
    pl.ncn = chunks(bh * pl.ktiles, band);
    pl.ncp = pl.kp ? chunks(bh * pl.kp, all) : 1;
    if (pl.ncp < pl.ncn) pl.ncp = pl.ncn;
    const long slots = (pl.ncp > 1 ? (long)pl.kp * pl.ncp : 0) + (pl.ncn > 1 ? (long)(pl.ktiles - pl.kp) * pl.ncn : 0);
    pl.part_floats = bh * slots * 2 * KT * hd;
    return pl;
}

// One kernel for short sequences in bf16: where its workgroups, one per K/V head, fill the card or have few rows to go over one
// after the other.  Measured in us, one kernel against the two (229 keys, all rows | 32 rows; H = Hkv):
//   96 channels,  16 heads:  26 /  26 |  9 / 15     64 channels,  16 heads:  24 /  23 |  8 / 14     32 channels,  16 heads: 23 / 17 |  7 / 11
//                256 heads:  35 /  43 | 14 / 21                  256 heads:  31 /  37 | 11 / 18                  256 heads: 27 / 29 |  8 / 13
//                512 heads:  62 /  79 | 27 / 35                  512 heads:  56 /  63 | 22 / 27                  512 heads: 51 / 42 | 15 / 18
//               1024 heads: 126 / 147                           1024 heads: 105 / 102                           1024 heads: 96 / 72
// (and 64 keys, 512 heads: 19 / 21, 16 / 17, 16 / 14).  With 32 channels the products are too small a part of a step; with 128 the
// accumulators, V and the fragments no longer fit the registers.
template <typename T, int HD> constexpr bool HAS_SHORT = sizeof(T) == 2 && (HD == 64 || HD == 96);
bool win_bwd_short(long bh, long rows, int S) { return S <= SK && (rows <= 256 || bh >= 256); }
bool win_bwd_one_kernel(int dtype, int hd, long bh, long rows, int S) {
    return dtype == CAPDEC_BF16 && (hd == 64 ? HAS_SHORT<bf16_t, 64> : hd == 96 && HAS_SHORT<bf16_t, 96>) && win_bwd_short(bh, rows, S);
}

template <typename T, int HD, bool DROP>
int bwd_go(WinArgs& a, hipStream_t st) {
    using G = WinGeo<T, HD>;
    const long bh = (long)a.B * a.Hkv;
    if constexpr (HAS_SHORT<T, HD>) {
        if (win_bwd_short(bh, a.rows, a.S)) {
            auto kfn = win_bwd_short_kernel<HD, DROP>;
            static_assert(ShortGeo<HD>::LDS <= 160 * 1024, "LDS of a CU");
            ensure_dynamic_lds((const void*)kfn, ShortGeo<HD>::LDS);
            hipLaunchKernelGGL(kfn, dim3((unsigned)bh), dim3(512), ShortGeo<HD>::LDS, st, a);
            CAPDEC_LAUNCH_CHECK();
            return CAPDEC_OK;
        }
    }
    {
        const bool kw = win_few_rows(sizeof(T) == 4, bh, a.rows);
        a.tiles = (a.rows + (kw ? 31 : 127)) / (kw ? 32 : 128);
        CAPDEC_CHECK(bh * a.tiles < (1L << 31), "attn_window_bwd: grid too large");
        auto go = [&](auto kfn, int lds) {
            if (lds > 64 * 1024) ensure_dynamic_lds((const void*)kfn, lds);
            hipLaunchKernelGGL(kfn, dim3((unsigned)(bh * a.tiles)), dim3(256), lds, st, a);
        };
        if (kw) go(win_dq_kernel<T, HD, 1, 4, DROP>, DqLds<T, HD, 1, 4>::BYTES);
        else go(win_dq_kernel<T, HD, 4, 1, DROP>, DqLds<T, HD, 4, 1>::BYTES);
        CAPDEC_LAUNCH_CHECK();
    }
    const long grid = bh * ((long)a.kp * a.ncp + (long)(a.ktiles - a.kp) * a.ncn);
    CAPDEC_CHECK(grid < (1L << 31), "attn_window_bwd: grid too large");
    auto kfn = win_dkv_kernel<T, HD, DROP>;
    constexpr int lds = 2 * (2 * RB * G::PB + 3 * RB * 4) + KT * G::PB;
    if (lds > 64 * 1024) ensure_dynamic_lds((const void*)kfn, lds);
    hipLaunchKernelGGL(kfn, dim3((unsigned)grid), dim3(256), lds, st, a);
    CAPDEC_LAUNCH_CHECK();
    const int cut = (a.ncp > 1 ? a.kp : 0) + (a.ncn > 1 ? a.ktiles - a.kp : 0);
    if (cut > 0) {
        hipLaunchKernelGGL((win_dkv_join_kernel<T, HD>), dim3((2 * KT * HD / 4 + 255) / 256, cut, (unsigned)bh), dim3(256), 0, st, a);
        CAPDEC_LAUNCH_CHECK();
    }
    return CAPDEC_OK;
}
template <typename T, int HD> int bwd_hd(WinArgs& a, hipStream_t st) {
    return a.drop_thr ? bwd_go<T, HD, true>(a, st) : bwd_go<T, HD, false>(a, st);
}
template <typename T> int bwd_type(WinArgs& a, int hd, hipStream_t st) {
    switch (hd) {
        case 32: return bwd_hd<T, 32>(a, st);
        case 64: return bwd_hd<T, 64>(a, st);
        case 96: return bwd_hd<T, 96>(a, st);
        default: return bwd_hd<T, 128>(a, st);
    }
}

}  // namespace

extern "C" long capdec_attn_window_bwd_workspace(int B, int H, int Hkv, int S, int nq, int hd, int window, int prefix_len) {
    if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || S <= 0 || nq <= 0 || hd <= 0 || window < 0 || prefix_len < 0) return 0;
    return bwd_plan(B, H, Hkv, S, nq, hd, window, prefix_len).part_floats * 4;
}

extern "C" int capdec_attn_window_bwd(const capdec_attn_window_bwd_desc* d, void* stream) {
    CAPDEC_CHECK(d != nullptr, "attn_window_bwd: null descriptor");
    WinArgs a;
    const int rc = win_fill(&d->fwd, a, "attn_window_bwd");
    if (rc != CAPDEC_OK) return rc;
    CAPDEC_CHECK(d->dout && d->dq && d->dk && d->dv && d->delta && a.lse, "attn_window_bwd: null pointer");
    CAPDEC_CHECK(aligned16(d->dout) && aligned16(d->dq) && aligned16(d->dk) && aligned16(d->dv), "attn_window_bwd: operands must be 16-byte aligned");
    const int per16 = d->fwd.dtype == CAPDEC_BF16 ? 8 : 4;
    const long strides[] = {d->do_bs, d->do_hs, d->do_ss, d->dq_bs, d->dq_hs, d->dq_ss, d->dk_bs, d->dk_hs, d->dk_ss, d->dv_bs, d->dv_hs, d->dv_ss};
    for (long s : strides) CAPDEC_CHECK(s >= 0 && s % per16 == 0, "attn_window_bwd: stride %ld (must be a non-negative multiple of %d elements)", s, per16);
    BwdPlan pl = bwd_plan(a.B, a.H, a.Hkv, a.S, a.nq, d->fwd.hd, d->fwd.window, a.prefix);
    if (win_bwd_one_kernel(d->fwd.dtype, d->fwd.hd, (long)a.B * a.Hkv, a.rows, a.S)) pl.part_floats = 0;       // (no partial sums there)
    CAPDEC_CHECK((long)a.B * a.Hkv < 65536 || pl.part_floats == 0, "attn_window_bwd: B * Hkv %ld", (long)a.B * a.Hkv);
    if (pl.part_floats > 0) {
        if (!d->fwd.workspace || d->fwd.workspace_bytes < pl.part_floats * 4) {
            capdec_set_error("attn_window_bwd: workspace %ld bytes < %ld", d->fwd.workspace ? d->fwd.workspace_bytes : 0L, pl.part_floats * 4);
            return CAPDEC_ERR_WORKSPACE;
        }
        CAPDEC_CHECK(aligned16(d->fwd.workspace), "attn_window_bwd: workspace must be 16-byte aligned");
    }
    a.dout = d->dout; a.do_bs = d->do_bs; a.do_hs = d->do_hs; a.do_ss = d->do_ss;
    a.dq = d->dq; a.dq_bs = d->dq_bs; a.dq_hs = d->dq_hs; a.dq_ss = d->dq_ss;
    a.dk = d->dk; a.dk_bs = d->dk_bs; a.dk_hs = d->dk_hs; a.dk_ss = d->dk_ss;
    a.dv = d->dv; a.dv_bs = d->dv_bs; a.dv_hs = d->dv_hs; a.dv_ss = d->dv_ss;
    a.dq_scale = d->dq_scale; a.delta = d->delta;
    a.ktiles = pl.ktiles; a.kp = pl.kp; a.ncp = pl.ncp; a.ncn = pl.ncn; a.part = (float*)d->fwd.workspace;
    return d->fwd.dtype == CAPDEC_BF16 ? bwd_type<bf16_t>(a, d->fwd.hd, (hipStream_t)stream) : bwd_type<float>(a, d->fwd.hd, (hipStream_t)stream);
}

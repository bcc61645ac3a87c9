// A K/V cache held in 4 bits per value, and attention of one token per sequence over it.
//
// Format.  A row (one position, one head, K or V) is cut into groups of 32 channels; a group keeps a bf16 scale and a bf16
// offset next to its 32 levels 0..15, and stands for offset + scale * level (scale * level is exact in f32, the sum is rounded
// once on read-back; the attention applies offset and scale apart, so it can differ from that in the last bit):
//     offset = bf16(min), scale = bf16((max - min) * f32(1/15)), level = clamp(rint((x - offset) * (1 / scale)), 0, 15)
// in f32 steps (all levels 0 where the scale is 0).  5 bits a value against 16.
//
// Layout.  One contiguous piece per (sequence, K/V head): K levels, V levels, K scales, V scales, for smax rounded up to
// 32 rows.  The levels lie as the matrix cores take them, so that the attention neither transposes nor moves anything
// between lanes (16x16x32 products: lane l holds index l & 15 of one operand and eight consecutive k = 8 (l >> 4) + e):
//   K, tiles of 16 keys:  [tile][g = l >> 4][key][32-channel group t]  one 32-bit word = channels 32 t + 8 g + 0..7 of a key
//   V, blocks of 32 keys: [block][half][g][channel c][w]               one word = 8 keys of channel 16 (half * DW + w) + c,
//                         keys 4 g + 0..3 and 16 + 4 g + 0..3
//   nibble j holds k = 2 j, nibble j + 4 holds k = 2 j + 1: (x << 3 >> 4 j) & 0x00780078 | 0x3F803F80 is the pair (k = 2 j, 2 j + 1) as
//   two bf16 numbers 1 + level / 16 -- one shift and one and-or for two operands, no conversion.
//   scales: [key][t] words, scale in the low half, offset in the high half.
//
// Attention over it, in bf16.  With the level as 1 + n/16 and q' = 16 q:  sum_c q n = sum_c q' (1 + n/16) - sum_c q', the correction
// being the product's initial accumulator.  S [head][key] has one key per lane, so a key's scales are that lane's own
// loads:  s = sum_t scale_t (q . n)_t + offset_t (sum of q over t).  For O, p scale_t 16 becomes the bf16 operand r (rounded once, half a
// step), and what the operand carries beyond p's own weight is taken out around the middle level:
//     sum_j p (offset + scale n) = sum_j r (1 + n/16)  +  sum_j [ p (offset + 7.5 scale) - r (1 + 7.5/16) ]  up to  (r - 16 p scale) (n - 7.5) / 16,
// the bracket kept per lane and added at the end (around level 0 the rounding's share was twice as large).
// In f32 the levels become n - 7.5 instead (more instructions; 1 + n/16 costs the sums 23.5 / 4.6 of their digits), q and
// p scale_t are split into three bf16 parts, which together are the f32 numbers: three products instead of one, on matrix
// cores that are idle most of the time anyway.
// What bounds it is HBM: 5 bits a value, read once (the vector unit is active 0.52-0.62 of the time, unpacking).  Four waves of a workgroup take alternate blocks of 32 keys, each with its next block's
// loads in flight, and join at the end; few sequences are cut along the keys, joined by kv4_join_kernel.
//
// Measured (bf16, us): 4 sequences of up to 131072 rows (32 heads on 8 of 128) 85 = 410 MB at 4.8 TB/s; 256
// sequences of 229 rows (8 heads of 96) 14.4-16 = 57 MB at 3.6-4 TB/s, two blocks a wave, the rest is starting and joining.  Append of
// 256 x 198 rows 65 (3.2 TB/s read and written; 48 when nothing wrote before it), read-back of them to f32 70 (5.1 TB/s).
#include "common.h"

namespace {

constexpr float LOG2E = 1.44269504088896340736f;

template <int HD> struct K4 {
    static constexpr int NG = HD / 32;                   // groups of a row = words of K per lane and tile
    static constexpr int NL = HD > 64 ? 2 : 1;           // loads of V per lane and block
    static constexpr int DW = HD / 16 / NL;              // words of each
    static constexpr int DT = HD / 16;
};
// byte offsets inside a (sequence, head) piece; sm = smax rounded up to 32
__host__ __device__ __forceinline__ long k4_piece(long sm, int hd) { return sm * (hd + hd / 4); }
__device__ __forceinline__ long k4_v(long sm, int hd) { return sm * (hd / 2); }
__device__ __forceinline__ long k4_ks(long sm, int hd) { return sm * hd; }
__device__ __forceinline__ long k4_vs(long sm, int hd) { return sm * (hd + hd / 8); }
template <int HD> __device__ __forceinline__ long k4_k_word(int key, int t, int g) { return (((long)(key >> 4) * 64 + g * 16 + (key & 15)) * K4<HD>::NG + t) * 4; }
template <int HD> __device__ __forceinline__ long k4_v_word(int block, int dt, int g, int c) {
    using G = K4<HD>;
    return (((long)block * G::NL + dt / G::DW) * 64 + g * 16 + c) * (G::DW * 4) + (dt % G::DW) * 4;
}

template <int N> __device__ __forceinline__ void load_words(unsigned (&w)[N], const char* at) { __builtin_memcpy(w, __builtin_assume_aligned(at, N == 3 ? 4 : 4 * N), 4 * N); }

// eight levels of a word as bf16 numbers 1 + n / 16, in k order
__device__ __forceinline__ bf16x8 k4_expand(unsigned w) {
    return __builtin_bit_cast(bf16x8, (u32x4{((w << 3) & 0x00780078u) | 0x3F803F80u, ((w >> 1) & 0x00780078u) | 0x3F803F80u,
                                             ((w >> 5) & 0x00780078u) | 0x3F803F80u, ((w >> 9) & 0x00780078u) | 0x3F803F80u}));
}
// the same as n - 7.5 (five bits: exact)
__device__ __forceinline__ bf16x8 k4_centred(unsigned w) {
    u32x4 out;
#pragma unroll
    for (int j = 0; j < 4; ++j) {                                            // k = 2 j in nibble j, k = 2 j + 1 in nibble j + 4
        const float lo = (float)((w >> (4 * j)) & 15u) - 7.5f, hi = (float)((w >> (4 * j + 16)) & 15u) - 7.5f;
        out[j] = (__float_as_uint(lo) >> 16) | (__float_as_uint(hi) & 0xFFFF0000u);
    }
    return __builtin_bit_cast(bf16x8, out);
}
__device__ __forceinline__ float k4_scale(unsigned w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float k4_offset(unsigned w) { return __uint_as_float(w & 0xFFFF0000u); }

// ------------------------------------------------------------------ quantise and append
struct AppendArgs {
    const void* k; const void* v; long k_bs, k_hs, k_ss, v_bs, v_hs, v_ss;
    char* cache; long smax, sm; int B, Hkv, n; int start; const int32_t* starts; const int32_t* counts;
};

// the levels of one group of 32 values (low to high channel), and its scale word
__device__ __forceinline__ unsigned k4_quantise(const float (&x)[32], unsigned char (&level)[32]) {
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int e = 1; e < 32; ++e) { lo = fminf(lo, x[e]); hi = fmaxf(hi, x[e]); }
    const bf16_t off_b = (bf16_t)lo, scale_b = (bf16_t)((hi - lo) * (1.0f / 15.0f));
    const float off = (float)off_b, scale = (float)scale_b;
    const float inv = scale == 0.f ? 0.f : 1.0f / scale;
#pragma unroll
    for (int e = 0; e < 32; ++e) level[e] = (unsigned char)(int)fminf(fmaxf(rintf((x[e] - off) * inv), 0.f), 15.f);
    return (unsigned)__builtin_bit_cast(unsigned short, scale_b) | ((unsigned)__builtin_bit_cast(unsigned short, off_b) << 16);
}

// One workgroup: the 32 keys of one block of one (sequence, head).  A thread quantises one group of one row; K's words are
// its own to write, V's levels meet in LDS and leave as words of eight keys, with the levels that were there kept where the
// new rows cover a word only in part.  Bound by reading the rows (the quarter of that written comes on top).
template <typename T, int HD>
__global__ __launch_bounds__(256) void kv4_append_kernel(AppendArgs p) {
    using G = K4<HD>;
    __shared__ __attribute__((aligned(16))) unsigned char lev[32][HD + 4];
    const int bh = blockIdx.x, b = bh / p.Hkv, h = bh - b * p.Hkv, tid = threadIdx.x;
    const long start = p.starts ? p.starts[b] : p.start;
    const int cnt = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
    const long s0 = start > 0 ? start : 0;                                   // rows that fall outside 0..smax-1 are dropped
    const long s1 = start + cnt < p.smax ? start + cnt : p.smax;
    if (s1 <= s0) return;
    const long block = s0 / 32 + blockIdx.y;
    if (block * 32 >= s1) return;
    const int r0 = (int)(s0 > block * 32 ? s0 - block * 32 : 0), r1 = (int)(s1 - block * 32 < 32 ? s1 - block * 32 : 32);    // new rows of the block
    char* piece = p.cache + bh * k4_piece(p.sm, HD);
    for (int task = tid; task < 2 * 32 * G::NG; task += 256) {
        const int which = task / (32 * G::NG), row = (task / G::NG) & 31, t = task % G::NG;
        if (row < r0 || row >= r1) continue;
        const long key = block * 32 + row, src = key - start;
        const T* at = which == 0 ? reinterpret_cast<const T*>(p.k) + (long)b * p.k_bs + (long)h * p.k_hs + src * p.k_ss
                                 : reinterpret_cast<const T*>(p.v) + (long)b * p.v_bs + (long)h * p.v_hs + src * p.v_ss;
        float x[32];
        unsigned char level[32];
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const bf16x8 y = *reinterpret_cast<const bf16x8*>(at + 32 * t + 8 * c);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[8 * c + e] = (float)y[e];
            }
        } else {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const f32x4 y = *reinterpret_cast<const f32x4*>(at + 32 * t + 4 * c);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * c + e] = y[e];
            }
        }
        const unsigned sw = k4_quantise(x, level);
        *reinterpret_cast<unsigned*>(piece + (which == 0 ? k4_ks(p.sm, HD) : k4_vs(p.sm, HD)) + (key * G::NG + t) * 4) = sw;
        if (which == 0) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                unsigned w = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) w |= (unsigned)level[8 * g + 2 * j] << (4 * j) | (unsigned)level[8 * g + 2 * j + 1] << (16 + 4 * j);
                *reinterpret_cast<unsigned*>(piece + k4_k_word<HD>((int)key, t, g)) = w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
                *reinterpret_cast<unsigned*>(&lev[row][32 * t + e]) =
                    (unsigned)level[e] | (unsigned)level[e + 1] << 8 | (unsigned)level[e + 2] << 16 | (unsigned)level[e + 3] << 24;
        }
    }
    __syncthreads();
    char* vw = piece + k4_v(p.sm, HD);
    for (int u = tid; u < 4 * HD; u += 256) {
        const int g = u / HD, ch = u - g * HD, dt = ch >> 4, c = ch & 15;
        unsigned w = 0, mine = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int row = 4 * g + (j & 3) + 16 * (j >> 2);
            if (row >= r0 && row < r1) { w |= (unsigned)lev[row][ch] << (4 * j); mine |= 15u << (4 * j); }
        }
        if (mine == 0) continue;
        unsigned* at = reinterpret_cast<unsigned*>(vw + k4_v_word<HD>((int)block, dt, g, c));
        *at = mine == 0xFFFFFFFFu ? w : (w | (*at & ~mine));
    }
}

// ------------------------------------------------------------------ read rows back
struct UnpackArgs {
    const char* cache; long smax, sm; int B, Hkv, n; int start; const int32_t* starts;
    void* k; void* v; long k_bs, k_hs, k_ss, v_bs, v_hs, v_ss;
};
// One workgroup: the 32 keys of one block of one (sequence, head), as they are appended.  A thread writes eight channels of a row of
// K or V, neighbouring threads neighbouring channels, so that whole lines leave.  Eight channels of K are one word and one scale;
// a word of V holds eight keys of one channel, so the block's words pass through LDS.  Bound by the rows written.
template <typename T, int HD>
__global__ __launch_bounds__(256) void kv4_unpack_kernel(UnpackArgs p) {
    using G = K4<HD>;
    constexpr int CH = HD / 8, J = 2 * 32 * CH / 256;                        // tasks of a row; of a thread
    __shared__ __attribute__((aligned(16))) unsigned vl[4 * HD];
    const int bh = blockIdx.x, b = bh / p.Hkv, h = bh - b * p.Hkv, tid = threadIdx.x;
    const long start = p.starts ? p.starts[b] : p.start;
    const long s0 = start > 0 ? start : 0, s1 = start + p.n < p.smax ? start + p.n : p.smax;       // rows outside 0..smax-1 are left as they are
    const char* piece = p.cache + bh * k4_piece(p.sm, HD);
    for (long block = s0 / 32 + blockIdx.y; block * 32 < s1; block += gridDim.y) {
        unsigned word[J], scale[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int task = tid + 256 * j, which = task / (32 * CH), row = (task / CH) & 31, ch = task % CH;
            const int key = (int)block * 32 + row;                           // (inside the piece, which is whole blocks)
            scale[j] = *reinterpret_cast<const unsigned*>(piece + (which == 0 ? k4_ks(p.sm, HD) : k4_vs(p.sm, HD)) + ((long)key * G::NG + (ch >> 2)) * 4);
            word[j] = which == 0 ? *reinterpret_cast<const unsigned*>(piece + k4_k_word<HD>(key, ch >> 2, ch & 3)) : 0u;
        }
        if (tid < HD) *reinterpret_cast<u32x4*>(vl + 4 * tid) = *reinterpret_cast<const u32x4*>(piece + k4_v(p.sm, HD) + block * (16 * HD) + 16 * tid);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int task = tid + 256 * j, which = task / (32 * CH), row = (task / CH) & 31, ch = task % CH;
            const long key = block * 32 + row, src = key - start;
            T* const base = reinterpret_cast<T*>(which == 0 ? p.k : p.v);
            if (key < s0 || key >= s1 || !base) continue;
            struct __attribute__((aligned(16))) Eight { T x[8]; } out;
            const int shift = 4 * ((row & 3) + 4 * (row >> 4)), dt = ch >> 1;
            const unsigned* vw = vl + ((dt / G::DW) * 64 + ((row & 15) >> 2) * 16 + 8 * (ch & 1)) * G::DW + dt % G::DW;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const unsigned level = which == 0 ? (word[j] >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15u : (vw[e * G::DW] >> shift) & 15u;
                out.x[e] = from_f32<T>(fmaf(k4_scale(scale[j]), (float)level, k4_offset(scale[j])));
            }
            const long at = which == 0 ? (long)b * p.k_bs + (long)h * p.k_hs + src * p.k_ss : (long)b * p.v_bs + (long)h * p.v_hs + src * p.v_ss;
            *reinterpret_cast<Eight*>(base + at + 8 * ch) = out;
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------ attention
struct Dec4Args {
    const void* q; const char* cache; void* o;
    int B, H, Hkv, G, nhg; long sm; int len; const int32_t* lens; int window, prefix;
    int nsplit; float* part_o; float* part_ml;
};

// x as NP bf16 numbers that add up to it (NP = 3: all 24 bits)
template <int NP> __device__ __forceinline__ void split_bf16(float x, bf16_t (&part)[NP]) {
#pragma unroll
    for (int i = 0; i < NP; ++i) { part[i] = (bf16_t)x; x -= (float)part[i]; }
}

// Head hh of the group (of at most 16) is row 4 (hh & 3) + (hh >> 2) of the products, i.e. rows 4 g + i of lane group g are
// heads g + 4 i: up to four heads use one accumulator row per lane (NI = 1), up to eight two, else four.
template <typename T, int HD, int NI>
__global__ __launch_bounds__(256, 2) void kv4_decode_kernel(Dec4Args p) {
    using G = K4<HD>;
    constexpr bool WIDE = sizeof(T) == 4;                                    // (f32: centred levels, three parts)
    constexpr int NP = WIDE ? 3 : 1;
    constexpr float UNIT = WIDE ? 1.f : 16.f;                                // q' and r per q and p scale
    constexpr int PP = 80;                                                   // bytes per row of P in LDS: 32 bf16 and a pad against bank conflicts
    constexpr int PW = NP * G::NG * 16 * PP;                                 // per wave
    constexpr int PJ = HD + 4;
    constexpr int JB = 4 * (4 * NI) * (PJ + 2) * 4;
    __shared__ __attribute__((aligned(16))) char smem[4 * PW > JB ? 4 * PW : JB];
    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int split = blockIdx.x % p.nsplit, rest = blockIdx.x / p.nsplit;
    const int hg = rest % p.nhg, bh = rest / p.nhg;
    const int b = bh / p.Hkv, hkv = bh - b * p.Hkv;
    const int h0 = hkv * p.G + hg * 16, nh = min(16, p.G - hg * 16);
    const int n = p.lens ? min(max(p.lens[b], 0), p.len) : p.len;
    // visible keys of position n - 1: j < a or lo <= j < n; blocks of 32: 0..ns-1, then ws..
    const int lo = max(0, n - p.window), a = min(p.prefix, n);
    const int ns = (a + 31) >> 5, ws = max(ns, lo >> 5), nt = ns + max(0, ((n + 31) >> 5) - ws);
    const int each = nt / p.nsplit, more = nt - each * p.nsplit;                // (the first "more" splits have one block more)
    const int t_begin = split * each + min(split, more), t_end = t_begin + each + (split < more ? 1 : 0);
    const char* piece = p.cache + bh * k4_piece(p.sm, HD);
    const char* kw = piece + (long)lane * (G::NG * 4);
    const char* vw = piece + k4_v(p.sm, HD) + (long)lane * (G::DW * 4);
    const char* ks = piece + k4_ks(p.sm, HD) + (long)l16 * (G::NG * 4);
    const char* vs = piece + k4_vs(p.sm, HD) + (long)l16 * (G::NG * 4);

    struct Block { unsigned k[2][G::NG], v[G::NL][G::DW], ks[2][G::NG], vs[2][G::NG]; };
    auto fetch = [&](Block& x, int idx) {
        const long blk = idx < ns ? idx : ws + idx - ns;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            load_words<G::NG>(x.k[i], kw + (blk * 2 + i) * (64 * G::NG * 4));
            load_words<G::NG>(x.ks[i], ks + (blk * 32 + i * 16) * (G::NG * 4));
            load_words<G::NG>(x.vs[i], vs + (blk * 32 + i * 16) * (G::NG * 4));
        }
#pragma unroll
        for (int i = 0; i < G::NL; ++i) load_words<G::DW>(x.v[i], vw + (blk * G::NL + i) * (64 * G::DW * 4));
    };
    Block cur, nxt;
    int idx = t_begin + wave;
    if (idx < t_end) fetch(cur, idx);

    // q' of row l16, channels 32 t + 8 g + e, and its sums over each group for rows 4 g + i
    bf16x8 qf[NP][G::NG];
    float qsum[NI][G::NG];
    {
        const int hh = (l16 >> 2) + 4 * (l16 & 3);
        const T* row = reinterpret_cast<const T*>(p.q) + ((long)b * p.H + h0 + min(hh, nh - 1)) * HD + 8 * g;
        struct __attribute__((aligned(16))) Eight { T x[8]; } q8[G::NG];
#pragma unroll
        for (int t = 0; t < G::NG; ++t) q8[t] = *reinterpret_cast<const Eight*>(row + 32 * t);          // (rows past the group repeat its last)
        const float on = hh < nh ? UNIT : 0.f;
#pragma unroll
        for (int t = 0; t < G::NG; ++t) {
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = on * to_f32<T>(q8[t].x[e]);
                bf16_t part[NP];
                split_bf16<NP>(x, part);
#pragma unroll
                for (int c = 0; c < NP; ++c) qf[c][t][e] = part[c];
                sum += x;
            }
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
#pragma unroll
            for (int i = 0; i < NI; ++i) qsum[i][t] = __shfl(sum, 4 * g + i, 64);
        }
    }
    f32x4 acc[G::DT];
    float corr[NI][G::NG], m[NI], l[NI];
#pragma unroll
    for (int d = 0; d < G::DT; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int t = 0; t < G::NG; ++t) corr[i][t] = 0.f;
    }
    char* pl = smem + wave * PW;

    for (; idx < t_end; idx += 4) {
        if (idx + 4 < t_end) fetch(nxt, idx + 4);
        const int key0 = (idx < ns ? idx : ws + idx - ns) * 32;
        // scores
        float s[2][NI];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int r = 0; r < NI; ++r) s[i][r] = 0.f;
#pragma unroll
            for (int t = 0; t < G::NG; ++t) {
                const bf16x8 kf = WIDE ? k4_centred(cur.k[i][t]) : k4_expand(cur.k[i][t]);
                f32x4 x = {0.f, 0.f, 0.f, 0.f};
                if constexpr (!WIDE) {
#pragma unroll
                    for (int r = 0; r < NI; ++r) x[r] = -qsum[r][t];
                }
#pragma unroll
                for (int c = 0; c < NP; ++c) x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qf[c][t], kf, x, 0, 0, 0);
                const float sc = k4_scale(cur.ks[i][t]), off = WIDE ? fmaf(7.5f, sc, k4_offset(cur.ks[i][t])) : k4_offset(cur.ks[i][t]) * 0.0625f;
#pragma unroll
                for (int r = 0; r < NI; ++r) s[i][r] += fmaf(sc, x[r], off * qsum[r][t]);
            }
        }
        const bool whole = key0 + 32 <= a || (key0 >= lo && key0 + 32 <= n);
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int key = key0 + 16 * i + l16;
                const bool see = (key < a) | ((key >= lo) & (key < n));
#pragma unroll
                for (int r = 0; r < NI; ++r) s[i][r] = see ? s[i][r] : -INFINITY;
#pragma unroll
                for (int t = 0; t < G::NG; ++t) cur.vs[i][t] = see ? cur.vs[i][t] : 0u;          // (a row never written may hold anything)
            }
        }
        // the reference moves when some score has passed it by more than 8 / log2(e)
        bool up = false;
#pragma unroll
        for (int r = 0; r < NI; ++r) up |= fmaxf(s[0][r], s[1][r]) > m[r] + 8.f / LOG2E;
        if (__any(up)) {
#pragma unroll
            for (int r = 0; r < NI; ++r) {
                const float mn = fmaxf(m[r], max16(fmaxf(s[0][r], s[1][r])));
                const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[r] - mn) * LOG2E);
                m[r] = mn;
                l[r] *= alpha;
#pragma unroll
                for (int t = 0; t < G::NG; ++t) corr[r][t] *= alpha;
#pragma unroll
                for (int d = 0; d < G::DT; ++d) acc[d][r] *= alpha;
            }
        }
        // probabilities, times each group's scale, as the operand of the second product
#pragma unroll
        for (int r = 0; r < NI; ++r) {
            const float mu = m[r] == -INFINITY ? 0.f : m[r];
            float pr[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                pr[i] = __builtin_amdgcn_exp2f((s[i][r] - mu) * LOG2E);
                l[r] += pr[i];
            }
#pragma unroll
            for (int t = 0; t < G::NG; ++t) {
                bf16_t part[2][NP];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float sc = k4_scale(cur.vs[i][t]);
                    split_bf16<NP>(UNIT * pr[i] * sc, part[i]);
                    corr[r][t] = fmaf(pr[i], fmaf(7.5f, sc, k4_offset(cur.vs[i][t])), corr[r][t]);
                    if constexpr (!WIDE) corr[r][t] = fmaf(-1.46875f, (float)part[i][0], corr[r][t]);
                }
#pragma unroll
                for (int c = 0; c < NP; ++c) {
                    const unsigned two = (unsigned)__builtin_bit_cast(unsigned short, part[0][c]) | (unsigned)__builtin_bit_cast(unsigned short, part[1][c]) << 16;
                    *reinterpret_cast<unsigned*>(pl + ((c * G::NG + t) * 16 + 4 * g + r) * PP + l16 * 4) = two;
                }
            }
        }
        // (LDS operations of one wave complete in order; the fence keeps the compiler from moving the reads up)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int t = 0; t < G::NG; ++t) {
            const unsigned w0 = cur.v[(2 * t) / G::DW][(2 * t) % G::DW], w1 = cur.v[(2 * t + 1) / G::DW][(2 * t + 1) % G::DW];
            const bf16x8 v0 = WIDE ? k4_centred(w0) : k4_expand(w0), v1 = WIDE ? k4_centred(w1) : k4_expand(w1);
#pragma unroll
            for (int c = 0; c < NP; ++c) {
                const bf16x8 pf = *reinterpret_cast<const bf16x8*>(pl + ((c * G::NG + t) * 16 + l16) * PP + 16 * g);
                acc[2 * t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf, v0, acc[2 * t], 0, 0, 0);
                acc[2 * t + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf, v1, acc[2 * t + 1], 0, 0, 0);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        cur = nxt;
    }
    // join the four waves: [wave][head][HD + 4] f32, then [wave][head][m, l]
    __syncthreads();
    float* jo = reinterpret_cast<float*>(smem);
    float* jm = jo + 4 * (4 * NI) * PJ;
#pragma unroll
    for (int r = 0; r < NI; ++r) {
        const int hh = g + 4 * r;
        l[r] = sum16(l[r]);
#pragma unroll
        for (int t = 0; t < G::NG; ++t) corr[r][t] = sum16(corr[r][t]);
#pragma unroll
        for (int d = 0; d < G::DT; ++d) jo[(wave * 4 * NI + hh) * PJ + 16 * d + l16] = acc[d][r] + corr[r][d >> 1];
        if (l16 == 0) { jm[(wave * 4 * NI + hh) * 2] = m[r]; jm[(wave * 4 * NI + hh) * 2 + 1] = l[r]; }
    }
    __syncthreads();
    for (int u = tid; u < nh * (HD / 4); u += 256) {
        const int hh = u / (HD / 4), c = (u - hh * (HD / 4)) * 4;
        float mm = -INFINITY, ll = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, jm[(w * 4 * NI + hh) * 2]);
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float mw = jm[(w * 4 * NI + hh) * 2];
            const float f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mw - mm) * LOG2E);
            ll += f * jm[(w * 4 * NI + hh) * 2 + 1];
            v += f * *reinterpret_cast<const f32x4*>(jo + (w * 4 * NI + hh) * PJ + c);
        }
        const long row = (long)b * p.H + h0 + hh;
        if (p.nsplit > 1) {
            const long at = (long)split * p.B * p.H + row;
            *reinterpret_cast<f32x4*>(p.part_o + at * HD + c) = v;
            if (c == 0) { p.part_ml[2 * at] = mm; p.part_ml[2 * at + 1] = ll; }
        } else {
            const float inv = ll != 0.f ? 1.f / ll : 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) reinterpret_cast<T*>(p.o)[row * HD + c + e] = from_f32<T>(v[e] * inv);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void kv4_join_kernel(T* o, const float* part_o, const float* part_ml, long rows, int hd, int nsplit) {
    join_parts<T>(part_o, part_ml, rows, blockIdx.x, hd, nsplit, o + (long)blockIdx.x * hd, nullptr);
}

int dec4_splits(int B, int H, int Hkv, int smax, int window, int prefix) {
    const int G = H / Hkv;
    const long wgs = (long)B * Hkv * ((G + 15) / 16);
    const long w = window == 0 || window > smax ? smax : window, seen = w + prefix < smax ? w + prefix : smax;
    // Four workgroups per CU, none with fewer than four blocks for each wave.  Measured (us), not cut | aimed at 512 | 1024 | 2048
    // workgroups, then 1024 of at least two | eight blocks a wave:
    //   8 x 4096 rows, 32 heads on 8 of 128:  33 | 15.6 | 15.4 | 15.4,  17.1 | 15.7      1 x 4096: 32 | 10.7 | 10.7 | 10.7,  9.5 | 14.4
    //   1 x 32768:                           234 | 18.2 | 17.9 | 17.7,  21.8 | 16.5      4 x 131072: 933 | 125 | 137 | 129,  136 | 136
    //   32 x 1024, 8 heads of 96:            9.5 | 12.1 | 12.0 | 12.1,  12.3 | 9.4
    long ns = (1024 + wgs - 1) / wgs;
    const long most = (seen / 32 + 2) / 16;
    if (ns > most) ns = most;
    if (ns > 1024) ns = 1024;
    return (int)(ns < 1 ? 1 : ns);
}

template <typename T, int HD> int dec4_launch(const Dec4Args& a, hipStream_t st) {
    const long grid = (long)a.B * a.Hkv * a.nhg * a.nsplit;
    CAPDEC_CHECK(grid < (1L << 31), "attn_decode_kv4: grid too large");
    const int gw = a.G < 16 ? a.G : 16;
    if (gw <= 4) hipLaunchKernelGGL((kv4_decode_kernel<T, HD, 1>), dim3((unsigned)grid), dim3(256), 0, st, a);
    else if (gw <= 8) hipLaunchKernelGGL((kv4_decode_kernel<T, HD, 2>), dim3((unsigned)grid), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv4_decode_kernel<T, HD, 4>), dim3((unsigned)grid), dim3(256), 0, st, a);
    CAPDEC_LAUNCH_CHECK();
    if (a.nsplit > 1) {
        const long rows = (long)a.B * a.H;
        hipLaunchKernelGGL((kv4_join_kernel<T>), dim3((unsigned)rows), dim3(256), 0, st, (T*)a.o, a.part_o, a.part_ml, rows, HD, a.nsplit);
        CAPDEC_LAUNCH_CHECK();
    }
    return CAPDEC_OK;
}
template <typename T> int dec4_type(const Dec4Args& a, int hd, hipStream_t st) {
    switch (hd) {
        case 32: return dec4_launch<T, 32>(a, st);
        case 64: return dec4_launch<T, 64>(a, st);
        case 96: return dec4_launch<T, 96>(a, st);
        default: return dec4_launch<T, 128>(a, st);
    }
}

bool k4_hd(int hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128; }
int k4_check(const void* cache, int B, int Hkv, int smax, int hd, const char* what) {
    CAPDEC_CHECK(cache != nullptr && aligned16(cache), "%s: the cache must be given, 16-byte aligned", what);
    CAPDEC_CHECK(B > 0 && Hkv > 0 && (long)B * Hkv < (1L << 31) && smax > 0 && smax < (1 << 28), "%s: B %d, Hkv %d, smax %d", what, B, Hkv, smax);
    CAPDEC_CHECK(k4_hd(hd), "%s: head dim %d (32, 64, 96 or 128)", what, hd);
    return CAPDEC_OK;
}

}  // namespace

extern "C" long capdec_kv4_head_bytes(int smax, int hd) {
    if (smax <= 0 || !k4_hd(hd)) return 0;
    return k4_piece((smax + 31L) / 32 * 32, hd);
}

extern "C" int capdec_kv4_append(const capdec_kv4_rows* r, void* cache, int B, int Hkv, int smax, int hd, int start, const int32_t* starts,
                                 const int32_t* counts, void* stream) {
    int rc = k4_check(cache, B, Hkv, smax, hd, "kv4_append");
    if (rc != CAPDEC_OK) return rc;
    CAPDEC_CHECK(r && r->k && r->v && r->n > 0, "kv4_append: no rows");
    CAPDEC_CHECK(r->dtype == CAPDEC_BF16 || r->dtype == CAPDEC_F32, "kv4_append: bad dtype");
    CAPDEC_CHECK(starts || (start >= 0 && (long)start + r->n <= smax), "kv4_append: rows %d..%ld outside a cache of %d", start, (long)start + r->n, smax);
    const int per16 = r->dtype == CAPDEC_BF16 ? 8 : 4;
    const long strides[] = {r->k_bs, r->k_hs, r->k_ss, r->v_bs, r->v_hs, r->v_ss};
    for (long s : strides) CAPDEC_CHECK(s >= 0 && s % per16 == 0, "kv4_append: stride %ld (must be a non-negative multiple of %d elements)", s, per16);
    CAPDEC_CHECK(aligned16(r->k) && aligned16(r->v), "kv4_append: rows must be 16-byte aligned");
    AppendArgs a = {r->k, r->v, r->k_bs, r->k_hs, r->k_ss, r->v_bs, r->v_hs, r->v_ss, (char*)cache, smax, (smax + 31L) / 32 * 32, B, Hkv, r->n, start, starts, counts};
    // blocks a sequence's rows can touch: wherever they start, one more than they fill
    const long blocks = starts ? (r->n + 30L) / 32 + 1 : ((long)start + r->n - 1) / 32 - start / 32 + 1;
    CAPDEC_CHECK(blocks < 65536, "kv4_append: %d rows at once", r->n);
    const dim3 grid((unsigned)(B * Hkv), (unsigned)blocks);
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto kfn) { hipLaunchKernelGGL(kfn, grid, dim3(256), 0, st, a); };
    if (r->dtype == CAPDEC_BF16) {
        if (hd == 32) go(kv4_append_kernel<bf16_t, 32>); else if (hd == 64) go(kv4_append_kernel<bf16_t, 64>);
        else if (hd == 96) go(kv4_append_kernel<bf16_t, 96>); else go(kv4_append_kernel<bf16_t, 128>);
    } else {
        if (hd == 32) go(kv4_append_kernel<float, 32>); else if (hd == 64) go(kv4_append_kernel<float, 64>);
        else if (hd == 96) go(kv4_append_kernel<float, 96>); else go(kv4_append_kernel<float, 128>);
    }
    CAPDEC_LAUNCH_CHECK();
    return CAPDEC_OK;
}

extern "C" int capdec_kv4_unpack(const void* cache, const capdec_kv4_rows* r, int B, int Hkv, int smax, int hd, int start, const int32_t* starts, void* stream) {
    int rc = k4_check(cache, B, Hkv, smax, hd, "kv4_unpack");
    if (rc != CAPDEC_OK) return rc;
    CAPDEC_CHECK(r && (r->k || r->v) && r->n > 0, "kv4_unpack: no rows");
    CAPDEC_CHECK(r->dtype == CAPDEC_BF16 || r->dtype == CAPDEC_F32, "kv4_unpack: bad dtype");
    CAPDEC_CHECK(starts || (start >= 0 && (long)start + r->n <= smax), "kv4_unpack: rows %d..%ld outside a cache of %d", start, (long)start + r->n, smax);
    UnpackArgs a = {(const char*)cache, smax, (smax + 31L) / 32 * 32, B, Hkv, r->n, start, starts, (void*)r->k, (void*)r->v,
                    r->k_bs, r->k_hs, r->k_ss, r->v_bs, r->v_hs, r->v_ss};
    const int per16 = r->dtype == CAPDEC_BF16 ? 8 : 4;
    const long strides[] = {r->k_bs, r->k_hs, r->k_ss, r->v_bs, r->v_hs, r->v_ss};
    for (long s : strides) CAPDEC_CHECK(s >= 0 && s % per16 == 0, "kv4_unpack: stride %ld (must be a non-negative multiple of %d elements)", s, per16);
    CAPDEC_CHECK(aligned16(r->k) && aligned16(r->v), "kv4_unpack: rows must be 16-byte aligned");
    const long blocks = starts ? (r->n + 30L) / 32 + 1 : ((long)start + r->n - 1) / 32 - start / 32 + 1;
    const dim3 grid((unsigned)(B * Hkv), (unsigned)(blocks < 4096 ? blocks : 4096));
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto kfn) { hipLaunchKernelGGL(kfn, grid, dim3(256), 0, st, a); };
    if (r->dtype == CAPDEC_BF16) {
        if (hd == 32) go(kv4_unpack_kernel<bf16_t, 32>); else if (hd == 64) go(kv4_unpack_kernel<bf16_t, 64>);
        else if (hd == 96) go(kv4_unpack_kernel<bf16_t, 96>); else go(kv4_unpack_kernel<bf16_t, 128>);
    } else {
        if (hd == 32) go(kv4_unpack_kernel<float, 32>); else if (hd == 64) go(kv4_unpack_kernel<float, 64>);
        else if (hd == 96) go(kv4_unpack_kernel<float, 96>); else go(kv4_unpack_kernel<float, 128>);
    }
    CAPDEC_LAUNCH_CHECK();
    return CAPDEC_OK;
}

extern "C" long capdec_attn_decode_kv4_workspace(int B, int H, int Hkv, int hd, int smax, int window, int prefix_len) {
    if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || smax <= 0 || !k4_hd(hd) || window < 0 || prefix_len < 0) return 0;
    const int ns = dec4_splits(B, H, Hkv, smax, window, prefix_len);
    return ns > 1 ? (long)ns * B * H * (hd + 2) * 4 : 0;
}

extern "C" int capdec_attn_decode_kv4(const void* q, const void* cache, void* o, int dtype, int B, int H, int Hkv, int hd, int smax, int len,
                                      const int32_t* lens, int window, int prefix_len, void* workspace, long workspace_bytes, void* stream) {
    int rc = k4_check(cache, B, Hkv, smax, hd, "attn_decode_kv4");
    if (rc != CAPDEC_OK) return rc;
    CAPDEC_CHECK(q && o && aligned16(q) && aligned16(o), "attn_decode_kv4: q and o must be given, 16-byte aligned");
    CAPDEC_CHECK(dtype == CAPDEC_BF16 || dtype == CAPDEC_F32, "attn_decode_kv4: bad dtype");
    CAPDEC_CHECK(H > 0 && H % Hkv == 0, "attn_decode_kv4: H %d, Hkv %d (Hkv must divide H)", H, Hkv);
    CAPDEC_CHECK(len > 0 && len <= smax, "attn_decode_kv4: length %d outside 1..%d", len, smax);
    CAPDEC_CHECK(window >= 0 && prefix_len >= 0, "attn_decode_kv4: window %d, prefix %d", window, prefix_len);
    Dec4Args a;
    memset(&a, 0, sizeof(a));
    a.q = q; a.cache = (const char*)cache; a.o = o;
    a.B = B; a.H = H; a.Hkv = Hkv; a.G = H / Hkv; a.nhg = (a.G + 15) / 16;
    a.sm = (smax + 31L) / 32 * 32;
    a.len = len; a.lens = lens;
    a.window = window == 0 ? 1 << 30 : window;
    a.prefix = prefix_len;
    a.nsplit = 1;
    const int ns = dec4_splits(B, H, Hkv, len, window, prefix_len);
    if (ns > 1 && workspace) {
        const long need = (long)ns * B * H * (hd + 2) * 4;
        if (workspace_bytes < need) {
            capdec_set_error("attn_decode_kv4: workspace %ld bytes < %ld", workspace_bytes, need);
            return CAPDEC_ERR_WORKSPACE;
        }
        CAPDEC_CHECK(aligned16(workspace), "attn_decode_kv4: workspace must be 16-byte aligned");
        a.nsplit = ns;
        a.part_o = (float*)workspace;
        a.part_ml = a.part_o + (long)ns * B * H * hd;
    }
    return dtype == CAPDEC_BF16 ? dec4_type<bf16_t>(a, hd, (hipStream_t)stream) : dec4_type<float>(a, hd, (hipStream_t)stream);
}

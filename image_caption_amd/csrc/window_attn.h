// Attention under a sliding window with first keys that stay visible: what its forward (window_fwd.hip) and backward
// (window_bwd.hip) share -- the visibility rule, the row packing and the two matrix-core forms everything is made of.
//
// Rows.  The G = H / Hkv query heads that share a K/V head are packed into one row axis: row r = i * G + g is query i of
// head hkv * G + g.  A tile of 32 (or 4 x 32) consecutive rows then shares every K/V tile it reads, one token with G heads
// is the same case as G tokens with one head, and the gradients of a shared head are summed where they are formed.
//
// Visibility.  Key j of a query at position i in a sequence of n rows: two intervals of j,
//     j < a  or  lo <= j < hi,   hi = min(i + 1, n), lo = i - window + 1, a = min(prefix, open ? n : hi),
// all empty when i >= n.  Only key tiles that meet one of them are visited, and only tiles that are not wholly inside one
// of them for every row pay for element masks.
//
// Matrix-core forms (32x32 accumulators: lane l holds column l & 31, rows 8 (e >> 2) + 4 (l >> 5) + (e & 3), e = 0..15):
//   mma_rows  acc[x][y] += sum_d  L[x][d] f[y][d]    L: 32 rows in LDS, f: one row per lane in registers
//   mma_cols  acc[d][y] += sum_x  L[x][d] p[x][y]    p: an accumulator of the first kind, used as it lies: the reduction
//             index of this product may run in any order as long as both operands agree, and the order in which a lane
//             holds x is such an order -- the transposing LDS read (bf16) or a strided one (f32) follows it.
// So scores, probabilities and their gradients never leave the registers.
#pragma once
#include "common.h"

typedef __attribute__((ext_vector_type(16))) float f32x16;

struct WinArgs {
    const void* q; const void* k; const void* v; void* o;
    long q_bs, q_hs, q_ss, k_bs, k_hs, k_ss, v_bs, v_hs, v_ss, o_bs, o_hs, o_ss;
    int B, H, Hkv, G, S, nq, q_start, last;      // last: the one query of sequence b sits at its last position, lens[b] - 1
    unsigned g_magic;                            // floor(2^32 / G) + 1
    int rows;                                    // nq * G
    int window, prefix, open;                    // window: 1 << 30 for "no limit"
    const int32_t* lens;
    uint32_t drop_thr, drop_k0, drop_k1; float drop_scale; int S4;
    float* lse;                                  // [B][H][nq] or null
    int tiles, nsplit; float* part_o; float* part_ml;
    // backward
    const void* dout; long do_bs, do_hs, do_ss;
    void* dq; long dq_bs, dq_hs, dq_ss;
    void* dk; long dk_bs, dk_hs, dk_ss;
    void* dv; long dv_bs, dv_hs, dv_ss;
    float dq_scale; float* delta;
    int ktiles, kp, ncp, ncn; float* part;       // key tiles, those that meet the prefix, chunks of either kind, their partial sums
};

constexpr float WIN_LOG2E = 1.44269504088896340736f;

__device__ __forceinline__ int win_len(const WinArgs& p, int b) { return p.lens ? min(max(p.lens[b], 0), p.S) : p.S; }
__device__ __forceinline__ int win_row_query(const WinArgs& p, int r) { return p.G == 1 ? r : (int)__umulhi((unsigned)r, p.g_magic); }

// the two intervals of visible keys of a query at position pos
struct WinSpan { int a, lo, hi; };
__device__ __forceinline__ WinSpan win_span(const WinArgs& p, int pos, int n) {
    WinSpan s;
    const bool live = pos < n;
    s.hi = live ? min(pos + 1, n) : 0;
    s.lo = max(0, pos - p.window + 1);
    s.a = live ? min(p.prefix, p.open ? n : s.hi) : 0;
    return s;
}
// the keys that some query at pos0..pos1 sees: what lies outside may be anything, and is zero before it meets a probability of 0
__device__ __forceinline__ WinSpan win_union(const WinArgs& p, int pos0, int pos1, int n) {
    WinSpan s;
    const bool live = pos0 < n;
    s.hi = live ? min(pos1 + 1, n) : 0;
    s.lo = max(0, pos0 - p.window + 1);
    s.a = live ? min(p.prefix, p.open ? n : s.hi) : 0;
    return s;
}
// How many of the first packed rows see one key alone: that key's probability is 1 whatever its score, so the score has no gradient,
// which dP - delta, two sums of the same numbers in different orders, would only come near.  (A query past the first position
// sees its own key and another one unless window 1 stands alone; an open prefix of two shows them to all.)
__device__ __forceinline__ int win_single_rows(const WinArgs& p, int n) {
    return p.window == 1 && p.prefix == 0 ? p.rows : p.q_start > 0 || (p.open && min(p.prefix, n) > 1) ? 0 : p.G;
}
// (bitwise, and used in selects only: a branch per element costs more, and a conditional store into a vector's element has
// come out of the compiler without the store)
__device__ __forceinline__ bool win_sees(const WinSpan& s, int key) { return (key < s.a) | ((key >= s.lo) & (key < s.hi)); }

// workgroups b, b + 8, ... share an XCD: each XCD takes a contiguous run of logical ids, so neighbours in the grid (tiles that
// read the same keys) share an L2
__device__ __forceinline__ int win_xcd_id(int w, int n) {
    const int per = n >> 3, rem = n & 7, xcd = w & 7;
    return (xcd < rem ? xcd * (per + 1) : rem * (per + 1) + (xcd - rem) * per) + (w >> 3);
}

// Rows in LDS: PB bytes each, no padding, their 16-byte chunks permuted by the row so that neither kind of read meets itself in
// one of the 64 banks: mma_rows reads one chunk of 16 consecutive rows at a time (16 lanes of 16 bytes a cycle), mma_cols four
// chunks of four rows (32 lanes of 8 bytes).  Rows of whole 256, of 128 or of 64 bytes leave groups of GROUP = 16, 8 or 4
// chunks whose banks come again with the next, the second, the fourth row: a chunk's place in its group is XORed with the
// row's low four bits reversed, cut to the group.  Sixteen rows then differ in a chunk's place, and four consecutive ones in its
// upper bits, i.e. in which four chunks.  (Permuted for 32 banks both kinds of read took twice their cycles, 8 and 4: 3 % of the
// captioning stack's backward, nothing of the prompt's forward -- LDS latency counts there, not its bandwidth.)
template <typename T, int HD> struct WinGeo {
    static constexpr int PB = HD * (int)sizeof(T);
    static constexpr int CPR = PB / 16;                          // 16-byte chunks per row
    static constexpr int DT = HD / 32;
    static constexpr int GROUP = PB % 256 == 0 ? 16 : PB % 128 == 0 ? 8 : 4;
    static __device__ __forceinline__ int mix(int row) {
        return ((row & 1) << 3 | (row & 2) << 1 | (row & 4) >> 1 | (row & 8) >> 3) & (GROUP - 1);
    }
    static __device__ __forceinline__ int at(int row, int chunk) { return row * PB + ((chunk ^ mix(row)) << 4); }
};

// one row per lane (row = lane & 31; the two halves of the wave hold alternate pieces of it), as mma_rows wants it
template <typename T, int HD> struct RowFrag;
template <int HD> struct RowFrag<bf16_t, HD> {
    bf16x8 f[HD / 16];
    __device__ __forceinline__ void load(const bf16_t* row, int lane) {
#pragma unroll
        for (int s = 0; s < HD / 16; ++s) f[s] = *reinterpret_cast<const bf16x8*>(row + 16 * s + 8 * (lane >> 5));
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int s = 0; s < HD / 16; ++s) f[s] = __builtin_bit_cast(bf16x8, (u32x4{0, 0, 0, 0}));
    }
    // the loads have landed here: left to itself the compiler may sink them to a loop's first use, where their wait would be
    // a wait for every later load as well, in every pass
    __device__ __forceinline__ void landed() {
#pragma unroll
        for (int s = 0; s < HD / 16; ++s) asm volatile("" : "+v"(f[s]));
    }
    // sum over this lane's half of the row
    __device__ __forceinline__ float dot(const RowFrag& o) const {
        float a = 0.f;
#pragma unroll
        for (int s = 0; s < HD / 16; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) a = fmaf((float)f[s][e], (float)o.f[s][e], a);
        return a;
    }
};
template <int HD> struct RowFrag<float, HD> {
    f32x4 f[HD / 8];
    __device__ __forceinline__ void load(const float* row, int lane) {
#pragma unroll
        for (int s = 0; s < HD / 8; ++s) f[s] = *reinterpret_cast<const f32x4*>(row + 8 * s + 4 * (lane >> 5));
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int s = 0; s < HD / 8; ++s) f[s] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void landed() {
#pragma unroll
        for (int s = 0; s < HD / 8; ++s) asm volatile("" : "+v"(f[s]));
    }
    __device__ __forceinline__ float dot(const RowFrag& o) const {
        float a = 0.f;
#pragma unroll
        for (int s = 0; s < HD / 8; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) a = fmaf(f[s][e], o.f[s][e], a);
        return a;
    }
};

// Where a lane reads in a tile.  row(s): chunk 2 s + (lane >> 5) of row lane & 31, for mma_rows; col(dt): the transposing read of
// mma_cols, four rows 4 (lane >> 5) .. of columns 16 (lane >> 4 & 1) .. + 15 of tile dt, and col8(dt) the same eight rows on.
// XORs of one register each (and one instruction with the tile's address), for sixteen registers that would hold them all.
template <typename T, int HD> struct RowAt {
    using G = WinGeo<T, HD>;
    static constexpr int P = G::GROUP / 2;
    int r0;
    __device__ __forceinline__ RowAt(int lane) : r0(G::at(lane & 31, lane >> 5)) {}
    __device__ __forceinline__ int row(int s) const { return (r0 ^ ((s % P) << 5)) + (s / P) * (32 * P); }
};
// fresh(): the same, of which the compiler may not keep XORs from one tile to the next (it would spill for them)
template <typename T, int HD> struct LaneAt;
template <int HD> struct LaneAt<bf16_t, HD> : RowAt<bf16_t, HD> {
    using G = WinGeo<bf16_t, HD>;
    static constexpr int P = G::GROUP / 4;
    int c0;
    __device__ __forceinline__ LaneAt(int lane) : RowAt<bf16_t, HD>(lane) {
        const int g = lane >> 4, i = lane & 15, row = 4 * (g >> 1) + (i >> 2);
        c0 = G::at(row, 2 * (g & 1) + ((i & 3) >> 1)) + 8 * (i & 1);
    }
    __device__ __forceinline__ LaneAt fresh() const {
        LaneAt x = *this;
        asm volatile("" : "+v"(x.r0), "+v"(x.c0));
        return x;
    }
    __device__ __forceinline__ int col(int dt) const { return (c0 ^ ((dt % P) << 6)) + (dt / P) * (64 * P); }
    __device__ __forceinline__ int col8(int dt) const { return (c0 ^ ((dt % P) << 6 | 16)) + (dt / P) * (64 * P) + 8 * G::PB; }
};
template <int HD> struct LaneAt<float, HD> : RowAt<float, HD> {
    int lane;
    __device__ __forceinline__ LaneAt(int lane_) : RowAt<float, HD>(lane_), lane(lane_) {}
    __device__ __forceinline__ LaneAt fresh() const { return *this; }
};

template <int HD> __device__ __forceinline__ void mma_rows(f32x16& acc, const char* lds, const RowFrag<bf16_t, HD>& b, const LaneAt<bf16_t, HD>& at) {
#pragma unroll
    for (int s = 0; s < HD / 16; ++s)
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(lds + at.row(s)), b.f[s], acc, 0, 0, 0);
}
template <int HD> __device__ __forceinline__ void mma_rows(f32x16& acc, const char* lds, const RowFrag<float, HD>& b, const LaneAt<float, HD>& at) {
#pragma unroll
    for (int s = 0; s < HD / 8; ++s) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(lds + at.row(s));
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b.f[s][e], acc, 0, 0, 0);
    }
}

// the same with the second operand's rows in LDS as well
template <int HD> __device__ __forceinline__ void mma_rows_lds(f32x16& acc, const char* lds, const char* rows, const LaneAt<float, HD>& at) {
#pragma unroll
    for (int s = 0; s < HD / 8; ++s) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(lds + at.row(s)), b = *reinterpret_cast<const f32x4*>(rows + at.row(s));
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], acc, 0, 0, 0);
    }
}

// x + the sum of eight bf16 numbers, in f32
__device__ __forceinline__ float win_sum8(const bf16x8& b, float x) {
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
    const bf16x2 one = {(bf16_t)1.f, (bf16_t)1.f};
    x = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(b, b, 0, 1), one, x, false);
    x = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(b, b, 2, 3), one, x, false);
    x = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(b, b, 4, 5), one, x, false);
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(b, b, 6, 7), one, x, false);
}

// p is rounded to bf16 (half a step, 2^-8 of each term) to be an operand: the products' own inputs have no more bits.
// SUM: sum += this lane's rounded p (half of its row's, the other half lies in lane ^ 32)
template <int HD, bool SUM = false>
__device__ __forceinline__ void mma_cols(f32x16 (&acc)[HD / 32], const char* lds, const f32x16& p, const LaneAt<bf16_t, HD>& at, float* sum = nullptr) {
    constexpr int PB = WinGeo<bf16_t, HD>::PB, DT = HD / 32, A = 3 < 2 * DT ? 3 : 2 * DT;
    bf16x8 a[2 * DT], pb[2];
    auto read = [&](int i) {
        const char* from = lds + 16 * (i / DT) * PB;
        const bf16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, from + at.col(i % DT)));
        const bf16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, from + at.col8(i % DT)));
        a[i] = __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7);
    };
#pragma unroll
    for (int i = 0; i < A; ++i) read(i);
#pragma unroll
    for (int i = 0; i < 2 * DT; ++i) {
        if (i + A < 2 * DT) read(i + A);
        if (i % DT == 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) pb[i / DT][e] = (bf16_t)p[8 * (i / DT) + e];
            if constexpr (SUM) *sum = win_sum8(pb[i / DT], *sum);
        }
        __builtin_amdgcn_sched_barrier(0x6);
        acc[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], pb[i / DT], acc[i % DT], 0, 0, 0);
    }
}
template <int HD> __device__ __forceinline__ void mma_cols(f32x16 (&acc)[HD / 32], const char* lds, const f32x16& p, const LaneAt<float, HD>& at) {
    using G = WinGeo<float, HD>;
    const int h = at.lane >> 5, d = at.lane & 31;
#pragma unroll
    for (int e = 0; e < 16; ++e)
#pragma unroll
        for (int dt = 0; dt < HD / 32; ++dt) {
            const int row = 8 * (e >> 2) + (e & 3);               // + 4 h
            const int off = (row + 4 * h) * G::PB + (((8 * dt + (d >> 2)) ^ G::mix(row) ^ h << 1) << 4) + 4 * (d & 3);
            acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(*reinterpret_cast<const float*>(lds + off), p[e], acc[dt], 0, 0, 0);
        }
}

// Two products of rows one after the other, and columns, with the reads of LDS AH instructions ahead of the matrix instruction
// that takes them
constexpr int AH = 2;
template <int HD>
__device__ __forceinline__ void mma_rows2(f32x16& s, const char* l0, const RowFrag<bf16_t, HD>& b0, f32x16& t, const char* l1, const RowFrag<bf16_t, HD>& b1,
                                          const LaneAt<bf16_t, HD>& at) {
    constexpr int N = HD / 16;
    bf16x8 a[2 * N];
    auto read = [&](int i) { a[i] = *reinterpret_cast<const bf16x8*>((i < N ? l0 : l1) + at.row(i % N)); };
#pragma unroll
    for (int i = 0; i < AH; ++i) read(i);
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
        if (i + AH < 2 * N) read(i + AH);
        __builtin_amdgcn_sched_barrier(0x6);
        if (i < N) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b0.f[i % N], s, 0, 0, 0);
        else t = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b1.f[i % N], t, 0, 0, 0);
    }
}
template <int HD>
__device__ __forceinline__ void mma_rows2(f32x16& s, const char* l0, const RowFrag<float, HD>& b0, f32x16& t, const char* l1, const RowFrag<float, HD>& b1,
                                          const LaneAt<float, HD>& at) {
    mma_rows<HD>(s, l0, b0, at);
    mma_rows<HD>(t, l1, b1, at);
}

// Rows of a strided matrix from row0 on, as a buffer of which rows nrows.. lie past the end: their loads bring zeros and touch no
// memory.  (Stride 0 -- one row for all -- has no such end; what is repeated there is a row that is in use.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t win_rows(const char* base, long row0, int nrows, long ss, int row_bytes) {
    const long bytes = nrows > 0 ? (nrows - 1) * ss + row_bytes : 0;
    return __builtin_amdgcn_make_buffer_rsrc((void*)(base + row0 * ss), 0, (int)(bytes > 0xFFFFFFF0L ? 0xFFFFFFF0u : (unsigned)bytes), 0x00020000);
}

// NROWS rows of two strided matrices on their way to LDS.  Loads by offset from a bounded buffer: the offsets are the same for
// every tile, nothing is masked or zeroed by instructions (plain loads under a row test spent 80 instructions a tile on
// that, and a fifth of the forward's time)
// ANEW: its offsets are made from tile to tile, for kernels that would spill for 2 U of them kept (dQ of few rows at 128 channels, 84 -> 70 us
// at 2 x 8 K/V heads of 8 x 237 rows; the forward is 1 % faster with them kept)
template <typename T, int HD, int NROWS, int NT, bool ANEW = false> struct TilePair {
    static constexpr int CPR = WinGeo<T, HD>::CPR, U = NROWS * CPR / NT;
    static_assert(NROWS * CPR % NT == 0, "a tile is whole rounds of 16-byte loads");
    u32x4 a[U], b[U];
    // tiles of 128 rows are two buffers of 64: offsets inside a buffer stay below 2^31 for rows up to 32 MiB apart
    static constexpr int H = NROWS > 64 ? 2 : 1, UH = U / H, RH = NROWS / H;
    static_assert(NROWS % H == 0 && RH <= 64 && U % H == 0 && RH * CPR % NT == 0, "a half of a tile is whole rounds of loads too");
    __device__ __forceinline__ void fetch(const char* base0, long ss0, const char* base1, long ss1, long row0, int nvalid, int tid) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const __amdgpu_buffer_rsrc_t r0 = win_rows(base0, row0 + h * RH, nvalid - h * RH, ss0, WinGeo<T, HD>::PB),
                                         r1 = win_rows(base1, row0 + h * RH, nvalid - h * RH, ss1, WinGeo<T, HD>::PB);
            if constexpr (ANEW && NT % CPR == 0) {                          // (load j lies NT / CPR rows on)
                unsigned o0 = (unsigned)(tid / CPR) * (unsigned)ss0 + tid % CPR * 16, o1 = (unsigned)(tid / CPR) * (unsigned)ss1 + tid % CPR * 16;
                asm volatile("" : "+v"(o0), "+v"(o1));
#pragma unroll
                for (int j = 0; j < UH; ++j) {
                    a[h * UH + j] = __builtin_amdgcn_raw_buffer_load_b128(r0, o0 + (unsigned)(j * (NT / CPR)) * (unsigned)ss0, 0, 0);
                    b[h * UH + j] = __builtin_amdgcn_raw_buffer_load_b128(r1, o1 + (unsigned)(j * (NT / CPR)) * (unsigned)ss1, 0, 0);
                }
            } else {
#pragma unroll
                for (int j = 0; j < UH; ++j) {
                    const int u = tid + j * NT, row = u / CPR, ch = u - row * CPR;
                    a[h * UH + j] = __builtin_amdgcn_raw_buffer_load_b128(r0, (unsigned)row * (unsigned)ss0 + ch * 16, 0, 0);
                    b[h * UH + j] = __builtin_amdgcn_raw_buffer_load_b128(r1, (unsigned)row * (unsigned)ss1 + ch * 16, 0, 0);
                }
            }
        }
    }
    // rows before0..from1-1 (relative to the tile) put to zero
    __device__ __forceinline__ void drop(int before0, int from1, int tid) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int row = (tid + j * NT) / CPR;
            const u32x4 z = {0, 0, 0, 0};
            const bool out = (row >= before0) & (row < from1);
            a[j] = out ? z : a[j];
            b[j] = out ? z : b[j];
        }
    }
    __device__ __forceinline__ void commit(char* lds0, char* lds1, int tid) const {
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int u = tid + j * NT, row = u / CPR, ch = u - row * CPR;
            *reinterpret_cast<u32x4*>(lds0 + WinGeo<T, HD>::at(row, ch)) = a[j];
            *reinterpret_cast<u32x4*>(lds1 + WinGeo<T, HD>::at(row, ch)) = b[j];
        }
    }
};

// the key tiles (BK keys each) that rows at positions p0..p1 can see: tiles 0..ns-1, then ws.., nt in all
struct WinTiles {
    int ns, ws, nt;
    __device__ __forceinline__ int at(int idx) const { return idx < ns ? idx : ws + idx - ns; }
};
template <int BK> __device__ __forceinline__ WinTiles win_tiles(const WinArgs& p, int p0, int p1, int n) {
    WinTiles t{0, 0, 0};
    if (p0 >= n) return t;
    const int hi = min(p1 + 1, n), lo = max(0, p0 - p.window + 1), a = min(p.prefix, p.open ? n : hi);
    t.ns = (a + BK - 1) / BK;
    t.ws = max(t.ns, lo / BK);
    t.nt = t.ns + max(0, (hi + BK - 1) / BK - t.ws);
    return t;
}

// four consecutive values d0 + 8 jj + 4 h .. of this lane's row from accumulator e = 4 jj .. 4 jj + 3; in bf16 the two halves
// of the wave swap pieces so that a lane stores 16 bytes
template <int HD> __device__ __forceinline__ void store_rows(const f32x16 (&acc)[HD / 32], float scale, float* row, bool ok, int lane) {
    if (!ok) return;
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
        for (int jj = 0; jj < 4; ++jj)
            *reinterpret_cast<f32x4*>(row + 32 * dt + 8 * jj + 4 * (lane >> 5)) =
                f32x4{acc[dt][4 * jj] * scale, acc[dt][4 * jj + 1] * scale, acc[dt][4 * jj + 2] * scale, acc[dt][4 * jj + 3] * scale};
}
__device__ __forceinline__ unsigned win_pack(float a, float b) {
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
    bf16x2 t;
    t[0] = (bf16_t)a; t[1] = (bf16_t)b;
    return __builtin_bit_cast(unsigned, t);
}
template <int HD> __device__ __forceinline__ void store_rows(const f32x16 (&acc)[HD / 32], float scale, bf16_t* row, bool ok, int lane) {
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
        for (int jp = 0; jp < 2; ++jp) {
            const unsigned x0 = win_pack(acc[dt][8 * jp] * scale, acc[dt][8 * jp + 1] * scale), x1 = win_pack(acc[dt][8 * jp + 2] * scale, acc[dt][8 * jp + 3] * scale);
            const unsigned y0 = win_pack(acc[dt][8 * jp + 4] * scale, acc[dt][8 * jp + 5] * scale), y1 = win_pack(acc[dt][8 * jp + 6] * scale, acc[dt][8 * jp + 7] * scale);
            const u32x2 s0 = __builtin_amdgcn_permlane32_swap(x0, y0, false, false);
            const u32x2 s1 = __builtin_amdgcn_permlane32_swap(x1, y1, false, false);
            // lower half: columns 16 jp .. + 7 (its own four and the upper half's four), upper half: 16 jp + 8 ..
            if (ok) *reinterpret_cast<u32x4*>(row + 32 * dt + 16 * jp + 8 * (lane >> 5)) = u32x4{s0[0], s1[0], s0[1], s1[1]};
        }
}

// ------------------------------------------------------------------ host side
// Four waves on the keys of 32 rows instead of on 32 rows each: for few rows, and where tiles of 128 rows would leave CUs idle.
// Measured in us, waves on rows | on keys (hd 64, 229 keys unless said otherwise):
//   forward, bf16, 2048 heads, 1 / 32 / 48 / 64 rows:  27.0 | 22.9   28.0 | 25.9   31.2 | 37.5   31.8 | 38.3     (hd 96: 39.8 | 40.0 at 32, 44.3 | 62.9 at 64)
//   forward, f32, 2048 heads, 1 / 32 / 64 rows:        104 | 63      106 | 70      157 | 123
//   backward, bf16, 2048 heads, 1 / 32 / 64 rows:      75.6 | 70.9   81.6 | 79.0   96.2 | 108.6                  (hd 128, where dQ spills: 179 | 196 at 32)
//   backward, f32, 2048 heads, 1 / 32 / 64 rows:       410 | 371     421 | 398     570 | 593                     (hd 96: 640 | 467 at 32, 773 | 735 at 64)
//   64 rows in bf16, hd 64 (causal), 256 / 320 / 512 / 768 / 2048 heads: 229 keys  8.5 | 8.2  10.2 | 9.8  11.2 | 13.9  14.3 | 17.8  31.7 | 38.1
//     1024 keys  43 | 17  52 | 21  26 | 30  36 | 38  111 | 126;  4096 keys  74 | 49  98 | 76  105 | 134  151 | 170  407 | 433
//     (backward, 1024 keys: 58 | 52  71 | 63  90 | 89  130 | 143  371 | 380)
//   tiles of 128 rows on 16 CUs (2 x 8 heads of 229 rows, hd 96): 9.0 | 7.9, on 64 (1 head, 8192 rows, hd 128): 48.6 | 30.1,
//   on 128: 9.3 | 10.2 and 19.8 | 16.4, on 256: 9.9 | 17.9 and 19.5 | 19.8
// So: up to 32 rows (f32: 64) always; up to 64 while their tiles do not give every CU two workgroups; more while they do not give it one.
inline bool win_few_rows(bool f32, long bh, long rows) {
    return rows <= (f32 ? 64 : 32) || bh * ((rows + 127) / 128) < (rows <= 64 ? 512 : 256);
}
int win_fill(const capdec_attn_window_desc* d, WinArgs& a, const char* what);
struct WinFwdPlan { int kw; int tiles; int nsplit; long part_floats; };   // kw: four waves share the keys of 32 rows (else 4 x 32 rows)
WinFwdPlan win_fwd_plan(bool f32, int B, int H, int Hkv, int S, int nq, int hd, int window, int prefix);
int win_fwd_launch(WinArgs& a, int dtype, int hd, void* workspace, long workspace_bytes, hipStream_t st);

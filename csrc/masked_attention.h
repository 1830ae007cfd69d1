// Shared parts of the masked attention kernels (masked_attention_fwd.hip, masked_attention_bwd.hip).
//
//   x_ij = scale q_i . k_j        y_ij = cap tanh(x_ij / cap)        s_ij = y_ij - slope_h |p_i - j|
//   o_i = sum_j softmax_j(s_ij) v_j over the visible keys  lo_i <= j < hi_i
//
// Every mask the op offers (causal, documents packed into a row, a prefix that is seen both ways,
// padded rows, a cache's valid length) leaves each query ONE interval of visible keys, so the kernels
// know masks only as two integers per query: a tile needs no per-key mask data, whole tiles are
// skipped or taken without a test from the intervals' bounds over 32 queries (qtab), and the dK / dV
// kernel finds the queries that see a block of keys in ktab.
#pragma once
#include "common.h"

#include <type_traits>

namespace mattn {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));   // (a class like uint4 selected by ?: would be selected by address: scratch)
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int QT = 32;    // queries per qtab entry
constexpr int KT = 128;   // keys per ktab entry
constexpr int64_t MAX_GRID = (1 << 24) - 1;   // workgroups of 256 threads: a launch takes less than 2^32 threads

// one argument block for every entry point (ops/masked_attention.py fills the same layout)
struct Args {
    const void *q, *k, *v, *dout;
    void *o, *dq, *dk, *dv;
    float *lse, *delta, *ws;
    uint32_t* rest;      // what the rounding of o left out (e5m2 of Rest::SCALE times it), [B][Tq][H][D] bytes; null: not kept
    const float* slopes;
    const int *lo, *hi, *pos;
    const int4* qtab;    // [B][ceil(Tq / 32)]: lowest lo, highest hi (rows that see something), highest lo, lowest hi (all rows)
    const int2* ktab;    // [B][ceil(Tk / 128)]: first and past-the-last qtab entry that sees a key of the block
    int64_t qs[3], ks[3], vs[3], os[3], dos[3], dqs[3], dks[3], dvs[3];   // strides in elements: batch, token, head
    int B, Tq, Tk, H, Hk, D, dtype, nsplit;
    float scale, cap;
};

// UP: a softmax's weights are rounded times 2^UP; bf16 has fp32's range
struct Bf16 {
    typedef bf16x8 vec;
    static constexpr int UP = 0;
    static constexpr uint32_t INF = 0x7f80, NANBITS = 0x7fc0;
    static __device__ __forceinline__ f32x16 mfma(vec a, vec b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ void mfma_acc(f32x16& c, vec a, vec b) {
        asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack2(a, b); }
    static __device__ __forceinline__ void unpack(uint32_t w, float& a, float& b) {
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xffff0000u);
    }
};
// Weights are at most 1, and fp16 rounds those below 2^-14 to steps of 2^-24: a long row's small weights were off by
// half a step each, all alike where they are equal.  2^12 times the weight leaves its normal range at 2^-26, for
// the price of a constant in the exponent; the factor cancels against the row's sum (forward) or goes with
// the last scale (backward), and room for weights up to 15 is left (a log-sum-exp rounded low).
struct F16 {
    typedef f16x8 vec;
    static constexpr int UP = 12;
    static constexpr uint32_t INF = 0x7c00, NANBITS = 0x7e00;
    static __device__ __forceinline__ f32x16 mfma(vec a, vec b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ void mfma_acc(f32x16& c, vec a, vec b) {
        asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {   // round to nearest even
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const h2 r = {(_Float16)a, (_Float16)b};
        return __builtin_bit_cast(uint32_t, r);
    }
    static __device__ __forceinline__ void unpack(uint32_t w, float& a, float& b) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const h2 r = __builtin_bit_cast(h2, w);
        a = (float)r[0];
        b = (float)r[1];
    }
};

// T::mfma_acc: c += a b with c in accumulation registers (AGPRs), for sums that only products touch: the
// 256 ordinary registers stay free for the scores.  In asm, because the compiler gives a whole kernel's
// products one form.  The wait states in front cover an operand that the vector ALU has just written.
// Nothing but mfma_acc may read such a sum until acc_done has run (a product takes 16 passes at most).
template <int N>
__device__ __forceinline__ void acc_done(f32x16 (&x)[N], f32x16 (&y)[N]) {
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+a"(x[i]), "+a"(y[i]));
    __builtin_amdgcn_sched_barrier(0);
}

template <class T>
__device__ __forceinline__ typename T::vec as_vec(u32x4 u) {
    return __builtin_bit_cast(typename T::vec, u);
}
// registers 8 half .. 8 half + 7 of an accumulator, rounded once to the input type: the operand that
// the next product takes (probabilities in [0, 1]; their sum is taken before the rounding)
template <class T>
__device__ __forceinline__ typename T::vec round8(const f32x16& v, int half) {
    u32x4 u;
    u.x = T::pack(v[8 * half], v[8 * half + 1]);
    u.y = T::pack(v[8 * half + 2], v[8 * half + 3]);
    u.z = T::pack(v[8 * half + 4], v[8 * half + 5]);
    u.w = T::pack(v[8 * half + 6], v[8 * half + 7]);
    return as_vec<T>(u);
}

// One LDS image of a [rows][DP] 16-bit tile serves both readers, ds_read_b128 of a row (lane l takes
// row l & 31) and the transposing ds_read_b64_tr_b16 (a 32-lane half takes 4 rows x 64 B): the 16-B
// chunk c of a row stands at c ^ key(row).  The row read needs 16 rows of a lane group in 16
// different 16-B slots of the 256-B bank line, the transposed one needs 4 neighbouring rows in 4
// different 64-B quarters; with the row's low bits as the chunk's HIGH bits both hold.
template <int DP>
__device__ __forceinline__ int swz_key(int row) {
    if (DP == 64) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);   // two 128-B rows per bank line
    return ((row & 3) << 2) | ((row >> 2) & 3);
}
template <int DP>
__device__ __forceinline__ int chunk_at(int row, int c) {   // element offset of chunk c of a row
    return row * DP + ((c ^ swz_key<DP>(row)) << 3);
}
template <int DP>
__device__ __forceinline__ int elem_at(int row, int col) {
    return row * DP + (((col >> 3) ^ swz_key<DP>(row)) << 3) + (col & 7);
}
__device__ __forceinline__ short4v tr_read(const bf16_t* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(p));
}
// operand of 32 columns x 16 rows, columns on the lanes: rows r .. r + 3 and r + 8 .. r + 11 of the
// lane's half, the order in which an accumulator holds its rows
template <class T>
__device__ __forceinline__ typename T::vec tr_pair(const bf16_t* lo, const bf16_t* hi) {
    const short4v a = tr_read(lo), b = tr_read(hi);
    const short8v c = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(typename T::vec, c);
}
template <class T, int DP>
__device__ __forceinline__ typename T::vec tr_pair(const bf16_t* img, int row, int col) {
    return tr_pair<T>(img + elem_at<DP>(row, col), img + elem_at<DP>(row + 8, col));
}

// f(0), f(1), .. f(N - 1) with compile-time indices
template <int N, int I = 0, class F>
__device__ __forceinline__ void unrolled(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        unrolled<N, I + 1>(f);
    }
}

// The backward pass takes delta_i = dO_i . o_i.  From the rounded o it would carry o's rounding error
// (2^-9 of |o| |dO|) into P (dP - delta), where peaked rows cancel: dQ and dK came out 1.8 times as far
// from the exact ones as their own rounding.  So a forward pass that will be differentiated keeps the
// remainder in 8 bits beside o: e5m2, 3 more bits of o, scaled into that type's range.
template <class T>
struct Rest {
    static constexpr float SCALE = T::INF == 0x7f80 ? 512.f : 4096.f, MAX = 57344.f;
    static __device__ __forceinline__ float clip(float x) { return __builtin_amdgcn_fmed3f(x * SCALE, -MAX, MAX); }
    // of four values and their two packed roundings
    static __device__ __forceinline__ uint32_t of(const float (&v)[4], uint2 r) {
        float a, b, c, d;
        T::unpack(r.x, a, b);
        T::unpack(r.y, c, d);
        int w = __builtin_amdgcn_cvt_pk_bf8_f32(clip(v[0] - a), clip(v[1] - b), 0, false);
        w = __builtin_amdgcn_cvt_pk_bf8_f32(clip(v[2] - c), clip(v[3] - d), w, true);
        return (uint32_t)w;
    }
    static __device__ __forceinline__ void back(uint32_t w, float (&v)[4]) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, true);
        v[0] = lo[0] * (1.f / SCALE);
        v[1] = lo[1] * (1.f / SCALE);
        v[2] = hi[0] * (1.f / SCALE);
        v[3] = hi[1] * (1.f / SCALE);
    }
};

// whether one of 8 values is an infinity or NaN (integer test on the exponent field)
template <class T>
__device__ __forceinline__ bool not_finite8(u32x4 u) {
    auto mag = [](uint32_t w) { return __builtin_bit_cast(ushort2v, w & 0x7fff7fffu); };
    ushort2v m = __builtin_elementwise_max(mag(u.x), mag(u.y));
    m = __builtin_elementwise_max(m, __builtin_elementwise_max(mag(u.z), mag(u.w)));
    return m.x >= T::INF || m.y >= T::INF;
}

// its finite values, zeros for the others
template <class T>
__device__ __forceinline__ u32x4 finite_only(u32x4 u) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t w = u[i];
        if ((w & 0x7fffu) >= T::INF) w &= 0xffff0000u;
        if (((w >> 16) & 0x7fffu) >= T::INF) w &= 0x0000ffffu;
        u[i] = w;
    }
    return u;
}
// The values that finite_only left out of the rows a lane sees: what a product with weights > 0 makes of
// infinities and NaN, as one bit per accumulator element (4 registers, touched hardly ever).
struct NotFinite {
    uint64_t up = 0, down = 0;   // + infinity, - infinity; NaN is both
    // row: where it stands in memory
    template <class T, int NO>
    __device__ __forceinline__ void note(const bf16_t* row, int D, int h, bool see) {
#pragma unroll 1
        for (int c = 0; c < 4 * NO; ++c) {   // (rolled: few registers and little code beside the hot loops)
            const int d = 8 * c + 4 * h;
            const uint2 u = *(const uint2*)(row + (d < D ? d : 0));
            const uint32_t w[2] = {u.x, u.y};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t x = (w[k >> 1] >> (16 * (k & 1))) & 0xffffu;
                const bool bad = see && d < D && (x & 0x7fffu) >= T::INF, inf = (x & 0x7fffu) == T::INF;
                const uint64_t bit = 1ull << (4 * c + k);
                if (bad && !(inf && (x & 0x8000u))) up |= bit;
                if (bad && !(inf && !(x & 0x8000u))) down |= bit;
            }
        }
    }
    __device__ __forceinline__ bool any() const { return (up | down) != 0; }
    // element e (a constant) of the finished sums
    __device__ __forceinline__ float operator()(float v, int e) const {
        const bool u = (up >> e) & 1, d = (down >> e) & 1;
        float nan = __uint_as_float(0x7fc00000u);
        asm volatile("" : "+v"(nan));   // (opaque: these files are compiled as if no value were NaN)
        return u && d ? nan : u ? INFINITY : d ? -INFINITY : v;
    }
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float max3(float a, float b, float c) { return __builtin_fmaxf(a, __builtin_fmaxf(b, c)); }
__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
    return v;
}

// Scores in units of log 2 (the softmax is taken with 2^x).  tanh u = 1 - 2 / (1 + e^(2 u)): exact to
// 2^-22 of 1 from v_exp and v_rcp, so of a capped score to cap x 2^-21 (the op takes cap <= 1000:
// 2^-11, the rounding of an fp16 probability), and it saturates without overflow.
template <bool CAP, bool ALIBI>
struct Score {
    static constexpr bool PLAIN = !CAP && !ALIBI;
    float mul;      // scale log2(e)
    float c2;       // 2 log2(e) scale / cap
    float capl;     // cap log2(e)
    float c1;       // -1 / (2 capl)
    float slope;    // slope log2(e)
    __device__ __forceinline__ void init(float scale, float cap, float sl) {
        mul = scale * LOG2E;
        if (CAP) {
            c2 = 2.f * LOG2E * scale / cap;
            capl = cap * LOG2E;
            c1 = -0.5f / capl;
        }
        slope = ALIBI ? sl * LOG2E : 0.f;
    }
    // 1 / (1 + e^(2 u)), u = x / cap: tanh u = 1 - 2 r, its derivative 4 r (1 - r)
    __device__ __forceinline__ float sat(float dot) const { return __builtin_amdgcn_rcpf(1.f + exp2_fast(dot * c2)); }
    // capped score less its bound, -2 capl / (1 + e^(2 u)): the factor rides in the sum's fma
    __device__ __forceinline__ float below(float dot) const { return __builtin_amdgcn_rcpf(fmaf(exp2_fast(dot * c2), c1, c1)); }
    __device__ __forceinline__ float capped(float r) const { return fmaf(-2.f * capl, r, capl); }
    // dist: the positions' difference, taken in integers (past 2^24 a float does not tell neighbours apart)
    __device__ __forceinline__ float biased(float y, float dist) const {
        return ALIBI ? fmaf(-slope, fabsf(dist), y) : y;
    }
    __device__ __forceinline__ float operator()(float dot, float dist) const {
        return biased(CAP ? capped(sat(dot)) : dot * mul, dist);
    }
};

// Workgroup -> (batch, KV head, query head of the group, block): the blocks of equal index of all heads
// are neighbours (the longest ones first, `flip`), and the dispatcher deals neighbours over the 8 XCDs,
// so with a multiple of 8 (batch, KV head) pairs all work on one pair's keys stays on one XCD's L2.
struct Where {
    int b, hk, h, blk;
};
__device__ __forceinline__ Where place(int L, const Args& a, int nblk, bool flip) {
    const int G = a.H / a.Hk, nkv = a.B * a.Hk, nbh = nkv * G;
    const int x = L % nbh, y = L / nbh;
    int kv, g;
    if ((nkv & 7) == 0) {
        const int j = x >> 3;
        g = j % G;
        kv = (j / G) * 8 + (x & 7);
    } else {
        kv = x / G;
        g = x - kv * G;
    }
    Where w;
    w.b = kv / a.Hk;
    w.hk = kv - w.b * a.Hk;
    w.h = w.hk * G + g;
    w.blk = flip ? nblk - 1 - y : y;
    return w;
}

// the sum of 8 bf16 values and c, in 32 bits
__device__ __forceinline__ float sum8(bf16x8 v, float c) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 one = {(__bf16)1.f, (__bf16)1.f};
    const u32x4 u = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = u[i];
        c = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), one, c, false);
    }
    return c;
}

// Staging of a [ROWS][DP] tile by NTHR threads: thread t takes the 16-B chunk t % (DP / 8) of rows
// t / (DP / 8) + j RPP.  Rows past the tensor are clamped when loaded (every load stays in bounds)
// and stored as zeros by put_masked.
template <class T, int DP, int ROWS, int NTHR>
struct Tile {
    static constexpr int NCH = DP / 8, RPP = NTHR / NCH, N = ROWS / RPP;
    static_assert(ROWS % RPP == 0, "whole passes");
    static __device__ __forceinline__ int row(int tid, int j) { return tid / NCH + j * RPP; }
    static __device__ __forceinline__ int chunk(int tid) { return tid % NCH; }
    // rows r0 .. of `base` (token stride ld, `last` = highest row that exists, D <= DP columns)
    static __device__ __forceinline__ void load(u32x4 (&v)[N], const bf16_t* base, int64_t ld, int r0, int last, int D, int tid) {
        const int c = chunk(tid) * 8 < D ? chunk(tid) * 8 : 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int r = min(r0 + row(tid, j), last);
            v[j] = *(const u32x4*)(base + (int64_t)r * ld + c);
        }
    }
    static __device__ __forceinline__ void put(bf16_t* img, const u32x4 (&v)[N], int tid) {
#pragma unroll
        for (int j = 0; j < N; ++j) *(u32x4*)(img + chunk_at<DP>(row(tid, j), chunk(tid))) = v[j];
    }
    // Tiles that not all of the block's rows see: rows outside [keep0, keep1) (relative to the tile)
    // and columns past D are zeros, and so are infinities and NaN (a product with a masked
    // probability 0 would make them NaN); `flags` gets a byte per chunk that says where.
    static __device__ __forceinline__ void put_masked(bf16_t* img, const u32x4 (&v)[N], int tid, int keep0, int keep1, int D,
                                                      uint8_t* flags) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int r = row(tid, j), c = chunk(tid);
            const bool in = r >= keep0 && r < keep1 && c * 8 < D;
            const bool bad = in && not_finite8<T>(v[j]);
            const u32x4 z = (u32x4)(0u);
            u32x4 u = in ? v[j] : z;
            if (bad) u = finite_only<T>(u);
            *(u32x4*)(img + chunk_at<DP>(r, c)) = u;
            flags[r * NCH + c] = bad ? 1 : 0;
        }
    }
};
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return __builtin_amdgcn_readfirstlane((uint32_t)(size_t)(const __attribute__((address_space(3))) char*)p);
}
// The same tile copied from memory straight into LDS: a wave's 64 copies land side by side, so the swizzle
// is on the memory side (thread t copies the chunk that belongs at place t of the image).  Nothing passes
// through registers, and a copy is waited for only where its tile is about to be read (landed()).
template <class T, int DP, int ROWS, int NTHR>
struct Copy {
    static constexpr int NCH = DP / 8, RPP = NTHR / NCH, N = ROWS / RPP;
    static_assert(ROWS % RPP == 0 && RPP % 16 == 0, "whole passes that keep the swizzle");
    static __device__ __forceinline__ int row(int tid, int j) { return tid / NCH + j * RPP; }
    static __device__ __forceinline__ int chunk(int tid) { return (tid % NCH) ^ swz_key<DP>(tid / NCH); }
    uint32_t off, step;
    __device__ __forceinline__ void init(int64_t ld, int D, int tid) {
        off = (uint32_t)(row(tid, 0) * ld + (chunk(tid) * 8 < D ? chunk(tid) * 8 : 0)) * 2u;   // (fix zeroes the columns past D)
        step = (uint32_t)(RPP * ld) * 2u;
    }
    // ROWS rows from `first`, of which `left` exist (those past the last are out of the resource's range), to
    // LDS address img; w: the wave's number
    __device__ __forceinline__ void start(uint32_t img, const bf16_t* first, int64_t ld, int left, int D, int w) const {
        const __amdgpu_buffer_rsrc_t b = __builtin_amdgcn_make_buffer_rsrc(
            (void*)first, 0, (uint32_t)((min(left, ROWS) - 1) * (uint32_t)ld + D) * 2u, 0x00020000);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            // (from asm: before a transposed LDS read the compiler waits for every copy it knows of, it cannot
            // tell the two buffers apart)
            const uint32_t at = __builtin_amdgcn_readfirstlane(img + (j * NTHR + w * 64) * 16);
            // (5 wait states before the first: the resource's registers might have been written by the vector ALU)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop %c3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(at),
                         "v"(off + j * step), "s"(b), "n"(j == 0 ? 4 : 0) : "memory", "m0");
        }
    }
    // the columns past D, in whose place column 0 was copied
    static __device__ __forceinline__ void trim(bf16_t* img, int tid, int D) {
        if (chunk(tid) * 8 >= D)
#pragma unroll
            for (int j = 0; j < N; ++j) *(u32x4*)(img + (j * NTHR + tid) * 8) = (u32x4)(0u);
    }
    // put_masked of a tile that has landed: each thread mends what it copied
    static __device__ __forceinline__ void fix(bf16_t* img, int tid, int keep0, int keep1, int D, uint8_t* flags) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int r = row(tid, j), c = chunk(tid);
            u32x4* p = (u32x4*)(img + (j * NTHR + tid) * 8);
            u32x4 u = *p;
            const bool in = r >= keep0 && r < keep1 && c * 8 < D;
            const bool bad = in && not_finite8<T>(u);
            if (bad) u = finite_only<T>(u);
            if (!in) u = (u32x4)(0u);
            if (bad || !in) *p = u;
            flags[r * NCH + c] = bad ? 1 : 0;
        }
    }
};
// all but the newest N of the wave's loads, copies and stores are done
template <int N>
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(%c0)" ::"n"(N) : "memory"); }
// barrier that leaves copies in flight (__syncthreads waits for them); LDS reads and writes are done
__device__ __forceinline__ void barrier_lds() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// the flagged rows of a tile: bit l set where a chunk of row `row` of lane l was not finite
template <int DP>
__device__ __forceinline__ uint64_t flagged_rows(const uint8_t* flags, int row) {
    const uint2* p = (const uint2*)(flags + row * (DP / 8));
    uint32_t any = p[0].x | p[0].y;
    if (DP == 128) any |= p[1].x | p[1].y;
    return __ballot(any != 0);
}
__device__ __forceinline__ uint64_t bits_below(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; }

}  // namespace mattn

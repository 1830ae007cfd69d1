// Masked attention, backward: two kernels without atomics, so the gradients are the same bits in
// every run (the stage audit recomputes them).  See masked_attention.h for the mathematics.
//   dQ     (query on the lane, as the forward): S^T and dP^T again, dX^T in registers is the B operand
//          of dQ^T += K^T dX^T; also delta = rowsum(dO o), which the second kernel reads
//   dK, dV (key on the lane): over all query heads of the group and the queries that see the block
//          (ktab), dV^T += dO^T P and dK^T += Q^T dX: a shared head's gradients are sums in registers
#include "masked_attention.h"

using namespace mattn;

// ============================================================================ fp16's range
// dX is rounded to the inputs' type for the last product.  In fp16 it would leave the normal range where
// probabilities (1 / T) and upstream gradients are small (1024 keys, |dO| ~ 1: steps of 6e-8 in values of
// 1e-5; dQ and dK 1.8 times as far off as their own rounding) and overflow where values or a loss scale make
// them large, so it is scaled by a power of two that follows from a bound of it:
//   dS_ij = P_ij dO_i . (v_j - o_i),   v_j - o_i = sum_{k != j} P_ik (v_j - v_k)
//   |dX_ij| <= |dS_ij| <= P (1 - P) |dO_i| 2 max|v| <= B = max|dO_i| max|v_j| / 2      (row norms, visible rows)
// 2^n B in [2^14, 2^15): half of the range is left for the roundings in P and delta, and the steps are 2^-39 B.
// First the largest squares of row norms (not finite elements left out: they make their rows NaN anyhow),
// one of each kind per workgroup.
constexpr int NMAX = 256;
// A wave takes 64 rows: (token, head) of dO, then neighbouring keys of a head of V, all loads of a row on their
// way at once.  Bound by latency: 4 x 777, 12 heads of 64: 10 us (a thread per key over all heads: 48 us).
template <class T, int DP>
__device__ __forceinline__ float row_square(const bf16_t* row, int D) {
    u32x4 u[DP / 8];
#pragma unroll
    for (int c = 0; c < DP / 8; ++c) u[c] = *(const u32x4*)(row + (8 * c < D ? 8 * c : 0));
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < DP / 8; ++c) {
        u[c] = finite_only<T>(u[c]);
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float x, y;
            T::unpack(u[c][k], x, y);
            t = fmaf(x, x, fmaf(y, y, t));
        }
        s += 8 * c < D ? t : 0.f;
    }
    return s;
}
// whether some query of batch row b sees the lane's key j (64 neighbours of one ktab block, j < Tk)
__device__ __forceinline__ bool key_seen(const Args& a, int b, int block, int j) {
    const int nq = (a.Tq + QT - 1) / QT, nk = (a.Tk + KT - 1) / KT, lane = threadIdx.x & 63;
    const int2 range = a.ktab[(int64_t)b * nk + block];
    bool seen = false;
    for (int t = range.x; t < range.y && !__all(seen || j >= a.Tk); ++t) {
        const int4 e = a.qtab[(int64_t)b * nq + t];
        seen |= j >= e.z && j < e.w;                          // all rows of the tile see it
        if (!__any(!seen && j >= e.x && j < e.y)) continue;   // (no row sees any other)
        const int i = min(t * QT + (lane & 31), a.Tq - 1);
        const int lo = a.lo[(int64_t)b * a.Tq + i], hi = a.hi[(int64_t)b * a.Tq + i];
#pragma unroll
        for (int r = 0; r < QT; ++r) seen |= j >= __builtin_amdgcn_readlane(lo, r) && j < __builtin_amdgcn_readlane(hi, r);
    }
    return seen && j < a.Tk;
}
template <class T, int DP>
__global__ __launch_bounds__(256) void mattn_norm_max_kernel(const Args a) {
    __shared__ uint32_t red[2][4];
    float m[2] = {0.f, 0.f};
    const int64_t rows = (int64_t)a.B * a.Tq * a.H;
    for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < rows; x += NMAX * 256) {
        const int64_t row = x / a.H, b = row / a.Tq;
        const int hh = (int)(x - row * a.H), t = (int)(row - b * a.Tq);
        const float q = row_square<T, DP>((const bf16_t*)a.dout + b * a.dos[0] + t * a.dos[1] + hh * a.dos[2], a.D);
        m[0] = fmaxf(m[0], a.lo[row] < a.hi[row] ? q : 0.f);
    }
    const int nb = (a.Tk + 63) / 64;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int64_t x = (int64_t)blockIdx.x * 4 + w; x < (int64_t)a.B * nb * a.Hk; x += NMAX * 4) {
        const int64_t y = x / nb;
        const int kb = (int)(x - y * nb), b = (int)(y / a.Hk), hh = (int)(y - (int64_t)b * a.Hk), j = kb * 64 + (threadIdx.x & 63);
        const float q = row_square<T, DP>((const bf16_t*)a.v + b * a.vs[0] + min(j, a.Tk - 1) * a.vs[1] + hh * a.vs[2], a.D);
        m[1] = fmaxf(m[1], key_seen(a, b, kb * 64 / KT, j) ? q : 0.f);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {   // (not negative: ordered as their bits)
        const int v = wave_max_i((int)__float_as_uint(m[k]));
        if ((threadIdx.x & 63) == 0) red[k][w] = (uint32_t)v;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        const uint32_t* r = red[threadIdx.x];
        ((uint32_t*)a.ws)[NMAX * threadIdx.x + blockIdx.x] = max(max(r[0], r[1]), max(r[2], r[3]));
    }
}
// the exponent n of the scale, 0 where dO or V is zero
template <class T>
__device__ __forceinline__ int scale_exponent(const Args& a) {
    if constexpr (T::INF == 0x7f80) return 0;   // bf16 has fp32's range
    float big[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const uint4 u = ((const uint4*)a.ws)[64 * k + (threadIdx.x & 63)];
        big[k] = __uint_as_float((uint32_t)wave_max_i((int)max(max(u.x, u.y), max(u.z, u.w))));
    }
    const float bound = 0.5f * sqrtf(big[0] * big[1]);   // (squares of fp16 norms: in [2^-48, 2^39], no product leaves fp32's range)
    return bound == 0.f ? 0 : 14 - (int)((__float_as_uint(bound) >> 23) - 127u);
}

// ============================================================================ dQ
// Workgroup and tiles as in the forward.  Bound by the vector ALU: 500 instructions for 64 keys of a capped
// score, 48 of them products.  Two waves a SIMD (three, for heads of 64: 88 against 85 us on 16 x 1024).
// 2 x 8192, 16 heads of 128 on 4, cap 50: 990 us (one wave a SIMD, tiles through registers: 1656 us);
// 16 x 1024 in documents, 16 heads of 64: 70 us.
template <class T, int DP, bool CAP, bool ALIBI>
__global__ __launch_bounds__(256, 2) void mattn_dq_kernel(const Args a) {
    constexpr int NW = 4, BM = QT * NW, BN = 64, NS = DP / 16, NO = DP / 32, NTHR = 64 * NW;
    typedef Copy<T, DP, BN, NTHR> CP;
    __shared__ __attribute__((aligned(16))) bf16_t Ks[2][BN * DP];
    __shared__ __attribute__((aligned(16))) bf16_t Vs[2][BN * DP];
    __shared__ __attribute__((aligned(16))) uint8_t kflag[2][BN * (DP / 8)];
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, r = lane & 31;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nblk = (a.Tq + BM - 1) / BM;
    const Where at = place(blockIdx.x, a, nblk, true);
    const int q0 = at.blk * BM + QT * w;
    const int qi = q0 + r, qc = min(qi, a.Tq - 1);
    const bf16_t* kbase = (const bf16_t*)a.k + at.b * a.ks[0] + at.hk * a.ks[2];
    const bf16_t* vbase = (const bf16_t*)a.v + at.b * a.vs[0] + at.hk * a.vs[2];
    const bf16_t* qrow = (const bf16_t*)a.q + at.b * a.qs[0] + at.h * a.qs[2] + (int64_t)qc * a.qs[1];
    const bf16_t* drow = (const bf16_t*)a.dout + at.b * a.dos[0] + at.h * a.dos[2] + (int64_t)qc * a.dos[1];
    const bf16_t* orow = (const bf16_t*)a.o + at.b * a.os[0] + at.h * a.os[2] + (int64_t)qc * a.os[1];
    const int64_t stat = ((int64_t)at.b * a.H + at.h) * a.Tq + qc;
    int lo = a.lo[(int64_t)at.b * a.Tq + qc], hi = a.hi[(int64_t)at.b * a.Tq + qc];
    if (qi >= a.Tq) lo = hi = 0;
    const float lse2 = a.lse[stat] * LOG2E;
    const int ex = scale_exponent<T>(a);
    const float up = ldexpf(1.f, ex);
    // delta = dO . (o + what its rounding left out); the halves of the wave hold the halves of each row
    const uint32_t* rest = a.rest + (((int64_t)at.b * a.Tq + qc) * a.H + at.h) * a.D / 4;
    typename T::vec qf[NS], df[NS];
    float delta = 0.f;
    u32x4 du[NS], ou[NS];
    uint2 rw[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {   // every load on its way before the first is waited for
        const int c = 16 * s + 8 * h, cc = c < a.D ? c : 0;
        const u32x4 z = (u32x4)(0u), qu = *(const u32x4*)(qrow + cc);
        du[s] = *(const u32x4*)(drow + cc);
        ou[s] = *(const u32x4*)(orow + cc);
        rw[s] = *(const uint2*)(rest + cc / 4);
        qf[s] = as_vec<T>(c < a.D ? qu : z);
        du[s] = c < a.D ? du[s] : z;
        ou[s] = c < a.D ? ou[s] : z;
        df[s] = as_vec<T>(du[s]);
    }
#pragma unroll
    for (int s = 0; s < NS; ++s) {   // (past D: 0 times 0 plus a finite remainder)
        float rv[8];
        Rest<T>::back(rw[s].x, *(float(*)[4])rv);
        Rest<T>::back(rw[s].y, *(float(*)[4])(rv + 4));
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float d0, d1, o0, o1;
            T::unpack(du[s][k], d0, d1);
            T::unpack(ou[s][k], o0, o1);
            delta = fmaf(d0, o0 + rv[2 * k], delta);
            delta = fmaf(d1, o1 + rv[2 * k + 1], delta);
        }
    }
    delta += __shfl_xor(delta, 32, 64);
    {   // for dK / dV: planes of lse log2(e) and -delta; behind the last row of a head infinity (a weight of
        // exactly 0, whatever bias its distance would have) and 0
        const int tp = (a.Tq + QT - 1) / QT * QT;
        float* st = a.delta + ((int64_t)at.b * a.H + at.h) * 2 * tp;
        if (h == 0 && qi < tp) {
            st[qi] = qi < a.Tq ? lse2 - (float)T::UP : INFINITY;   // (dK / dV's weights: times 2^UP)
            st[tp + qi] = qi < a.Tq ? -delta : 0.f;
        }
    }
    Score<CAP, ALIBI> sc;
    sc.init(a.scale, a.cap, ALIBI ? a.slopes[at.h] : 0.f);
    const int qpos = ALIBI ? a.pos[at.b] + qi : 0;

    const int nq = (a.Tq + QT - 1) / QT, t0 = at.blk * NW;
    int bl = 0x7fffffff, bh = 0, bfl = 0, bfh = 0x7fffffff;
    int wl = 0x7fffffff, wh = 0, wfl = 0, wfh = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        const int4 e = t0 + i < nq ? a.qtab[(int64_t)at.b * nq + t0 + i] : make_int4(0x7fffffff, 0, 0, 0);
        bl = min(bl, e.x);
        bh = max(bh, e.y);
        bfl = max(bfl, e.z);
        bfh = min(bfh, e.w);
        if (i == w) {
            wl = e.x;
            wh = e.y;
            wfl = e.z;
            wfh = e.w;
        }
    }
    f32x16 dq[NO];
#pragma unroll
    for (int i = 0; i < NO; ++i) dq[i] = (f32x16){};
    bool poison = false;
    const int kb0 = bh > bl ? bl / BN : 0, kb1 = bh > bl ? (bh + BN - 1) / BN : 0;
    const int tq = (lane & 15) >> 2, tcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    CP kc, vc;
    kc.init(a.ks[1], a.D, tid);
    vc.init(a.vs[1], a.D, tid);
    const uint32_t kat = lds_address(Ks), vat = lds_address(Vs);
    const bf16_t *kp = kbase + (int64_t)kb0 * BN * a.ks[1], *vp = vbase + (int64_t)kb0 * BN * a.vs[1];   // next to copy
    const int64_t kstep = BN * a.ks[1], vstep = BN * a.vs[1];
    auto fetch = [&](int kb, int buf) {   // kb0, then one after the other
        kc.start(kat + buf * (BN * DP * 2), kp, a.ks[1], a.Tk - kb * BN, a.D, w);
        vc.start(vat + buf * (BN * DP * 2), vp, a.vs[1], a.Tk - kb * BN, a.D, w);
        kp += kstep;
        vp += vstep;
    };
    auto whole = [&](int kb) { return kb * BN >= bfl && (kb + 1) * BN <= bfh && a.D == DP; };
    auto mend = [&](int kb, int buf) {
        // K meets masked zeros of dX in the last product: a masked key that is not finite is stored as
        // zeros, a visible one makes the row NaN through its flag
        landed<0>();
        if (whole(kb)) return;
        if (a.D != DP) CP::trim(Vs[buf], tid, a.D);
        CP::fix(Ks[buf], tid, bl - kb * BN, bh - kb * BN, a.D, kflag[buf]);
    };
    auto compute = [&](int kb, int buf) {
        if (kb * BN >= wh || (kb + 1) * BN <= wl) return;
        const bf16_t* K_ = Ks[buf];
        const bf16_t* V_ = Vs[buf];
        const bool part = kb * BN < wfl || (kb + 1) * BN > wfh;
        if (!whole(kb)) {
            const uint64_t bad = flagged_rows<DP>(kflag[buf], lane);
            if (bad != 0) poison |= (bad & bits_below(hi - kb * BN) & ~bits_below(lo - kb * BN)) != 0;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {   // 32 keys at a time: half the score registers
            f32x16 s = {}, p;
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] = -delta;   // the product leaves dP - delta
#pragma unroll
            for (int d = 0; d < NS; ++d) {
                const int at_ = chunk_at<DP>(32 * t + r, 2 * d + h);
                s = T::mfma(as_vec<T>(*(const u32x4*)(K_ + at_)), qf[d], s);
                p = T::mfma(as_vec<T>(*(const u32x4*)(V_ + at_)), df[d], p);
            }
            const float d0 = ALIBI ? (float)(kb * BN + 32 * t + 4 * h - qpos) : 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int kk = (i & 3) + 8 * (i >> 2);
                float e, x = p[i];
                if constexpr (Score<CAP, ALIBI>::PLAIN) {
                    e = exp2_fast(fmaf(s[i], sc.mul, -lse2));
                } else if constexpr (CAP) {
                    const float q4 = sc.sat(s[i]);
                    if constexpr (ALIBI) e = exp2_fast(sc.biased(sc.capped(q4), d0 + (float)kk) - lse2);
                    else e = exp2_fast(fmaf(-2.f * sc.capl, q4, sc.capl - lse2));
                    x *= fmaf(-q4, q4, q4);   // (1 - tanh^2) / 4
                } else {
                    e = exp2_fast(sc(s[i], d0 + (float)kk) - lse2);
                }
                s[i] = e * x;
                if constexpr (T::INF != 0x7f80) s[i] *= up;
            }
            if (part) {
                asm volatile("" : "+v"(s));   // (a branch, and not 3 instructions a score in every tile)
                const int k0 = kb * BN + 32 * t + 4 * h - lo;
                const uint32_t n = (uint32_t)(hi - lo);
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = (uint32_t)(k0 + (i & 3) + 8 * (i >> 2)) < n ? s[i] : 0.f;
            }
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                const typename T::vec ds = round8<T>(s, s2);
                const int row = 32 * t + 16 * s2 + 4 * h + tq;
#pragma unroll
                for (int i = 0; i < NO; ++i) dq[i] = T::mfma(tr_pair<T, DP>(K_, row, 32 * i + tcol), ds, dq[i]);
            }
        }
    };
    if (kb0 < kb1) {
        fetch(kb0, 0);
        mend(kb0, 0);
    }
    for (int kb = kb0; kb < kb1; ++kb) {
        const int buf = (kb - kb0) & 1;
        barrier_lds();   // tile kb is complete, the other buffer has been read
        if (kb + 1 < kb1) fetch(kb + 1, buf ^ 1);
        compute(kb, buf);
        if (kb + 1 < kb1) mend(kb + 1, buf ^ 1);
    }
    const float gscale = (CAP ? 4.f * a.scale : a.scale) * ldexpf(1.f, -ex);   // (with the 4 of the cap's derivative)
    if (qi < a.Tq) {
        bf16_t* out = (bf16_t*)a.dq + at.b * a.dqs[0] + at.h * a.dqs[2] + (int64_t)qi * a.dqs[1];
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * i + 8 * g + 4 * h;
                uint2 u;
                u.x = T::pack(dq[i][4 * g] * gscale, dq[i][4 * g + 1] * gscale);
                u.y = T::pack(dq[i][4 * g + 2] * gscale, dq[i][4 * g + 3] * gscale);
                if (poison) u.x = u.y = T::NANBITS | T::NANBITS << 16;
                if (d < a.D) *(uint2*)(out + d) = u;
            }
    }
}

// ============================================================================ dK, dV
// Workgroup = 128 keys of one KV head (a wave owns 32, key on the lane, K and V fragments resident);
// walks the 32-query tiles that see the block, head after head of the group.  One wave's work on tile t
// is three stages: A(t) the products S and dP, B(t) the 16 scores a lane holds (vector ALU alone), C(t)
// the products dV and dK.  Run one after the other the matrix unit idles through B and the ALU through A
// and C, and the registers (accumulators of 2 x DP x 32, fragments of K and V) leave only one or two
// waves per SIMD to fill in for it.  So the loop is pipelined in the wave: an iteration
// interleaves C(t - 1), B(t) and A(t + 1), two scores between every few products, each product's LDS
// fragment read two products ahead.  Eight places for tiles of Q / dO are in LDS: t - 1 .. t + 1 are
// read, t + 2 .. t + 4 are on their way (copies straight from memory); one barrier per tile.
// 2 x 8192, 16 heads of 128 on 4, cap 50: 1613 us, 3500 cycles a tile of which 1024 are products (reading
// fragments 4 or 5 products ahead gained nothing); 16 x 1024 in documents, 16 heads of 64: 105 us (115 without
// the pipeline).
template <class T, int DP, bool CAP, bool ALIBI>
__global__ __launch_bounds__(256, DP == 64 ? 2 : 1) void mattn_dkdv_kernel(const Args a) {
    constexpr int NS = DP / 16, NO = DP / 32, RING = 8;
    constexpr int NA = 2 * NS, NC = 4 * NO, STEPS = 8, AS = NA / STEPS, CS = NC / STEPS, AHEAD = 2;
    typedef Copy<T, DP, QT, 256> CP;
    typedef typename T::vec vec;
    constexpr int IMG = QT * DP;
    __shared__ __attribute__((aligned(16))) bf16_t tiles[RING][2 * IMG];   // Q, then dO
    // per query row: lse log2(e) - UP, -delta, lo, hi
    __shared__ __attribute__((aligned(16))) uint32_t rowc[RING][4 * QT];
    __shared__ __attribute__((aligned(16))) uint8_t qflag[RING][QT * (DP / 8)], dflag[RING][QT * (DP / 8)];
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, r = lane & 31;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nkv = a.B * a.Hk, G = a.H / a.Hk;
    const int kv = blockIdx.x % nkv, kbi = blockIdx.x / nkv, b = kv / a.Hk, hk = kv - b * a.Hk;
    const int nq = (a.Tq + QT - 1) / QT, nk = (a.Tk + KT - 1) / KT;
    const int k0 = kbi * KT + 32 * w, kj = k0 + r, kc = min(kj, a.Tk - 1);
    const int2 range = a.ktab[(int64_t)b * nk + kbi];
    const int total = (range.y - range.x) * G;

    vec kf[NS], vf[NS];
    {
        const bf16_t* krow = (const bf16_t*)a.k + b * a.ks[0] + hk * a.ks[2] + (int64_t)kc * a.ks[1];
        const bf16_t* vrow = (const bf16_t*)a.v + b * a.vs[0] + hk * a.vs[2] + (int64_t)kc * a.vs[1];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int c = 16 * s + 8 * h, cc = c < a.D ? c : 0;
            const u32x4 z = (u32x4)(0u), ku = *(const u32x4*)(krow + cc), vu = *(const u32x4*)(vrow + cc);
            kf[s] = as_vec<T>(c < a.D ? ku : z);
            vf[s] = as_vec<T>(c < a.D ? vu : z);
        }
    }
    f32x16 dk[NO], dv[NO];
#pragma unroll
    for (int i = 0; i < NO; ++i) dk[i] = dv[i] = (f32x16){};
    bool poison = false;
    NotFinite odd;
    const int tq = (lane & 15) >> 2, tcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    Score<CAP, ALIBI> sc;
    sc.init(a.scale, a.cap, 0.f);
    const int ex = scale_exponent<T>(a);
    const float up = ldexpf(1.f, ex - T::UP);   // (the weights have the rest)
    const int kpos = ALIBI ? kj - a.pos[b] : 0;   // the distance to query i is i - kpos

    const bf16_t* qbase = (const bf16_t*)a.q + b * a.qs[0] + (int64_t)hk * G * a.qs[2];
    const bf16_t* dbase = (const bf16_t*)a.dout + b * a.dos[0] + (int64_t)hk * G * a.dos[2];
    // a place in the walk: head of the group and query tile
    struct At {
        int g, t;
    };
    auto advance = [&](At& x) {
        if (++x.t == range.y) {
            x.t = range.x;
            ++x.g;
        }
    };
    // this lane's word of a tile's row constants (waves 2 and 3 copy what 0 and 1 do: every wave has the
    // same number of copies in flight)
    const int kind = 2 * (w & 1) + h, tp = nq * QT;
    const uint32_t* rbase = kind < 2 ? (const uint32_t*)a.delta + (((int64_t)b * a.H + hk * G) * 2 + kind) * tp
                                     : (const uint32_t*)(kind == 2 ? a.lo : a.hi) + (int64_t)b * a.Tq;
    const int rhead = kind < 2 ? 2 * tp : 0, rlast = kind < 2 ? tp - 1 : a.Tq - 1;
    CP qc, dc;
    qc.init(a.qs[1], a.D, tid);
    dc.init(a.dos[1], a.D, tid);
    constexpr int COPIES = 2 * CP::N + 1;   // a tile's, per wave
    const uint32_t tat = lds_address(tiles), rat = lds_address(rowc) + 256 * (w & 1);
    // the next tile to copy: the first rows, and how far to the next tile and from a head's last to the next head
    const bf16_t *qp = qbase + (int64_t)range.x * QT * a.qs[1], *dp = dbase + (int64_t)range.x * QT * a.dos[1];
    const uint32_t* rp = rbase;
    const int64_t qstep = QT * a.qs[1], dstep = QT * a.dos[1];
    const int64_t qhead = a.qs[2] - (range.y - range.x) * qstep, dhead = a.dos[2] - (range.y - range.x) * dstep;
    auto fetch = [&](At& x, int buf) __attribute__((always_inline)) {
        const int left = a.Tq - x.t * QT;
        qc.start(tat + buf * (4 * IMG), qp, a.qs[1], left, a.D, w);
        dc.start(tat + buf * (4 * IMG) + 2 * IMG, dp, a.dos[1], left, a.D, w);
        const uint32_t* p = rp + min(x.t * QT + r, rlast);
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(rat + buf * (16 * QT)), "v"(p) : "memory", "m0");
        qp += qstep;
        dp += dstep;
        if (++x.t == range.y) {
            x.t = range.x;
            ++x.g;
            qp += qhead;
            dp += dhead;
            rp += rhead;
        }
    };
    struct Bounds {
        int lo, hi, full_lo, full_hi;   // some row sees [lo, hi), every row sees [full_lo, full_hi)
    };
    // 64 entries of the table at a time stand in the wave's lanes (a scalar load in the loop would be waited
    // for by the next LDS read)
    int part_of_tab = -1;
    int4 tab;
    auto bounds = [&](const At& x) __attribute__((always_inline)) {
        const int i = x.t - range.x;
        if (i >> 6 != part_of_tab) {
            part_of_tab = i >> 6;
            tab = a.qtab[(int64_t)b * nq + min(x.t - (i & 63) + lane, nq - 1)];
            // (waited for here: a load that might be pending at the loop's head would be waited for there in
            // every iteration, and with it every copy in flight)
            asm volatile("" : "+v"(tab.x), "+v"(tab.y), "+v"(tab.z), "+v"(tab.w));
        }
        return Bounds{__builtin_amdgcn_readlane(tab.x, i & 63), __builtin_amdgcn_readlane(tab.y, i & 63),
                      __builtin_amdgcn_readlane(tab.z, i & 63), __builtin_amdgcn_readlane(tab.w, i & 63)};
    };
    // every key of the block is seen by every row of a tile
    auto whole = [&](const At& x, const Bounds& e) {
        return e.full_lo <= kbi * KT && e.full_hi >= (kbi + 1) * KT && a.D == DP && (x.t + 1) * QT <= a.Tq;
    };
    // of a tile that has landed: the rows past the last are zeros, and their weights too (lse log2(e) is
    // padded with infinities), so whatever interval their constants say they add nothing
    auto mend = [&](const At& x, const Bounds& e, int buf) __attribute__((always_inline)) {
        if (whole(x, e)) return;
        CP::fix(tiles[buf], tid, 0, a.Tq - x.t * QT, a.D, qflag[buf]);   // (as K in dQ)
        CP::fix(tiles[buf] + IMG, tid, 0, a.Tq - x.t * QT, a.D, dflag[buf]);
    };
    auto active = [&](const Bounds& e) { return e.lo < k0 + 32 && e.hi > k0; };   // some row sees a key of the wave

    // where the lane's fragments stand in a tile's image: chunks 2 d + h of its row; rows 4 h + tq (and
    // 8 further) of the columns 32 i + tcol (16 rows on, a chunk's place in its row is the same)
    int rowat[NS], colat[NO][2];
#pragma unroll
    for (int d = 0; d < NS; ++d) rowat[d] = chunk_at<DP>(r, 2 * d + h);
#pragma unroll
    for (int i = 0; i < NO; ++i) {
        colat[i][0] = elem_at<DP>(4 * h + tq, 32 * i + tcol);
        colat[i][1] = elem_at<DP>(4 * h + tq + 8, 32 * i + tcol);
    }
    struct Scores {
        f32x16 s, p;          // S, then P; dP - delta, then dX
    };
    vec pb[2], db[2];         // tile t - 1: P and dX, rounded
    float d0;
    auto init_b = [&](const At& x) {
        if (ALIBI) {
            sc.slope = a.slopes[hk * G + x.g] * LOG2E;
            d0 = (float)(x.t * QT + 4 * h - kpos);
        }
    };
    auto score = [&](Scores& y, auto xc, float ls) __attribute__((always_inline)) {
        constexpr int i = decltype(xc)::value, qq = (i & 3) + 8 * (i >> 2);
        float e, x = y.p[i];
        if constexpr (Score<CAP, ALIBI>::PLAIN) {
            e = exp2_fast(fmaf(y.s[i], sc.mul, -ls));
        } else if constexpr (CAP) {
            const float q4 = sc.sat(y.s[i]);
            if constexpr (ALIBI) e = exp2_fast(sc.biased(sc.capped(q4), d0 + (float)qq) - ls);
            else e = exp2_fast(fmaf(-2.f * sc.capl, q4, sc.capl - ls));
            x *= fmaf(-q4, q4, q4);
        } else {
            e = exp2_fast(sc(y.s[i], d0 + (float)qq) - ls);
        }
        x *= e;
        if constexpr (T::INF != 0x7f80) x *= up;
        asm volatile("" : "+v"(e), "+v"(x));   // here, between the products, and not sunk behind them
        y.s[i] = e;
        y.p[i] = x;
    };
    // masks of tile t, and the operands of C(t)
    auto finish_b = [&](const At& x, const Bounds& bnd, Scores& y, int buf) __attribute__((always_inline)) {
        f32x16 &s = y.s, &p = y.p;
        const bool part = bnd.full_lo > k0 || bnd.full_hi < k0 + 32;
        const uint32_t* rw = rowc[buf];
        if (part) {
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const int4 l4 = *(const int4*)((const int*)rw + 2 * QT + 8 * g4 + 4 * h);
                const int4 h4 = *(const int4*)((const int*)rw + 3 * QT + 8 * g4 + 4 * h);
                const int ll[4] = {l4.x, l4.y, l4.z, l4.w}, hh[4] = {h4.x, h4.y, h4.z, h4.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const bool see = kj >= ll[k] && kj < hh[k];
                    s[4 * g4 + k] = see ? s[4 * g4 + k] : 0.f;
                    p[4 * g4 + k] = see ? p[4 * g4 + k] : 0.f;
                }
            }
        }
        if (!whole(x, bnd)) {   // a query that is not finite: NaN for the keys it sees
            uint32_t bad = (uint32_t)flagged_rows<DP>(qflag[buf], r);
            while (bad != 0) {
                const int q = __builtin_ctz(bad);
                bad &= bad - 1;
                poison |= kj >= (int)rw[2 * QT + q] && kj < (int)rw[3 * QT + q];
            }
            bad = (uint32_t)flagged_rows<DP>(dflag[buf], r);   // dO: dP, so dK, is NaN by itself
            while (bad != 0) {
                const int q = __builtin_ctz(bad);
                bad &= bad - 1;
                odd.note<T, NO>(dbase + x.g * a.dos[2] + (int64_t)(x.t * QT + q) * a.dos[1], a.D, h,
                                kj >= (int)rw[2 * QT + q] && kj < (int)rw[3 * QT + q]);
            }
        }
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) pb[s2] = round8<T>(s, s2), db[s2] = round8<T>(p, s2);
    };
    // (DP 128: one wave per SIMD, sums in AGPRs; DP 64: two, all in ordinary registers)
    auto mul_acc = [&](f32x16& c, const vec& x, const vec& y) __attribute__((always_inline)) {
        if constexpr (DP == 128) T::mfma_acc(c, x, y);
        else c = T::mfma(x, y, c);
    };
    // one iteration: C of the tile in LDS slot bc, B of tile x (bounds bnd, scores y) in slot bb, A of slot ba
    // (scores yn), as far as they are wanted
    auto run = [&](auto cc, auto bc_, auto ac, const At& x, const Bounds& bnd, Scores& y, Scores& yn, int bc, int bb,
                   int ba) __attribute__((always_inline)) {
        constexpr bool C = decltype(cc)::value, B = decltype(bc_)::value, A = decltype(ac)::value;
        vec fa[NA], fc[NC];
        auto load_a = [&](auto ic) {
            constexpr int i = decltype(ic)::value;
            if constexpr (i < NA) fa[i] = as_vec<T>(*(const u32x4*)(tiles[ba] + rowat[i / 2] + (i & 1 ? IMG : 0)));
        };
        auto load_c = [&](auto ic) {
            constexpr int i = decltype(ic)::value;
            if constexpr (i < NC)
                fc[i] = tr_pair<T>(tiles[bc] + colat[i / 2 % NO][0] + (i & 1 ? 0 : IMG) + 16 * DP * (i / (2 * NO)),
                                   tiles[bc] + colat[i / 2 % NO][1] + (i & 1 ? 0 : IMG) + 16 * DP * (i / (2 * NO)));
        };
        if constexpr (A) {
            yn.s = (f32x16){};
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const float4 c = *(const float4*)((const float*)rowc[ba] + QT + 8 * g4 + 4 * h);
                yn.p[4 * g4] = c.x, yn.p[4 * g4 + 1] = c.y, yn.p[4 * g4 + 2] = c.z, yn.p[4 * g4 + 3] = c.w;
            }
            unrolled<AHEAD>(load_a);
        }
        if constexpr (C) unrolled<AHEAD>(load_c);
        if constexpr (B) init_b(x);
        unrolled<STEPS>([&](auto sc_) {
            constexpr int st = decltype(sc_)::value;
            const float2 ls = *(const float2*)((const float*)rowc[bb] + (2 * st & 3) + 8 * (st >> 1) + 4 * h);
            if constexpr (C)
                unrolled<CS>([&](auto k) {
                    constexpr int i = st * CS + decltype(k)::value, s2 = i / (2 * NO), o = i / 2 % NO;
                    load_c(std::integral_constant<int, i + AHEAD>{});
                    if constexpr (i & 1) mul_acc(dk[o], fc[i], db[s2]);
                    else mul_acc(dv[o], fc[i], pb[s2]);
                });
            if constexpr (A)
                unrolled<AS>([&](auto k) {
                    constexpr int i = st * AS + decltype(k)::value;
                    load_a(std::integral_constant<int, i + AHEAD>{});
                    if constexpr (i & 1) yn.p = T::mfma(fa[i], vf[i / 2], yn.p);
                    else yn.s = T::mfma(fa[i], kf[i / 2], yn.s);
                });
            if constexpr (B) {   // scores 2 st, 2 st + 1: neighbouring rows
                score(y, std::integral_constant<int, 2 * st>{}, ls.x);
                score(y, std::integral_constant<int, 2 * st + 1>{}, ls.y);
            }
            __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (B) finish_b(x, bnd, y, bb);
    };
    constexpr std::true_type Y{};
    constexpr std::false_type N{};

    At ld{0, range.x}, tb{0, range.x}, st{0, range.x}, cur{0, range.x};   // next to copy, to look up, to mend; tile t
    Scores y0, y1;
    Bounds e0{0, 0, 0, 0}, e1{0, 0, 0, 0}, e2{0, 0, 0, 0};   // of tiles t, t + 1, t + 2
    bool acc_ = false;   // tile t - 1 has work for this wave
#pragma unroll
    for (int i = 0; i < 2; ++i) pb[i] = db[i] = as_vec<T>((u32x4)(0u));
    auto look_up = [&]() __attribute__((always_inline)) {   // past the last tile: no work
        Bounds e{0, 0, 0, 0};
        if (tb.g < G) e = bounds(tb);
        advance(tb);
        return e;
    };
    auto copy_next = [&](int t) __attribute__((always_inline)) {
        if (t < total) fetch(ld, t & (RING - 1));
    };
    // tile t is complete but for the barrier; tiles up to t + 2 may be on their way
    auto await = [&](int t, const Bounds& e) __attribute__((always_inline)) {
        if (t >= total) return;
        if (t + 2 < total) landed<2 * COPIES>();
        else landed<0>();
        mend(st, e, t & (RING - 1));
        advance(st);
    };
    if (total > 0) {
        // the last place stands for tile -1: finite values for the weights 0 of the first C
        for (int i = tid; i < 2 * IMG / 8; i += 256) ((u32x4*)tiles[RING - 1])[i] = (u32x4)(0u);
#pragma unroll
        for (int i = 0; i < 4; ++i) copy_next(i);
        e0 = look_up();
        e1 = look_up();
        e2 = look_up();
        await(0, e0);
        await(1, e1);
        barrier_lds();
        run(N, N, Y, cur, e0, y1, y0, 0, 0, 0);
    }
    // tile t: its scores in y, the next tile's in yn
    auto iter = [&](int t, Scores& y, Scores& yn) __attribute__((always_inline)) {
        copy_next(t + 4);
        const Bounds e3 = look_up();
        const bool act = active(e0);
        // a tile without work inside the pipeline counts with weights 0 (its masks leave nothing); the
        // products of a tile past the last are not used
        if (acc_ || act || active(e1)) {
            run(Y, Y, Y, cur, e0, y, yn, (t - 1) & (RING - 1), t & (RING - 1), (t + 1) & (RING - 1));
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) pb[i] = db[i] = as_vec<T>((u32x4)(0u));
        }
        await(t + 2, e2);
        acc_ = act;
        e0 = e1;
        e1 = e2;
        e2 = e3;
        advance(cur);
        barrier_lds();
    };
    for (int t = 0; t < total; t += 2) {
        iter(t, y0, y1);
        if (t + 1 < total) iter(t + 1, y1, y0);
    }
    if (total > 0) run(Y, N, N, cur, e0, y0, y1, (total - 1) & (RING - 1), 0, 0);
    if constexpr (DP == 128) acc_done(dk, dv);
    const float gscale = (CAP ? 4.f * a.scale : a.scale) * ldexpf(1.f, -ex), vscale = ldexpf(1.f, -T::UP);
    if (kj < a.Tk) {
        bf16_t* dkr = (bf16_t*)a.dk + b * a.dks[0] + hk * a.dks[2] + (int64_t)kj * a.dks[1];
        bf16_t* dvr = (bf16_t*)a.dv + b * a.dvs[0] + hk * a.dvs[2] + (int64_t)kj * a.dvs[1];
        if (odd.any()) {
#pragma unroll
            for (int i = 0; i < NO; ++i)
#pragma unroll
                for (int k = 0; k < 16; ++k) dv[i][k] = odd(dv[i][k], 16 * i + k);
        }
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * i + 8 * g + 4 * h;
                uint2 u, v;
                u.x = T::pack(dk[i][4 * g] * gscale, dk[i][4 * g + 1] * gscale);
                u.y = T::pack(dk[i][4 * g + 2] * gscale, dk[i][4 * g + 3] * gscale);
                v.x = T::pack(dv[i][4 * g] * vscale, dv[i][4 * g + 1] * vscale);
                v.y = T::pack(dv[i][4 * g + 2] * vscale, dv[i][4 * g + 3] * vscale);
                if (poison) u.x = u.y = v.x = v.y = T::NANBITS | T::NANBITS << 16;
                if (d < a.D) {
                    *(uint2*)(dkr + d) = u;
                    *(uint2*)(dvr + d) = v;
                }
            }
    }
}

// ============================================================================ host
template <class T, int DP, bool CAP, bool ALIBI>
static int bwd_launch(const Args& a, hipStream_t s) {
    const int64_t gq = (int64_t)a.B * a.H * ((a.Tq + 127) / 128), gk = (int64_t)a.B * a.Hk * ((a.Tk + KT - 1) / KT);
    if (gq > MAX_GRID || gk > MAX_GRID) return (int)hipErrorInvalidValue;
    int rc = 0;
    if constexpr (T::INF != 0x7f80) {
        mattn_norm_max_kernel<T, DP><<<NMAX, 256, 0, s>>>(a);
        rc = (int)hipGetLastError();
        if (rc) return rc;
    }
    mattn_dq_kernel<T, DP, CAP, ALIBI><<<(int)gq, 256, 0, s>>>(a);
    rc = (int)hipGetLastError();
    if (rc || a.dk == nullptr) return rc;   // no gradient of the keys and values wanted
    mattn_dkdv_kernel<T, DP, CAP, ALIBI><<<(int)gk, 256, 0, s>>>(a);
    TDL_LAUNCH_CHECK();
}

template <class T, int DP>
static int bwd_score(const Args& a, hipStream_t s) {
    const bool cap = a.cap > 0.f, al = a.slopes != nullptr;
    if (cap && al) return bwd_launch<T, DP, true, true>(a, s);
    if (cap) return bwd_launch<T, DP, true, false>(a, s);
    if (al) return bwd_launch<T, DP, false, true>(a, s);
    return bwd_launch<T, DP, false, false>(a, s);
}

// args: mattn::Args with o, lse and rest from the forward; delta: planes of [B H][2][Tq padded to 32]
// floats, ws: 512 words (fp16), both written and read
TDL_API int tdl_masked_attn_bwd(const void* args, hipStream_t s) {
    const Args& a = *(const Args*)args;
    if (a.B <= 0 || a.Tq <= 0 || a.Tk <= 0 || a.H <= 0 || a.Hk <= 0 || a.H % a.Hk || a.D <= 0 || a.D > 128 || a.D % 8 ||
        (a.dtype != 1 && a.dtype != 2) || !(a.scale > 0.f) || a.cap < 0.f)
        return (int)hipErrorInvalidValue;
    if (a.dtype == 1) return a.D <= 64 ? bwd_score<Bf16, 64>(a, s) : bwd_score<Bf16, 128>(a, s);
    return a.D <= 64 ? bwd_score<F16, 64>(a, s) : bwd_score<F16, 128>(a, s);
}

// Masked attention, backward: two kernels without atomics, so the gradients are the same bits in
// every run (the stage audit recomputes them).  See masked_attention.h for the mathematics.
//   dQ     (query on the lane, as the forward): S^T and dP^T again, dX^T in registers is the B operand
//          of dQ^T += K^T dX^T; also delta = rowsum(dO o), which the second kernel reads
//   dK, dV (key on the lane): over all query heads of the group and the queries that see the block
//          (ktab), dV^T += dO^T P and dK^T += Q^T dX: a shared head's gradients are sums in registers
#include "masked_attention.h"

using namespace mattn;

// ============================================================================ dQ
template <class T, int DP, bool CAP, bool ALIBI, int NW>
__global__ __launch_bounds__(64 * NW, DP == 64 ? 8 / NW : 1) void mattn_dq_kernel(const Args a) {
    constexpr int BM = QT * NW, BN = 64, NS = DP / 16, NO = DP / 32, NTHR = 64 * NW;
    typedef Tile<T, DP, BN, NTHR> TL;
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
    // delta: both factors as the forward left them; the halves of the wave hold the halves of each row
    typename T::vec qf[NS], df[NS];
    float delta = 0.f;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int c = 16 * s + 8 * h, cc = c < a.D ? c : 0;
        const u32x4 z = (u32x4)(0u);
        const u32x4 qu = *(const u32x4*)(qrow + cc), du = *(const u32x4*)(drow + cc), ou = *(const u32x4*)(orow + cc);
        qf[s] = as_vec<T>(c < a.D ? qu : z);
        df[s] = as_vec<T>(c < a.D ? du : z);
        if (c < a.D) {
            const uint32_t dw[4] = {du.x, du.y, du.z, du.w}, ow[4] = {ou.x, ou.y, ou.z, ou.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float d0, d1, o0, o1;
                T::unpack(dw[k], d0, d1);
                T::unpack(ow[k], o0, o1);
                delta = fmaf(d0, o0, delta);
                delta = fmaf(d1, o1, delta);
            }
        }
    }
    delta += __shfl_xor(delta, 32, 64);
    if (h == 0 && qi < a.Tq) a.delta[stat] = delta;
    Score<CAP, ALIBI> sc;
    sc.init(a.scale, a.cap, ALIBI ? a.slopes[at.h] : 0.f);
    const float qpos = ALIBI ? (float)(a.pos[at.b] + qi) : 0.f;

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
    u32x4 kr[TL::N], vr[TL::N];
    auto gload = [&](int kb) {
        TL::load(kr, kbase, a.ks[1], kb * BN, a.Tk - 1, a.D, tid);
        TL::load(vr, vbase, a.vs[1], kb * BN, a.Tk - 1, a.D, tid);
    };
    auto whole = [&](int kb) { return kb * BN >= bfl && (kb + 1) * BN <= bfh && a.D == DP; };
    auto sstore = [&](int kb, int buf) {
        // K meets masked zeros of dX in the last product: a masked key that is not finite is stored as
        // zeros, a visible one makes the row NaN through its flag
        if (whole(kb)) TL::put(Ks[buf], kr, tid);
        else TL::put_masked(Ks[buf], kr, tid, bl - kb * BN, bh - kb * BN, a.D, kflag[buf]);
        TL::put(Vs[buf], vr, tid);
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
            const float d0 = ALIBI ? (float)(kb * BN + 32 * t + 4 * h) - qpos : 0.f;
            const int k0 = kb * BN + 32 * t + 4 * h - lo;
            const uint32_t n = (uint32_t)(hi - lo);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int kk = (i & 3) + 8 * (i >> 2);
                float e, x = p[i];
                if constexpr (Score<CAP, ALIBI>::PLAIN) {
                    e = exp2_fast(fmaf(s[i], sc.mul, -lse2));
                } else if constexpr (CAP) {
                    const float q4 = sc.sat(s[i]);
                    e = exp2_fast(sc.biased(sc.capped(q4), d0 + (float)kk) - lse2);
                    x *= fmaf(-4.f * q4, q4, 4.f * q4);   // 1 - tanh^2
                } else {
                    e = exp2_fast(sc(s[i], d0 + (float)kk) - lse2);
                }
                e *= x;
                if (part) e = (uint32_t)(k0 + kk) < n ? e : 0.f;
                s[i] = e;
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
        gload(kb0);
        sstore(kb0, 0);
        __syncthreads();
    }
    for (int kb = kb0; kb < kb1; ++kb) {
        const int buf = (kb - kb0) & 1;
        const bool next = kb + 1 < kb1;
        if (next) gload(kb + 1);
        compute(kb, buf);
        if (next) sstore(kb + 1, buf ^ 1);
        __syncthreads();
    }
    if (qi < a.Tq) {
        bf16_t* out = (bf16_t*)a.dq + at.b * a.dqs[0] + at.h * a.dqs[2] + (int64_t)qi * a.dqs[1];
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * i + 8 * g + 4 * h;
                uint2 u;
                u.x = T::pack(dq[i][4 * g] * a.scale, dq[i][4 * g + 1] * a.scale);
                u.y = T::pack(dq[i][4 * g + 2] * a.scale, dq[i][4 * g + 3] * a.scale);
                if (poison) u.x = u.y = T::NANBITS | T::NANBITS << 16;
                if (d < a.D) *(uint2*)(out + d) = u;
            }
    }
}

// ============================================================================ dK, dV
// Workgroup = 128 keys of one KV head (a wave owns 32, key on the lane, K and V fragments resident);
// walks the 32-query tiles that see the block, head after head of the group, with the next tile's
// Q / dO rows and row constants loaded into registers during the current one (one barrier per tile).
template <class T, int DP, bool CAP, bool ALIBI>
__global__ __launch_bounds__(256, DP == 64 ? 2 : 1) void mattn_dkdv_kernel(const Args a) {
    constexpr int NS = DP / 16, NO = DP / 32;
    typedef Tile<T, DP, QT, 256> TL;
    __shared__ __attribute__((aligned(16))) bf16_t Qs[2][QT * DP];
    __shared__ __attribute__((aligned(16))) bf16_t Ds[2][QT * DP];
    // per query row: lse log2(e), -delta, lo, hi; then the tile's qtab entry
    __shared__ __attribute__((aligned(16))) uint32_t rowc[2][4 * QT + 4];
    __shared__ __attribute__((aligned(16))) uint8_t qflag[2][64 * (DP / 8)], dflag[2][64 * (DP / 8)];
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, r = lane & 31;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nkv = a.B * a.Hk, G = a.H / a.Hk;
    const int kv = blockIdx.x % nkv, kbi = blockIdx.x / nkv, b = kv / a.Hk, hk = kv - b * a.Hk;
    const int nq = (a.Tq + QT - 1) / QT, nk = (a.Tk + KT - 1) / KT;
    const int k0 = kbi * KT + 32 * w, kj = k0 + r, kc = min(kj, a.Tk - 1);
    const int2 range = a.ktab[(int64_t)b * nk + kbi];
    const int nt = range.y - range.x, total = nt * G;
    for (int i = tid; i < 2 * 64 * (DP / 8); i += 256) (&qflag[0][0])[i] = (&dflag[0][0])[i] = 0;   // rows 32 .. 63 stay clear

    typename T::vec kf[NS], vf[NS];
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
    const int tq = (lane & 15) >> 2, tcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    Score<CAP, ALIBI> sc;
    sc.init(a.scale, a.cap, 0.f);
    const float kpos = ALIBI ? (float)(kj - a.pos[b]) : 0.f;   // the distance to query i is i - kpos

    const bf16_t* qbase = (const bf16_t*)a.q + b * a.qs[0] + (int64_t)hk * G * a.qs[2];
    const bf16_t* dbase = (const bf16_t*)a.dout + b * a.dos[0] + (int64_t)hk * G * a.dos[2];
    const int64_t srow = ((int64_t)b * a.H + hk * G) * a.Tq;
    u32x4 qr[TL::N], dr[TL::N];
    uint32_t rc;   // this thread's row constant of the staged tile
    int ng = 0, ntile = range.x;   // the tile that gload takes next: head of the group, query tile
    auto gload = [&]() {
        TL::load(qr, qbase + ng * a.qs[2], a.qs[1], ntile * QT, a.Tq - 1, a.D, tid);
        TL::load(dr, dbase + ng * a.dos[2], a.dos[1], ntile * QT, a.Tq - 1, a.D, tid);
        const int kind = tid >> 5, q = min(ntile * QT + (tid & 31), a.Tq - 1);
        const uint32_t* p = kind == 0   ? (const uint32_t*)a.lse + srow + (int64_t)ng * a.Tq + q
                            : kind == 1 ? (const uint32_t*)a.delta + srow + (int64_t)ng * a.Tq + q
                            : kind == 2 ? (const uint32_t*)a.lo + (int64_t)b * a.Tq + q
                            : kind == 3 ? (const uint32_t*)a.hi + (int64_t)b * a.Tq + q
                                        : (const uint32_t*)(a.qtab + (int64_t)b * nq + ntile) + (tid & 3);
        rc = *p;
    };
    int cg = 0, ct = range.x;   // the tile in registers, then in LDS
    auto sstore = [&](int buf) {
        const int4 e = a.qtab[(int64_t)b * nq + ct];
        const bool whole = e.z <= kbi * KT && e.w >= (kbi + 1) * KT;
        if (whole && a.D == DP) {
            TL::put(Qs[buf], qr, tid);
            TL::put(Ds[buf], dr, tid);
        } else {
            TL::put_masked(Qs[buf], qr, tid, 0, a.Tq - ct * QT, a.D, qflag[buf]);   // (as K in dQ)
            TL::put_masked(Ds[buf], dr, tid, 0, a.Tq - ct * QT, a.D, dflag[buf]);
        }
        const int kind = tid >> 5;
        uint32_t v = rc;
        if (kind == 0) v = __float_as_uint(__uint_as_float(rc) * LOG2E);
        if (kind == 1) v = __float_as_uint(-__uint_as_float(rc));
        if ((kind == 2 || kind == 3) && ct * QT + (tid & 31) >= a.Tq) v = 0;   // no such query: sees nothing
        if (tid < 4 * QT + 4) rowc[buf][tid] = v;
    };
    auto compute = [&](int qt, int buf) {
        const uint32_t* rw = rowc[buf];
        const int el = __builtin_amdgcn_readfirstlane((int)rw[4 * QT]), eh = __builtin_amdgcn_readfirstlane((int)rw[4 * QT + 1]);
        const int efl = __builtin_amdgcn_readfirstlane((int)rw[4 * QT + 2]), efh = __builtin_amdgcn_readfirstlane((int)rw[4 * QT + 3]);
        if (el >= k0 + 32 || eh <= k0) return;
        const bool part = efl > k0 || efh < k0 + 32;
        const bf16_t* Q_ = Qs[buf];
        const bf16_t* D_ = Ds[buf];
        f32x16 s = {}, p;
        float ls[16];
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
            const float4 c = *(const float4*)((const float*)rw + QT + 8 * g4 + 4 * h);
            const float4 e = *(const float4*)((const float*)rw + 8 * g4 + 4 * h);
            p[4 * g4] = c.x, p[4 * g4 + 1] = c.y, p[4 * g4 + 2] = c.z, p[4 * g4 + 3] = c.w;
            ls[4 * g4] = e.x, ls[4 * g4 + 1] = e.y, ls[4 * g4 + 2] = e.z, ls[4 * g4 + 3] = e.w;
        }
#pragma unroll
        for (int d = 0; d < NS; ++d) {
            const int at_ = chunk_at<DP>(r, 2 * d + h);
            s = T::mfma(as_vec<T>(*(const u32x4*)(Q_ + at_)), kf[d], s);
            p = T::mfma(as_vec<T>(*(const u32x4*)(D_ + at_)), vf[d], p);
        }
        const float d0 = ALIBI ? (float)(qt * QT + 4 * h) - kpos : 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int qq = (i & 3) + 8 * (i >> 2);
            float e, x = p[i];
            if constexpr (Score<CAP, ALIBI>::PLAIN) {
                e = exp2_fast(fmaf(s[i], sc.mul, -ls[i]));
            } else if constexpr (CAP) {
                const float q4 = sc.sat(s[i]);
                e = exp2_fast(sc.biased(sc.capped(q4), d0 + (float)qq) - ls[i]);
                x *= fmaf(-4.f * q4, q4, 4.f * q4);
            } else {
                e = exp2_fast(sc(s[i], d0 + (float)qq) - ls[i]);
            }
            s[i] = e;
            p[i] = e * x;
        }
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
        if (part || a.D != DP) {   // a query that is not finite: NaN for the keys it sees
            uint64_t bad = flagged_rows<DP>(qflag[buf], lane);
            while (bad != 0) {
                const int q = __builtin_ctzll(bad);
                bad &= bad - 1;
                poison |= kj >= (int)rw[2 * QT + q] && kj < (int)rw[3 * QT + q];
            }
            bad = flagged_rows<DP>(dflag[buf], lane);   // dO: dP, so dK, is NaN by itself
            while (bad != 0) {
                const int q = __builtin_ctzll(bad);
                bad &= bad - 1;
                add_not_finite<T>(dv, dbase + cg * a.dos[2] + (int64_t)(qt * QT + q) * a.dos[1], a.D, h,
                                  kj >= (int)rw[2 * QT + q] && kj < (int)rw[3 * QT + q]);
            }
        }
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
            const typename T::vec pb = round8<T>(s, s2), db = round8<T>(p, s2);
            const int row = 16 * s2 + 4 * h + tq;
#pragma unroll
            for (int i = 0; i < NO; ++i) {
                dv[i] = T::mfma(tr_pair<T, DP>(D_, row, 32 * i + tcol), pb, dv[i]);
                dk[i] = T::mfma(tr_pair<T, DP>(Q_, row, 32 * i + tcol), db, dk[i]);
            }
        }
    };
    auto advance = [&](int& g, int& t) {
        if (++t == range.y) {
            t = range.x;
            ++g;
        }
    };
    __syncthreads();   // the flags are clear
    if (total > 0) {
        gload();
        advance(ng, ntile);
        sstore(0);
        __syncthreads();
    }
    for (int it = 0; it < total; ++it) {
        const int buf = it & 1;
        const bool next = it + 1 < total;
        if (next) gload();
        if (ALIBI) sc.slope = a.slopes[hk * G + cg] * LOG2E;
        compute(ct, buf);
        advance(cg, ct);
        if (next) {
            advance(ng, ntile);
            sstore(buf ^ 1);
        }
        __syncthreads();
    }
    if (kj < a.Tk) {
        bf16_t* dkr = (bf16_t*)a.dk + b * a.dks[0] + hk * a.dks[2] + (int64_t)kj * a.dks[1];
        bf16_t* dvr = (bf16_t*)a.dv + b * a.dvs[0] + hk * a.dvs[2] + (int64_t)kj * a.dvs[1];
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * i + 8 * g + 4 * h;
                uint2 u, v;
                u.x = T::pack(dk[i][4 * g] * a.scale, dk[i][4 * g + 1] * a.scale);
                u.y = T::pack(dk[i][4 * g + 2] * a.scale, dk[i][4 * g + 3] * a.scale);
                v.x = T::pack(dv[i][4 * g], dv[i][4 * g + 1]);
                v.y = T::pack(dv[i][4 * g + 2], dv[i][4 * g + 3]);
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
    if (gq > 0x7fffffff || gk > 0x7fffffff) return (int)hipErrorInvalidValue;
    mattn_dq_kernel<T, DP, CAP, ALIBI, 4><<<(int)gq, 256, 0, s>>>(a);
    const int rc = (int)hipGetLastError();
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

// args: mattn::Args with o, lse from the forward; delta [B H Tq] floats is written and read
TDL_API int tdl_masked_attn_bwd(const void* args, hipStream_t s) {
    const Args& a = *(const Args*)args;
    if (a.B <= 0 || a.Tq <= 0 || a.Tk <= 0 || a.H <= 0 || a.Hk <= 0 || a.H % a.Hk || a.D <= 0 || a.D > 128 || a.D % 8 ||
        (a.dtype != 1 && a.dtype != 2) || !(a.scale > 0.f) || a.cap < 0.f)
        return (int)hipErrorInvalidValue;
    if (a.dtype == 1) return a.D <= 64 ? bwd_score<Bf16, 64>(a, s) : bwd_score<Bf16, 128>(a, s);
    return a.D <= 64 ? bwd_score<F16, 64>(a, s) : bwd_score<F16, 128>(a, s);
}

// Masked attention, forward: the mask's plan, the tiled kernel for many queries, the split kernel for
// few (single tokens against a cache) and its join.  See masked_attention.h for the mathematics.
#include "masked_attention.h"

using namespace mattn;

// ============================================================================ the mask's plan
// One workgroup per batch row.  Documents are runs of equal ids: the start of position j's run is a
// running maximum of run heads, its end (and the first unmarked position at or after j) a running
// minimum from the right.  Launch- and latency-bound (2 KiB of ids a row at 1024 tokens); made once per
// batch and used by every layer.
constexpr int PT = 1024;

// inclusive scan of one value per thread over the workgroup; `right` scans from the last thread
template <bool MAX>
__device__ __forceinline__ int block_scan(int v, bool right, int* red) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    auto op = [](int a, int b) { return MAX ? max(a, b) : min(a, b); };
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = right ? __shfl_down(v, o, 64) : __shfl_up(v, o, 64);
        if (right ? lane + o < 64 : lane >= o) v = op(v, u);
    }
    __syncthreads();
    if (lane == (right ? 0 : 63)) red[w] = v;
    __syncthreads();
    if (right) {
        for (int i = w + 1; i < PT / 64; ++i) v = op(v, red[i]);
    } else {
        for (int i = 0; i < w; ++i) v = op(v, red[i]);
    }
    return v;
}

template <class Id>
__global__ __launch_bounds__(PT) void attn_mask_kernel(const Id* __restrict__ documents, const int* __restrict__ prefix_rows,
                                                       const uint8_t* __restrict__ prefix_marks, const int* __restrict__ lengths,
                                                       const int* __restrict__ q_start, int Tq, int Tk, int causal, int* ws,
                                                       int* __restrict__ lo, int* __restrict__ hi, int* __restrict__ pos,
                                                       int4* qtab, int2* __restrict__ ktab) {
    __shared__ int red[PT / 64];
    __shared__ int carry;
    const int b = blockIdx.x, tid = threadIdx.x;
    const int big = 0x7fffffff;
    const int len = lengths != nullptr ? min(max(lengths[b], 0), Tk) : Tk;
    // the first query's position: given, or the queries are the last Tq valid positions of the row
    // (as many queries as keys: position 0)
    const int p0 = q_start != nullptr ? q_start[b] : (Tq < Tk ? len - Tq : 0);
    const Id* ids = documents != nullptr ? documents + (int64_t)b * Tk : nullptr;
    const uint8_t* marks = prefix_marks != nullptr ? prefix_marks + (int64_t)b * Tk : nullptr;
    int* start = ws + (int64_t)b * 3 * Tk;
    int* end = start + Tk;
    int* unmarked = end + Tk;
    const int chunks = (Tk + PT - 1) / PT;
    if (ids != nullptr) {
        if (tid == 0) carry = -1;
        for (int c = 0; c < chunks; ++c) {
            const int j = c * PT + tid;
            int v = -1;
            if (j < Tk && (j == 0 || ids[j] != ids[j - 1])) v = j;
            v = block_scan<true>(v, false, red);
            v = max(v, carry);
            if (j < Tk) start[j] = v;
            __syncthreads();
            if (tid == PT - 1) carry = v;
            __syncthreads();
        }
        if (tid == 0) carry = big;
        for (int c = chunks - 1; c >= 0; --c) {
            const int j = c * PT + tid;
            int v = big;
            if (j < Tk && (j + 1 == Tk || ids[j + 1] != ids[j])) v = j + 1;
            v = block_scan<false>(v, true, red);
            v = min(v, carry);
            if (j < Tk) end[j] = v;
            __syncthreads();
            if (tid == 0) carry = v;
            __syncthreads();
        }
    }
    if (marks != nullptr) {
        if (tid == 0) carry = big;
        for (int c = chunks - 1; c >= 0; --c) {
            const int j = c * PT + tid;
            int v = j < Tk && marks[j] == 0 ? j : big;
            v = block_scan<false>(v, true, red);
            v = min(v, carry);
            if (j < Tk) unmarked[j] = v;
            __syncthreads();
            if (tid == 0) carry = v;
            __syncthreads();
        }
    }
    __syncthreads();
    const int nq = (Tq + QT - 1) / QT, nk = (Tk + KT - 1) / KT;
    for (int i = tid; i < nq * QT; i += PT) {
        int l = 0, h = 0;
        const int64_t p = (int64_t)p0 + i;
        if (i < Tq && p >= 0 && p < len && (ids == nullptr || ids[p] >= 0)) {
            const int e = min(ids != nullptr ? end[p] : Tk, len);
            l = ids != nullptr ? start[p] : 0;
            h = e;
            if (causal) {
                int pe = 0;   // end of the prefix that this position's document (or row) starts with
                if (marks != nullptr) pe = unmarked[l];
                else if (prefix_rows != nullptr) pe = prefix_rows[b];
                h = max((int)p + 1, min(pe, e));
            }
        }
        if (i < Tq) {
            lo[(int64_t)b * Tq + i] = l;
            hi[(int64_t)b * Tq + i] = h;
        }
        int4 t = make_int4(h > l ? l : big, h, l, h);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            t.x = min(t.x, __shfl_xor(t.x, o, 32));
            t.y = max(t.y, __shfl_xor(t.y, o, 32));
            t.z = max(t.z, __shfl_xor(t.z, o, 32));
            t.w = min(t.w, __shfl_xor(t.w, o, 32));
        }
        if ((tid & 31) == 0) qtab[(int64_t)b * nq + i / QT] = t;
    }
    if (tid == 0) pos[b] = p0;
    __threadfence_block();
    __syncthreads();
    const int lane = tid & 63;
    for (int kb = tid >> 6; kb < nk; kb += PT / 64) {
        int f = big, l = 0;
        for (int t = lane; t < nq; t += 64) {
            const int4 e = qtab[(int64_t)b * nq + t];
            if (e.x < (kb + 1) * KT && e.y > kb * KT) {
                f = min(f, t);
                l = max(l, t + 1);
            }
        }
        f = wave_min_i(f);
        l = wave_max_i(l);
        if (lane == 0) ktab[(int64_t)b * nk + kb] = l > 0 ? make_int2(f, l) : make_int2(0, 0);
    }
}

// documents: int32 or (wide) int64 ids [B][Tk]; ws: 3 B Tk ints with documents or prefix_marks
TDL_API int tdl_attn_mask(const void* documents, int wide, const int* prefix_rows, const void* prefix_marks, const int* lengths,
                          const int* q_start, int B, int Tq, int Tk, int causal, int* ws, int* lo, int* hi, int* pos, void* qtab,
                          void* ktab, hipStream_t s) {
    if (B <= 0 || B >= 1 << 22 || Tq <= 0 || Tk < Tq || ((documents != nullptr || prefix_marks != nullptr) && ws == nullptr))
        return (int)hipErrorInvalidValue;
    const uint8_t* marks = (const uint8_t*)prefix_marks;
    if (wide)
        attn_mask_kernel<int64_t><<<B, PT, 0, s>>>((const int64_t*)documents, prefix_rows, marks, lengths, q_start, Tq, Tk, causal,
                                                   ws, lo, hi, pos, (int4*)qtab, (int2*)ktab);
    else
        attn_mask_kernel<int><<<B, PT, 0, s>>>((const int*)documents, prefix_rows, marks, lengths, q_start, Tq, Tk, causal, ws, lo,
                                               hi, pos, (int4*)qtab, (int2*)ktab);
    TDL_LAUNCH_CHECK();
}

// ============================================================================ many queries
// Workgroup = 128 queries of one head (a wave owns 32, query on the lane); keys in tiles of 64,
// copied straight into one of two LDS buffers while the other is read.  S^T = K Q^T leaves 16 keys of a
// 32-key tile on each lane, so a row's maximum and sum are lane-local (the two halves of the wave
// exchange their maximum), and the rounded S^T accumulator IS the B operand of O^T += V^T P^T.
// Bound by the vector ALU (16 scores a lane and 32-key tile: with a cap two exponentials, of 8 cycles each, a
// reciprocal, 8, and 3.5 others, 4, against 256 cycles of products for 64 columns), so three waves a SIMD
// (two from 65 columns on) take turns.  2 x 8192, 16 heads of 128 on 4, cap 50: 742 us; 8 x 2048, 25 heads of
// 64, cap 30: 201 us; 16 x 1024 in documents, 16 heads of 64: 56 us.
// FIXED: capped scores without a bias are taken less their bound, the cap (Score::below), so they lie in [-2 cap, 0].
// Up to a cap of 32 a bf16 softmax needs no running maximum then: its smallest weight is e^-64, well in
// bf16's range (not in fp16's).  The largest weight is not 1 as with a maximum, and its rounding, which a peaked row
// carries whole (2.3e-3 instead of 1.8e-3 of error at a cap of 30), cancels against the sum of the rounded weights.
// 8 x 2048, 25 heads of 64, whole calls: 191 us at a cap of 32, 208 at 33.
template <class T, int DP, bool CAP, bool ALIBI, bool FIXED>
__global__ __launch_bounds__(256, DP == 64 ? 3 : 2) void mattn_fwd_kernel(const Args a) {
    constexpr int NW = 4, BM = QT * NW, BN = 64, NS = DP / 16, NO = DP / 32, NTHR = 64 * NW;
    typedef Copy<T, DP, BN, NTHR> CP;
    __shared__ __attribute__((aligned(16))) bf16_t Ks[2][BN * DP];
    __shared__ __attribute__((aligned(16))) bf16_t Vs[2][BN * DP];
    __shared__ __attribute__((aligned(16))) uint8_t vflag[2][BN * (DP / 8)];
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, r = lane & 31;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);   // wave-uniform: tile tests are scalar branches
    const int nblk = (a.Tq + BM - 1) / BM;
    const Where at = place(blockIdx.x, a, nblk, true);
    const int q0 = at.blk * BM + QT * w;
    const int qi = q0 + r;
    const int qc = min(qi, a.Tq - 1);
    const bf16_t* kbase = (const bf16_t*)a.k + at.b * a.ks[0] + at.hk * a.ks[2];
    const bf16_t* vbase = (const bf16_t*)a.v + at.b * a.vs[0] + at.hk * a.vs[2];
    const bf16_t* qrow = (const bf16_t*)a.q + at.b * a.qs[0] + at.h * a.qs[2] + (int64_t)qc * a.qs[1];

    typename T::vec qf[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int c = 16 * s + 8 * h;
        const u32x4 u = *(const u32x4*)(qrow + (c < a.D ? c : 0));
        qf[s] = as_vec<T>(c < a.D ? u : (u32x4)(0u));
    }
    int lo = a.lo[(int64_t)at.b * a.Tq + qc], hi = a.hi[(int64_t)at.b * a.Tq + qc];
    if (qi >= a.Tq) lo = hi = 0;
    Score<CAP, ALIBI> sc;
    sc.init(a.scale, a.cap, ALIBI ? a.slopes[at.h] : 0.f);
    const int qpos = ALIBI ? a.pos[at.b] + qi : 0;

    // bounds of the intervals over the workgroup's and the wave's queries
    const int nq = (a.Tq + QT - 1) / QT, t0 = at.blk * NW;
    int bl = 0x7fffffff, bh = 0, bfl = 0, bfh = 0x7fffffff;   // some row sees [bl, bh); every row sees [bfl, bfh)
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
    f32x16 o[NO];
#pragma unroll
    for (int i = 0; i < NO; ++i) o[i] = (f32x16){};
    constexpr bool SAT = CAP && !ALIBI;
    static_assert(!FIXED || (SAT && T::INF == 0x7f80), "capped bf16 scores without a bias");
    float m = FIXED ? 0.f : -INFINITY, l = 0.f;
    float lr = 0.f;   // FIXED: the sum of the rounded weights
    NotFinite odd;
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
    auto whole = [&](int kb) { return kb * BN >= bfl && (kb + 1) * BN <= bfh && a.D == DP; };   // seen by every row
    auto mend = [&](int kb, int buf) {   // (a masked key's score is replaced, whatever it was; columns past D are not)
        landed<0>();
        if (whole(kb)) return;
        if (a.D != DP) CP::trim(Ks[buf], tid, a.D);
        CP::fix(Vs[buf], tid, bl - kb * BN, bh - kb * BN, a.D, vflag[buf]);
    };
    auto compute = [&](int kb, int buf) {
        if (kb * BN >= wh || (kb + 1) * BN <= wl) return;
        const bf16_t* K_ = Ks[buf];
        const bf16_t* V_ = Vs[buf];
        f32x16 s[2] = {(f32x16){}, (f32x16){}};
#pragma unroll
        for (int d = 0; d < NS; ++d) {
            const typename T::vec a0 = as_vec<T>(*(const u32x4*)(K_ + chunk_at<DP>(r, 2 * d + h)));
            const typename T::vec a1 = as_vec<T>(*(const u32x4*)(K_ + chunk_at<DP>(32 + r, 2 * d + h)));
            s[0] = T::mfma(a0, qf[d], s[0]);
            s[1] = T::mfma(a1, qf[d], s[1]);
        }
        if constexpr (SAT) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[t][i] = sc.below(s[t][i]);
        } else if constexpr (!Score<CAP, ALIBI>::PLAIN) {
            const float d0 = (float)(kb * BN + 4 * h - qpos);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[t][i] = sc(s[t][i], d0 + (float)(32 * t + (i & 3) + 8 * (i >> 2)));
        }
        if (kb * BN < wfl || (kb + 1) * BN > wfh) {   // some row of the wave sees only a part
            const int k0 = kb * BN + 4 * h - lo;
            const uint32_t n = (uint32_t)(hi - lo);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[t][i] = (uint32_t)(k0 + 32 * t + (i & 3) + 8 * (i >> 2)) < n ? s[t][i] : -INFINITY;
        }
        float mu = 0.f;   // what the exponents are less
        if constexpr (!FIXED) {
            float mx = max3(s[0][0], s[1][0], s[0][1]);
#pragma unroll
            for (int i = 1; i < 16; ++i) mx = max3(mx, s[1][i], i + 1 < 16 ? s[0][i + 1] : s[1][i]);
            const float ot = __shfl_xor(mx, 32, 64);
            mx = max3(mx, ot, ot);
            if constexpr (Score<CAP, ALIBI>::PLAIN) mx *= sc.mul;   // scale > 0: the maximum commutes with it
            const float mn = fmaxf(m, mx);
            const float ms = mn == -INFINITY ? 0.f : mn;   // nothing visible yet: 2^(-inf - 0) = 0
            if (__any(mn > m)) {   // the old sums keep their scale where no row's maximum rose
                const float alpha = exp2_fast(m - ms);
                l *= alpha;
#pragma unroll
                for (int i = 0; i < NO; ++i) o[i] *= alpha;
            }
            m = mn;
            mu = ms - (float)T::UP;
        }
        float rs = 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[t][i] = exp2_fast(Score<CAP, ALIBI>::PLAIN ? fmaf(s[t][i], sc.mul, -mu) : FIXED ? s[t][i] : s[t][i] - mu);
                rs += s[t][i];
            }
        l += rs;   // this half's keys; the halves are added at the end
        if (!whole(kb)) {
            uint64_t bad = flagged_rows<DP>(vflag[buf], lane);
            while (bad != 0) {
                const int k = kb * BN + __builtin_ctzll(bad);
                bad &= bad - 1;
                odd.note<T, NO>(vbase + (int64_t)k * a.vs[1], a.D, h, k >= lo && k < hi);
            }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2) {
                const typename T::vec pf = round8<T>(s[t], s2);
                if constexpr (FIXED) lr = sum8(pf, lr);
                const int row = 32 * t + 16 * s2 + 4 * h + tq;
#pragma unroll
                for (int i = 0; i < NO; ++i) o[i] = T::mfma(tr_pair<T, DP>(V_, row, 32 * i + tcol), pf, o[i]);
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
    l += __shfl_xor(l, 32, 64);
    if constexpr (FIXED) lr += __shfl_xor(lr, 32, 64);
    if (qi < a.Tq) {
        const float inv = l == 0.f ? 0.f : 1.f / (FIXED ? lr : l);   // nothing visible: 0
        bf16_t* orow = (bf16_t*)a.o + at.b * a.os[0] + at.h * a.os[2] + (int64_t)qi * a.os[1];
        if (odd.any()) {
#pragma unroll
            for (int i = 0; i < NO; ++i)
#pragma unroll
                for (int k = 0; k < 16; ++k) o[i][k] = odd(o[i][k], 16 * i + k);
        }
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * i + 8 * g + 4 * h;
                const float v[4] = {o[i][4 * g] * inv, o[i][4 * g + 1] * inv, o[i][4 * g + 2] * inv, o[i][4 * g + 3] * inv};
                uint2 u;
                u.x = T::pack(v[0], v[1]);
                u.y = T::pack(v[2], v[3]);
                if (d < a.D) {
                    *(uint2*)(orow + d) = u;
                    if (a.rest != nullptr) a.rest[((((int64_t)at.b * a.Tq + qi) * a.H + at.h) * a.D + d) / 4] = Rest<T>::of(v, u);
                }
            }
        if (h == 0 && a.lse != nullptr)
            a.lse[((int64_t)at.b * a.H + at.h) * a.Tq + qi] = l == 0.f ? -INFINITY : (m + (SAT ? sc.capl : 0.f) + (log2f(l) - T::UP)) * LN2;
    }
}

// ============================================================================ few queries
// four finished values of a row
template <class T>
__device__ __forceinline__ void put_out(const Args& a, const float (&acc)[4], float inv, int b, int h, int i, int d) {
    if (d >= a.D) return;
    const float v[4] = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
    uint2 u;
    u.x = T::pack(v[0], v[1]);
    u.y = T::pack(v[2], v[3]);
    *(uint2*)((bf16_t*)a.o + b * a.os[0] + h * a.os[2] + (int64_t)i * a.os[1] + d) = u;
    if (a.rest != nullptr) a.rest[((((int64_t)b * a.Tq + i) * a.H + h) * a.D + d) / 4] = Rest<T>::of(v, u);
}

// Single tokens (or a few) against a long cache: bound by reading K and V once.  The rows of a tile are
// the queries of ALL heads that share a KV head (row = g Tq + i), so the cache is read once per KV head;
// the keys are split over `nsplit` workgroups and, within one, over 4 waves that never wait for each
// other: a wave takes 32 keys at a time, K straight from memory into the operand registers, V through
// its own LDS for the transposing read, the next keys' loads in flight meanwhile.  Each workgroup joins
// its waves' (maximum, sum, O); mattn_join adds the splits.  48 caches of up to 8191 tokens, 32 heads of 128
// on 8: 272 us and 5 of joining, 3.8 TB/s; 4 caches of 5003, 7 queries: 18 us and 6 us of joining.
template <class T, int DP, bool CAP, bool ALIBI>
__global__ __launch_bounds__(256, 2) void mattn_few_kernel(const Args a) {
    constexpr int NS = DP / 16, NO = DP / 32, NW = 4, NCH = DP / 8;
    typedef Tile<T, DP, 32, 64> TL;   // one wave's V tile
    __shared__ __attribute__((aligned(16))) char smem[NW * 32 * DP * 2];   // V tiles; then halves of O, [wave][row][DP / 2] floats
    __shared__ float mls[NW][2][32];
    __shared__ __attribute__((aligned(16))) uint8_t vflag[NW][64 * NCH];
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, r = lane & 31;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int G = a.H / a.Hk, R = G * a.Tq, nkv = a.B * a.Hk;
    const int kv = blockIdx.x % nkv, y = blockIdx.x / nkv, split = y % a.nsplit, r0 = (y / a.nsplit) * 32;
    const int b = kv / a.Hk, hk = kv - b * a.Hk;
    const int nr = min(R - r0, 32);
    const int row = r0 + min(r, nr - 1), g = row / a.Tq, i0 = row - g * a.Tq, hq = hk * G + g;
    const bf16_t* kbase = (const bf16_t*)a.k + b * a.ks[0] + hk * a.ks[2];
    const bf16_t* vbase = (const bf16_t*)a.v + b * a.vs[0] + hk * a.vs[2];
    const bf16_t* qrow = (const bf16_t*)a.q + b * a.qs[0] + hq * a.qs[2] + (int64_t)i0 * a.qs[1];
    bf16_t* V_ = (bf16_t*)smem + w * 32 * DP;
    typename T::vec qf[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int c = 16 * s + 8 * h;
        const u32x4 u = *(const u32x4*)(qrow + (c < a.D ? c : 0));
        qf[s] = as_vec<T>(c < a.D ? u : (u32x4)(0u));
    }
    int lo = a.lo[(int64_t)b * a.Tq + i0], hi = a.hi[(int64_t)b * a.Tq + i0];
    if (r >= nr) lo = hi = 0;
    const int bl = wave_min_i(hi > lo ? lo : 0x7fffffff), bh = wave_max_i(hi);
    const int fl = wave_max_i(r < nr ? lo : 0), fh = wave_min_i(r < nr ? hi : 0x7fffffff);   // every row sees [fl, fh)
    Score<CAP, ALIBI> sc;
    sc.init(a.scale, a.cap, ALIBI ? a.slopes[hq] : 0.f);
    const int qpos = ALIBI ? a.pos[b] + i0 : 0;
    f32x16 o[NO];
#pragma unroll
    for (int i = 0; i < NO; ++i) o[i] = (f32x16){};
    float m = -INFINITY, l = 0.f;
    NotFinite odd;
    // this split's 32-key pieces u0 .. u1, dealt over the waves
    const int p0 = bh > bl ? bl / 32 : 0, np = bh > bl ? (bh + 31) / 32 - p0 : 0;
    const int per = (np + a.nsplit - 1) / a.nsplit;
    const int u0 = p0 + min(split * per, np), u1 = p0 + min((split + 1) * per, np);
    const int tq = (lane & 15) >> 2, tcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    u32x4 kr[NS], vr[TL::N];
    // 32 rows through a buffer resource that starts at the first: the lane's offsets never change (nor is
    // a 64-bit address held per load), keys past the tensor and columns past D (offset 2^31) read as zeros
    auto rows_of = [&](const bf16_t* base, int64_t ld, int u) {
        const int left = min(a.Tk - u * 32, 32);
        return __builtin_amdgcn_make_buffer_rsrc((void*)(base + (int64_t)u * 32 * ld), 0, (uint32_t)((left - 1) * ld + a.D) * 2u,
                                                 0x00020000);
    };
    const uint32_t koff = (uint32_t)(r * a.ks[1] + 8 * h) * 2u;
    const uint32_t voff = TL::chunk(lane) * 8 < a.D ? (uint32_t)(TL::row(lane, 0) * a.vs[1] + TL::chunk(lane) * 8) * 2u : 0x80000000u;
    const uint32_t vstep = (uint32_t)(TL::RPP * a.vs[1]) * 2u;   // (31 rows span less than 2 GiB: 2^31 + 31 rows stay out of range)
    auto gload = [&](int u) {
        const __amdgpu_buffer_rsrc_t kb_ = rows_of(kbase, a.ks[1], u), vb_ = rows_of(vbase, a.vs[1], u);
#pragma unroll
        for (int s = 0; s < NS; ++s)
            kr[s] = __builtin_amdgcn_raw_buffer_load_b128(kb_, 16 * s + 8 * h < a.D ? koff + 32 * s : 0x80000000u, 0, 0);
#pragma unroll
        for (int j = 0; j < TL::N; ++j) vr[j] = __builtin_amdgcn_raw_buffer_load_b128(vb_, voff + j * vstep, 0, 0);
    };
    int u = u0 + w;
    if (u < u1) gload(u);
    for (; u < u1; u += NW) {
        const int kb = u * 32;
        const bool part = kb < fl || kb + 32 > fh || a.D != DP;
        if (part) {
            TL::put_masked(V_, vr, lane, bl - kb, bh - kb, a.D, vflag[w]);
        } else {
            TL::put(V_, vr, lane);
        }
        f32x16 s = {};
#pragma unroll
        for (int d = 0; d < NS; ++d) s = T::mfma(as_vec<T>(kr[d]), qf[d], s);
        if (u + NW < u1) gload(u + NW);
        if constexpr (!Score<CAP, ALIBI>::PLAIN) {
            const float d0 = (float)(kb + 4 * h - qpos);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = sc(s[i], d0 + (float)((i & 3) + 8 * (i >> 2)));
        }
        if (part) {
            const int k0 = kb + 4 * h - lo;
            const uint32_t n = (uint32_t)(hi - lo);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = (uint32_t)(k0 + (i & 3) + 8 * (i >> 2)) < n ? s[i] : -INFINITY;
        }
        float mx = fmaxf(s[0], s[15]);
#pragma unroll
        for (int i = 1; i < 15; i += 2) mx = max3(mx, s[i], s[i + 1]);
        const float ot = __shfl_xor(mx, 32, 64);
        mx = max3(mx, ot, ot);
        if constexpr (Score<CAP, ALIBI>::PLAIN) mx *= sc.mul;
        const float mn = fmaxf(m, mx);
        const float ms = mn == -INFINITY ? 0.f : mn;
        if (__any(mn > m)) {
            const float alpha = exp2_fast(m - ms);
            l *= alpha;
#pragma unroll
            for (int i = 0; i < NO; ++i) o[i] *= alpha;
        }
        m = mn;
        const float mu = ms - (float)T::UP;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = exp2_fast(Score<CAP, ALIBI>::PLAIN ? fmaf(s[i], sc.mul, -mu) : s[i] - mu);
            l += s[i];
        }
        if (part) {
            uint32_t bad = (uint32_t)flagged_rows<DP>(vflag[w], lane & 31);
            while (bad != 0) {
                const int k = kb + __builtin_ctz(bad);
                bad &= bad - 1;
                odd.note<T, NO>(vbase + (int64_t)k * a.vs[1], a.D, h, k >= lo && k < hi);
            }
        }
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) {
            const typename T::vec pf = round8<T>(s, s2);
#pragma unroll
            for (int i = 0; i < NO; ++i) o[i] = T::mfma(tr_pair<T, DP>(V_, 16 * s2 + 4 * h + tq, 32 * i + tcol), pf, o[i]);
        }
    }
    l += __shfl_xor(l, 32, 64);
    // join the waves: weights 2^(m_w - M), O through LDS
    if (h == 0) {
        mls[w][0][r] = m;
        mls[w][1][r] = l;
    }
    __syncthreads();
    // (half of the columns at a time: no more LDS than the V tiles had)
    float* od = (float*)smem;
    constexpr int DH = DP / 2;
    if (odd.any()) {
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
            for (int k = 0; k < 16; ++k) o[i][k] = odd(o[i][k], 16 * i + k);
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
    if (half) __syncthreads();   // the first half has been read
    if (r < nr) {
#pragma unroll
        for (int i = 0; i < NO / 2; ++i)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                const f32x16& f = o[half * (NO / 2) + i];
                *(float4*)(od + ((w * nr + r) * DH + 32 * i + 8 * q4 + 4 * h)) =
                    make_float4(f[4 * q4], f[4 * q4 + 1], f[4 * q4 + 2], f[4 * q4 + 3]);
            }
    }
    __syncthreads();
    for (int e = tid; e < nr * (DH / 4); e += 256) {
        const int rr = e / (DH / 4), dh = (e - rr * (DH / 4)) * 4, d = half * DH + dh;
        float M = mls[0][0][rr];
#pragma unroll
        for (int x = 1; x < NW; ++x) M = fmaxf(M, mls[x][0][rr]);
        const float Ms = M == -INFINITY ? 0.f : M;
        float L = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < NW; ++x) {
            const float wt = exp2_fast(mls[x][0][rr] - Ms);
            const float4 f = *(const float4*)(od + ((x * nr + rr) * DH + dh));
            L += wt * mls[x][1][rr];
            acc[0] += wt * f.x;
            acc[1] += wt * f.y;
            acc[2] += wt * f.z;
            acc[3] += wt * f.w;
        }
        const int ro = r0 + rr, gg = ro / a.Tq, ii = ro - gg * a.Tq, hh = hk * G + gg;
        const int64_t out = ((int64_t)b * a.H + hh) * a.Tq + ii;
        if (a.nsplit > 1) {
            float* op = a.ws + (out * a.nsplit + split) * DP + d;
            float* ml = a.ws + ((int64_t)a.B * a.H * a.Tq * DP + out * 2) * a.nsplit + split * 2;
            *(float4*)op = make_float4(acc[0], acc[1], acc[2], acc[3]);
            if (d == 0) *(float2*)ml = make_float2(M, L);
        } else {
            const float inv = L == 0.f ? 0.f : 1.f / L;
            put_out<T>(a, acc, inv, b, hh, ii, d);
            if (d == 0 && a.lse != nullptr) a.lse[out] = L == 0.f ? -INFINITY : (M + (log2f(L) - T::UP)) * LN2;
        }
    }
    }
}

// one row per DP / 4 threads: the splits' (maximum, sum) and O, added in their order
template <class T, int DP>
__global__ __launch_bounds__(256) void mattn_join_kernel(const Args a) {
    constexpr int TPR = DP / 4;
    const int64_t rows = (int64_t)a.B * a.H * a.Tq;
    const int64_t out = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    const int d = (threadIdx.x % TPR) * 4;
    if (out >= rows) return;
    const float* op = a.ws + out * a.nsplit * DP + d;
    const float2* ml = (const float2*)(a.ws + (rows * DP + out * 2) * a.nsplit);
    float M = -INFINITY;
    for (int s = 0; s < a.nsplit; ++s) M = fmaxf(M, ml[s].x);
    const float Ms = M == -INFINITY ? 0.f : M;
    float L = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.nsplit; ++s) {
        const float2 e = ml[s];
        const float wt = exp2_fast(e.x - Ms);
        const float4 f = *(const float4*)(op + s * DP);
        L += wt * e.y;
        acc[0] += wt * f.x;
        acc[1] += wt * f.y;
        acc[2] += wt * f.z;
        acc[3] += wt * f.w;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int64_t bh = out / a.Tq;
    const int ii = (int)(out - bh * a.Tq), b = (int)(bh / a.H), hh = (int)(bh - (int64_t)b * a.H);
    put_out<T>(a, acc, inv, b, hh, ii, d);
    if (d == 0 && a.lse != nullptr) a.lse[out] = L == 0.f ? -INFINITY : (M + (log2f(L) - T::UP)) * LN2;
}

// ============================================================================ host
static bool bad_args(const Args& a) {
    return a.B <= 0 || a.Tq <= 0 || a.Tk <= 0 || a.H <= 0 || a.Hk <= 0 || a.H % a.Hk || a.D <= 0 || a.D > 128 || a.D % 8 ||
           (a.dtype != 1 && a.dtype != 2) || !(a.scale > 0.f) || a.cap < 0.f;
}

template <class T, int DP, bool CAP, bool ALIBI>
static int fwd_launch(const Args& a, hipStream_t s) {
    if (a.nsplit > 0) {
        const int R = (a.H / a.Hk) * a.Tq, rt = (R + 31) / 32;   // rows, tiles of 32
        const int64_t grid = (int64_t)a.B * a.Hk * a.nsplit * rt;
        const int rpb = 256 / (DP / 4);   // rows of the join per workgroup
        const int64_t joins = ((int64_t)a.B * a.H * a.Tq + rpb - 1) / rpb;
        if (grid > MAX_GRID || joins > MAX_GRID) return (int)hipErrorInvalidValue;
        mattn_few_kernel<T, DP, CAP, ALIBI><<<(int)grid, 256, 0, s>>>(a);
        if (a.nsplit > 1) {
            const int rc = (int)hipGetLastError();
            if (rc) return rc;
            mattn_join_kernel<T, DP><<<(int)joins, 256, 0, s>>>(a);
        }
        TDL_LAUNCH_CHECK();
    }
    const int64_t grid = (int64_t)a.B * a.H * ((a.Tq + 127) / 128);
    if (grid > MAX_GRID) return (int)hipErrorInvalidValue;
    if constexpr (CAP && !ALIBI && T::INF == 0x7f80) {
        if (a.cap <= 32.f) {
            mattn_fwd_kernel<T, DP, CAP, ALIBI, true><<<(int)grid, 256, 0, s>>>(a);
            TDL_LAUNCH_CHECK();
        }
    }
    mattn_fwd_kernel<T, DP, CAP, ALIBI, false><<<(int)grid, 256, 0, s>>>(a);
    TDL_LAUNCH_CHECK();
}

template <class T, int DP>
static int fwd_score(const Args& a, hipStream_t s) {
    const bool cap = a.cap > 0.f, al = a.slopes != nullptr;
    if (cap && al) return fwd_launch<T, DP, true, true>(a, s);
    if (cap) return fwd_launch<T, DP, true, false>(a, s);
    if (al) return fwd_launch<T, DP, false, true>(a, s);
    return fwd_launch<T, DP, false, false>(a, s);
}

// args: mattn::Args.  nsplit = 0: the tiled kernel; >= 1: the few-queries kernel over that many key
// ranges (ws: B H Tq nsplit (DP + 2) floats when nsplit > 1, DP = 64 or 128 >= D).
TDL_API int tdl_masked_attn_fwd(const void* args, hipStream_t s) {
    const Args& a = *(const Args*)args;
    if (bad_args(a)) return (int)hipErrorInvalidValue;
    if (a.dtype == 1) return a.D <= 64 ? fwd_score<Bf16, 64>(a, s) : fwd_score<Bf16, 128>(a, s);
    return a.D <= 64 ? fwd_score<F16, 64>(a, s) : fwd_score<F16, 128>(a, s);
}

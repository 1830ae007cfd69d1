// Distillation from a teacher's top logits, mixed with cross-entropy: loss and gradient in one pass over
// the student's logits.
//
//   q   = softmax over a row's teacher entries of t / tau            p_tau = softmax_j(z / tau),  p = softmax_j(z)
//   kd  = tau^2 sum_k q_k (log q_k - log p_tau(i_k))                 ce = -log p(label)
//   loss = alpha mean_kd + (1 - alpha) mean_ce    (means over the rows that have entries / a label)
//   dz_j = alpha tau / n_t (p_tau_j - sum_{k : i_k = j} q_k) + (1 - alpha) / n_l (p_j - [j = label])
//
// Bound by memory: the logits are read and their gradient written once each, 3.3 GB and 748 us a call (4.4 TB/s)
// for 16384 rows of 50304 bf16 logits.  A row belongs to one workgroup (a wave, for short rows) that
// keeps it in registers between the statistics and the gradient, or, where there are many long rows,
// reads it a second time from the Infinity Cache: 5 rows of 100 KB a CU are 130 MB of its 256 MB, and the
// gradient is stored past it (nontemporal: 834 instead of 886 us).
//
// The gradient at a row's few special columns (its teacher entries and label) is written over the
// row's stores by threads that own an entry, from the same fp32 terms and with one rounding: the
// lowest entry of several with the same index sums them in order, so no atomics, no fixed order lost.
#include "common.h"

namespace {

constexpr int MAX_K = 1024;
constexpr int MAX_DIM = 1 << 30;   // rows and columns stay below: an index plus a stride of the grid fits an int
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct F32 {
    typedef float S;
    static constexpr int E = 4;   // values of 16 bytes
    static __device__ __forceinline__ float get(S v) { return v; }
    static __device__ __forceinline__ S put(float v) { return v; }
    static __device__ __forceinline__ void unpack(const u32x4& u, float (&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(u[i]);
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[4]) {
        return u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    }
};
struct B16 {
    typedef uint16_t S;
    static constexpr int E = 8;
    static __device__ __forceinline__ float get(S v) { return bf2f(v); }
    static __device__ __forceinline__ S put(float v) { return f2bf(v); }
    static __device__ __forceinline__ void unpack(const u32x4& u, float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(u[i] << 16);
            f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
        return u32x4{pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7])};
    }
};
struct H16 {
    typedef uint16_t S;
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    static constexpr int E = 8;
    static __device__ __forceinline__ float get(S v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ __forceinline__ S put(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
    static __device__ __forceinline__ void unpack(const u32x4& u, float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = u[i];   // (bit_cast of the element itself was compiled as element 0 for all i)
            const h2 h = __builtin_bit_cast(h2, w);
            f[2 * i] = (float)h[0];
            f[2 * i + 1] = (float)h[1];
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
        u32x4 u;
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = __builtin_bit_cast(uint32_t, h2{(_Float16)f[2 * i], (_Float16)f[2 * i + 1]});
        return u;
    }
};

struct DistillArgs {
    const void* logits;
    void* grad;                 // null: the loss alone
    const void* index;          // [M][K]
    const void* teacher;        // [M][K]
    const int64_t* labels;      // null: no row has one
    const float* gscale;        // null (1), or the loss's upstream gradient
    float* rows;                // [M] loss shares
    int* counts;                // [G][2] rows with entries, rows with a label
    float* loss;
    int64_t ld, gld;
    int M, V, W, K, G;          // W: columns of the gradient (V real ones, zeros behind them)
    int dtype, index64, teacher_dtype, written;   // written: grad holds the gradient for gscale 1 already
    float tau, alpha, beta;     // beta = 1 - alpha, rounded from more than 32 bits
    uint64_t capture;           // written by every call: the graph capture that its launches belong to (0: none)
};

// the capture that a stream's launches go into: 0 for none, ~0 where that cannot be told
uint64_t capture_of(hipStream_t s) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (hipStreamGetCaptureInfo(s, &status, &id) != hipSuccess) {
        (void)hipGetLastError();
        return ~0ull;
    }
    return status == hipStreamCaptureStatusNone ? 0 : id;
}

__device__ __forceinline__ int entry_at(const DistillArgs& a, int64_t i) {   // -1 where unused
    if (a.index64) {
        const int64_t v = ((const int64_t*)a.index)[i];
        return v >= 0 && v < a.V ? (int)v : -1;
    }
    const int v = ((const int*)a.index)[i];
    return v >= 0 && v < a.V ? v : -1;
}
__device__ __forceinline__ float teacher_at(const DistillArgs& a, int64_t i) {
    if (a.teacher_dtype == 0) return ((const float*)a.teacher)[i];
    const uint16_t v = ((const uint16_t*)a.teacher)[i];
    return a.teacher_dtype == 1 ? bf2f(v) : (float)__builtin_bit_cast(_Float16, v);
}
__device__ __forceinline__ int label_of(const DistillArgs& a, int row) {
    if (a.labels == nullptr) return -1;
    const int64_t l = a.labels[row];
    return l >= 0 && l < a.V ? (int)l : -1;
}

// Workgroup g counts every G-th row's flags: rows with an entry, rows with a label.
__global__ __launch_bounds__(256) void distill_count_kernel(const DistillArgs a) {
    __shared__ int red[2][4];
    int nt = 0, nl = 0;
    for (int row = blockIdx.x * 256 + threadIdx.x; row < a.M; row += gridDim.x * 256) {
        bool any = false;
        for (int k = 0; k < a.K && !any; ++k) any = entry_at(a, (int64_t)row * a.K + k) >= 0;   // usually the first
        nt += any;
        nl += label_of(a, row) >= 0;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        nt += __shfl_xor(nt, o, 64);
        nl += __shfl_xor(nl, o, 64);
    }
    if ((threadIdx.x & 63) == 0) {
        red[0][threadIdx.x >> 6] = nt;
        red[1][threadIdx.x >> 6] = nl;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        int t = 0;
        for (int w = 0; w < 4; ++w) t += red[threadIdx.x][w];
        a.counts[2 * blockIdx.x + threadIdx.x] = t;
    }
}

// Adds the rows' shares (fixed order: thread t takes rows 4 t .. 4 t + 3 of every 4096; then a tree).
__global__ __launch_bounds__(1024) void distill_loss_kernel(const float* __restrict__ rows, float* __restrict__ loss, int M) {
    __shared__ float red[16];
    float s = 0.f;
    const int whole = M & ~4095;
    int i = threadIdx.x * 4;
#pragma unroll 4
    for (; i < whole; i += 4096) {
        const float4 v = *(const float4*)(rows + i);
        s += (v.x + v.y) + (v.z + v.w);
    }
    for (int r = whole + threadIdx.x; r < M; r += 1024) s += rows[r];
    s = block_sum(s, red);
    if (threadIdx.x == 0) *loss = s;
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// a value that all lanes hold alike, kept in a scalar register
__device__ __forceinline__ float uniform(float x) {
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x)));
}
__device__ __forceinline__ float zero_if_none(float m) { return m == -INFINITY ? 0.f : m; }
// Opaque to the optimiser: a piece stays packed (4 registers) between the passes and is unpacked in
// each, instead of living as 8 floats across them.
template <int N>
__device__ __forceinline__ void keep_packed(u32x4 (&q)[N]) {
#pragma unroll
    for (int t = 0; t < N; ++t) asm volatile("" : "+v"(q[t]));
}

// The two softmaxes of a row, 2^(d ct) and 2^(d log2 e) for d = z - (some maximum).  MODE -1: no
// cross-entropy, the first alone.  An exponential issues for 8 cycles where a product takes 4, so where
// the temperature allows the second one is a power of the first, e^d = (e^(d / tau))^tau: MODE 1, 2, 4
// for those temperatures.  MODE 0, any other one, takes both.
// The distance is taken before its product: a fma of z c with the rounded m c would leave that rounding,
// 2^-24 of |m c|, in the exponent, which differs from wave to wave and grows with the row's shift without
// bound (a row of bf16's lowest values: infinite).
template <class T, int MODE>
struct Soft {
    float ct;
    static __device__ __forceinline__ float one(float f, float m, float c) {
        return exp2_((f - m) * c);
    }
    // t = 2^((f - m) ct), o = 2^((f - m) log2 e)
    __device__ __forceinline__ void operator()(float f, float m, float& t, float& o) const {
        t = one(f, m, ct);
        if (MODE == 0) o = one(f, m, 1.4426950408889634f);
        else if (MODE > 0) o = MODE == 1 ? t : MODE == 2 ? t * t : (t * t) * (t * t);
    }
};

// NT threads a row.  NV: 16-byte pieces of the row per thread that stay in registers; 0: the row streams
// through twice.
template <class T, int NT, int NV, int MODE, bool GRAD>
__global__ __launch_bounds__(NT, 4) void distill_kernel(const DistillArgs a) {
    constexpr int E = T::E, NW = NT / 64, UN = 4;
    constexpr bool MIX = MODE >= 0;   // the cross-entropy term takes part (beta > 0)
    constexpr float L2E = 1.4426950408889634f;
    typedef typename T::S S;
    // the row's entries 0 .. K - 1, and its label as entry K: index, (t - max) / tau, e^that, logit
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ float red[NW][3];
    __shared__ float tred[3];
    __shared__ int cnt[2];
    int* sidx = (int*)smem;
    float* su = (float*)(sidx + a.K + 1);
    float* se = su + a.K + 1;
    float* sz = se + a.K + 1;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float gs = a.gscale != nullptr ? *a.gscale : 1.f;
    if (a.written && gs == 1.f) return;   // the forward wrote this gradient already
    if (w == 0) {   // the counts of the whole batch
        int nt = 0, nl = 0;
        for (int g = lane; g < a.G; g += 64) {
            nt += a.counts[2 * g];
            nl += a.counts[2 * g + 1];
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            nt += __shfl_xor(nt, o, 64);
            nl += __shfl_xor(nl, o, 64);
        }
        if (lane == 0) {
            cnt[0] = nt;
            cnt[1] = nl;
        }
    }
    const Soft<T, MODE> soft{L2E / a.tau};
    const float it = 1.f / a.tau;
    for (int row = blockIdx.x; row < a.M; row += gridDim.x) {
        const S* z = (const S*)a.logits + (int64_t)row * a.ld;
        // whole 16-byte pieces from the first boundary on; the elements before and behind them (less
        // than a piece each) are held by threads 0 and 1
        const int skew = (int)(((uintptr_t)z & 15) / sizeof(S));
        const int a0 = min(skew ? E - skew : 0, a.V), np = (a.V - a0) / E, a1 = a0 + np * E;
        const int e0 = tid == 0 ? 0 : a1, e1 = tid == 0 ? a0 : tid == 1 ? a.V : a1;   // this thread's edge elements
        const u32x4* zp = (const u32x4*)(z + a0);
        u32x4 q[NV > 0 ? NV : 1], qe;
#pragma unroll
        for (int t = 0; t < NV; ++t) {
            const int p = tid + t * NT;
            if (p < np) q[t] = zp[p];
        }
        {
            float f[E];
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] = e0 + i < e1 ? T::get(z[e0 + i]) : -INFINITY;
            qe = T::pack(f);   // exact: the values come from this type
        }
        // ---- the last wave takes the teacher's entries
        if (w == NW - 1) {
            float tm = -INFINITY, nan = 0.f, any = 0.f;
            for (int k = lane; k < a.K; k += 64) {
                const int64_t at = (int64_t)row * a.K + k;
                const int i = entry_at(a, at);
                const float t = i >= 0 ? teacher_at(a, at) : -INFINITY;
                sidx[k] = i;
                su[k] = t;
                sz[k] = i >= 0 ? T::get(z[i]) : 0.f;
                tm = fmaxf(tm, t);
                nan += t == t ? 0.f : 1.f;
                any += i >= 0 ? 1.f : 0.f;
            }
            tm = wave_max(tm);
            float ts = 0.f;
            for (int k = lane; k < a.K; k += 64) {
                const float u = (su[k] - tm) * it, e = su[k] == -INFINITY ? 0.f : __expf(u);
                su[k] = u;
                se[k] = e;
                ts += e;
            }
            ts = wave_sum(ts);
            nan = wave_sum(nan);
            any = wave_sum(any);
            if (lane == 0) {
                const int l = MIX ? label_of(a, row) : -1;
                sidx[a.K] = l;
                se[a.K] = 0.f;
                sz[a.K] = l >= 0 ? T::get(z[l]) : 0.f;
                tred[0] = nan > 0.f ? __uint_as_float(0x7fc00000u) : ts;
                tred[1] = any;
            }
        }
        // ---- the row's maximum and sums, each wave with its own maximum, joined through LDS
        float m = -INFINITY, st = 0.f, s1 = 0.f;
        auto top = [&](const u32x4& u) {
            float f[E];
            T::unpack(u, f);
            float t = f[0];
#pragma unroll
            for (int i = 1; i < E; ++i) t = fmaxf(t, f[i]);
            return t;
        };
        auto sums = [&](const u32x4& u, float mz) {
            float f[E], at = 0.f, a1_ = 0.f;
            T::unpack(u, f);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                float t, o = 0.f;
                soft(f[i], mz, t, o);
                at += t;
                a1_ += o;
            }
            st += at;
            if (MIX) s1 += a1_;
            asm volatile("" : "+v"(st), "+v"(s1));   // a piece is added before the next one's values are made
        };
        auto rescale = [&](float d) {   // the sums, taken against a maximum, against one higher by -d
            st *= exp2_(d * soft.ct);
            if (MIX) s1 *= exp2_(d * L2E);
        };
        if constexpr (NV > 0) {
            m = top(qe);
#pragma unroll
            for (int t = 0; t < NV; ++t) {
                if (tid + t * NT < np) m = fmaxf(m, top(q[t]));
                __builtin_amdgcn_sched_barrier(0);
            }
            keep_packed(q);
            m = wave_max(m);
            const float mz = zero_if_none(m);
            if (e0 < e1) sums(qe, mz);
#pragma unroll
            for (int t = 0; t < NV; ++t)
                if (tid + t * NT < np) sums(q[t], mz);
            keep_packed(q);
        } else {
            // running maximum of the wave; the sums are rescaled where it rises (seldom after the first
            // pieces), except from -infinity, where they are zero still.  The maximum is taken across lanes, so
            // every lane of a wave makes every trip; one without a piece of its own brings -infinity.  UN
            // loads of a thread in flight: the row streams through few registers
            auto take = [&](u32x4 (&u)[UN], int n) {
                float t = m;
#pragma unroll
                for (int x = 0; x < UN; ++x)
                    if (x < n) t = fmaxf(t, top(u[x]));
                if (__any(t > m)) {
                    t = wave_max(t);
                    if (m != -INFINITY) rescale(m - t);
                    m = t;
                }
                const float mz = zero_if_none(m);
                keep_packed(u);
#pragma unroll
                for (int x = 0; x < UN; ++x)
                    if (x < n) sums(u[x], mz);
            };
            float none_[E];
#pragma unroll
            for (int i = 0; i < E; ++i) none_[i] = -INFINITY;
            const u32x4 none = T::pack(none_);
            u32x4 u[UN];
            int p = tid;
            for (; p - lane + 63 + (UN - 1) * NT < np; p += UN * NT) {
#pragma unroll
                for (int x = 0; x < UN; ++x) u[x] = zp[p + x * NT];
                take(u, UN);
            }
            for (; p - lane < np; p += NT) {
                u[0] = none;
                if (p < np) u[0] = zp[p];
                take(u, 1);
            }
            if (w == 0) {   // (the edge elements are lanes 0 and 1)
                u[0] = qe;
                take(u, 1);
            }
        }
        st = wave_sum(st);
        if (MIX) s1 = wave_sum(s1);
        if (lane == 0) {
            red[w][0] = m;
            red[w][1] = st;
            red[w][2] = s1;
        }
        __syncthreads();
        // every wave joins the waves' sums, one per lane of a group of NW, in the same order
        const float mw = red[lane % NW][0];
        float M = mw;
#pragma unroll
        for (int o = NW / 2; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
        const float dw = mw == -INFINITY ? 0.f : mw - M;
        float S_t = red[lane % NW][1] * exp2_(dw * soft.ct), S_1 = MIX ? red[lane % NW][2] * exp2_(dw * L2E) : 0.f;
#pragma unroll
        for (int o = NW / 2; o > 0; o >>= 1) {
            S_t += __shfl_xor(S_t, o, 64);
            if (MIX) S_1 += __shfl_xor(S_1, o, 64);
        }
        M = uniform(M);
        S_t = uniform(S_t);
        S_1 = uniform(S_1);
        const float ts = uniform(tred[0]);
        // (no finite entry: nothing to learn from; NaN counts as one)
        const bool live = uniform(tred[1]) > 0.f && ts != 0.f && a.alpha > 0.f;
        const int label = MIX ? __builtin_amdgcn_readfirstlane(sidx[a.K]) : -1;
        const float n_t = uniform((float)max(cnt[0], 1)), n_l = uniform((float)max(cnt[1], 1));
        const float qt = live ? 1.f / ts : 0.f;
        const float gt = live ? a.alpha * a.tau / n_t * gs : 0.f, g1 = label >= 0 ? a.beta / n_l * gs : 0.f;
        // ---- loss share: the wave that holds the entries
        if (a.rows != nullptr && w == NW - 1) {
            float kd = 0.f;
            if (live) {
                const float base = logf(S_t) - logf(ts);   // u - log sum e^u - (d / tau - log S_t)
                for (int k = lane; k < a.K; k += 64) {
                    const float e = se[k];
                    if (e != 0.f) kd += e * qt * (su[k] - (sz[k] - M) * it + base);   // 0 log 0 = 0
                }
                kd = wave_sum(kd);
            }
            if (lane == 0) {
                float v = live ? a.alpha * a.tau * a.tau * kd / n_t : 0.f;
                if (label >= 0) v += a.beta / n_l * (logf(S_1) - (sz[a.K] - M));
                a.rows[row] = v;
            }
        }
        if constexpr (GRAD) {
            const float wt = gt / S_t, w1 = MIX ? g1 / S_1 : 0.f;
            const bool no_t = gt == 0.f, no_1 = g1 == 0.f;   // a row without the term: exactly none of it
            auto dz = [&](const float (&f)[E], float (&g)[E]) {
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    float t, o;
                    soft(f[i], M, t, o);
                    g[i] = no_t ? 0.f : wt * t;
                    if (MIX) g[i] = no_1 ? g[i] : fmaf(w1, o, g[i]);
                }
            };
            S* g = (S*)a.grad + (int64_t)row * a.gld;
            u32x4* gp = (u32x4*)(g + a0);   // (the host gives the gradient's rows the logits' alignment)
            auto store = [&](int p, const u32x4& u) {
                float f[E], d[E];
                T::unpack(u, f);
                dz(f, d);
                __builtin_nontemporal_store(T::pack(d), gp + p);
                __builtin_amdgcn_sched_barrier(0);
            };
            if constexpr (NV > 0) {
#pragma unroll
                for (int t = 0; t < NV; ++t)
                    if (tid + t * NT < np) store(tid + t * NT, q[t]);
            } else {
                u32x4 u[UN];
                int p = tid;
                for (; p + (UN - 1) * NT < np; p += UN * NT) {
#pragma unroll
                    for (int x = 0; x < UN; ++x) u[x] = zp[p + x * NT];
#pragma unroll
                    for (int x = 0; x < UN; ++x) store(p + x * NT, u[x]);
                }
                for (; p < np; p += NT) store(p, zp[p]);
            }
            if (e0 < e1) {
                float f[E], d[E];
                T::unpack(qe, f);
                dz(f, d);
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (e0 + i < e1) g[e0 + i] = T::put(d[i]);
            }
            for (int j = a.V + tid; j < a.W; j += NT) g[j] = T::put(0.f);
            __syncthreads();   // the special columns are written after the row
            for (int k = tid; k <= a.K; k += NT) {
                const int i = sidx[k];
                if (i < 0 || (k == a.K && !MIX)) continue;
                float wq = 0.f;
                bool first = true;
                for (int x = 0; x < a.K; ++x) {
                    const bool same = sidx[x] == i;
                    if (same && x < k) first = false;
                    if (same) wq += se[x];
                }
                if (!first) continue;
                float f[E], d[E];
                f[0] = sz[k];
#pragma unroll
                for (int y = 1; y < E; ++y) f[y] = 0.f;
                dz(f, d);
                g[i] = T::put(d[0] - (no_t ? 0.f : gt * (wq * qt)) - (i == label ? g1 : 0.f));
            }
        }
        __syncthreads();   // the next row's entries and sums replace this one's in LDS
    }
}

template <class T, int NT, int NV, int MODE>
int launch_mode(const DistillArgs& a, hipStream_t s) {
    const size_t lds = (size_t)(a.K + 1) * 16;
    // one workgroup a row (up to what a launch takes, 2^32 threads less one); the pass that most often has nothing
    // to do (written) as few as fill the chip
    const int most = a.written ? 1024 : 1 << 21, grid = a.M < most ? a.M : most;
    if (a.grad != nullptr) distill_kernel<T, NT, NV, MODE, true><<<grid, NT, lds, s>>>(a);
    else distill_kernel<T, NT, NV, MODE, false><<<grid, NT, lds, s>>>(a);
    return (int)hipGetLastError();
}

template <class T, int NT, int NV>
int launch(const DistillArgs& a, hipStream_t s) {
    if (!(a.beta > 0.f)) return launch_mode<T, NT, NV, -1>(a, s);
    if (a.tau == 1.f) return launch_mode<T, NT, NV, 1>(a, s);
    if (a.tau == 2.f) return launch_mode<T, NT, NV, 2>(a, s);
    if (a.tau == 4.f) return launch_mode<T, NT, NV, 4>(a, s);
    return launch_mode<T, NT, NV, 0>(a, s);
}

template <class T>
int by_length(const DistillArgs& a, hipStream_t s) {
    const int np = a.V / T::E;   // whole pieces, at most
    if (np <= 256) return launch<T, 64, 4>(a, s);
    if (np <= 1024) return launch<T, 256, 4>(a, s);
    // long rows: where there are rows for every CU twice over, workgroups of 4 waves that stream, 5 rows in
    // flight a CU, mix their loads, sums and stores best (16384 x 50304 bf16: 806 us; 1024 threads with
    // the row in registers, one row in flight: 1260 us); fewer rows want the whole workgroup on one
    // row (24 rows: 12.6 against 15.1 us)
    if (np <= 8192 && a.M < 512) return launch<T, 1024, 8>(a, s);
    return launch<T, 256, 0>(a, s);
}

}  // namespace

// args: DistillArgs.  rows not null: counts, loss rows, loss and (grad not null) the gradient.  rows
// null: the gradient alone, from counts that an earlier call left.
// written, with the capture of the call that wrote: it is believed only where both calls run eagerly or are nodes of one
// graph.  A graph of the gradient alone is replayed without that call, over what the last replay and its
// user left in grad.
TDL_API int tdl_distill(void* args, hipStream_t s) {
    const uint64_t capture = capture_of(s), before = ((DistillArgs*)args)->capture;
    ((DistillArgs*)args)->capture = capture;
    DistillArgs a = *(const DistillArgs*)args;
    if (capture != before || capture == ~0ull) a.written = 0;
    if (a.M <= 0 || a.M >= MAX_DIM || a.V <= 0 || a.W < a.V || a.W >= MAX_DIM || a.K <= 0 || a.K > MAX_K || a.G <= 0 || a.dtype < 0 || a.dtype > 2 || !(a.tau > 0.f) ||
        !(a.alpha >= 0.f && a.alpha <= 1.f) ||
        !(a.beta >= 0.f && a.beta <= 1.f) || (a.beta > 0.f && a.labels == nullptr) || (a.rows == nullptr && a.grad == nullptr))
        return (int)hipErrorInvalidValue;
    if (a.rows != nullptr) {
        distill_count_kernel<<<a.G, 256, 0, s>>>(a);
        const int rc = (int)hipGetLastError();
        if (rc) return rc;
    }
    const int rc = a.dtype == 0 ? by_length<F32>(a, s) : a.dtype == 1 ? by_length<B16>(a, s) : by_length<H16>(a, s);
    if (rc || a.rows == nullptr) return rc;
    distill_loss_kernel<<<1, 1024, 0, s>>>(a.rows, a.loss, a.M);
    TDL_LAUNCH_CHECK();
}

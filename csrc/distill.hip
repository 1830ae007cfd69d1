// Distillation from a teacher's top logits, mixed with cross-entropy: loss and gradient in one pass over
// the student's logits.
//
//   q   = softmax over a row's teacher entries of t / tau            p_tau = softmax_j(z / tau),  p = softmax_j(z)
//   kd  = tau^2 sum_k q_k (log q_k - log p_tau(i_k))                 ce = -log p(label)
//   loss = alpha mean_kd + (1 - alpha) mean_ce    (means over the rows that have entries / a label)
//   dz_j = alpha tau / n_t (p_tau_j - sum_{k : i_k = j} q_k) + (1 - alpha) / n_l (p_j - [j = label])
//
// A row belongs to one workgroup that keeps it in REGISTERS between the statistics and the gradient, so
// memory sees the logits once and the gradient once: the bound.  1024 threads hold a row of 50304
// 16-bit logits in 7 16-byte registers each; two such workgroups fit a CU, one loading while the other
// stores.  Rows too long for the registers are read a second time.
//
// The gradient at a row's few special columns (its teacher entries and label) is written over the
// row's stores by threads that own an entry, from the same fp32 terms and with one rounding: the
// lowest entry of several with the same index sums them in order, so no atomics, no fixed order lost.
#include "common.h"

namespace {

constexpr int MAX_K = 1024;
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
};

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

// Adds the rows' shares (fixed order: thread t takes rows t, t + 1024, ...; then a tree).
__global__ __launch_bounds__(1024) void distill_loss_kernel(const float* __restrict__ rows, float* __restrict__ loss, int M) {
    __shared__ float red[16];
    float s = 0.f;
    for (int i = threadIdx.x; i < M; i += 1024) s += rows[i];
    s = block_sum(s, red);
    if (threadIdx.x == 0) *loss = s;
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Opaque to the optimiser: a piece stays packed (4 registers) between the passes and is unpacked in
// each, instead of living as 8 floats across them.
template <int N>
__device__ __forceinline__ void keep_packed(u32x4 (&q)[N]) {
#pragma unroll
    for (int t = 0; t < N; ++t) asm volatile("" : "+v"(q[t]));
}

// the unpacked values of a piece die before the next piece's are made
__device__ __forceinline__ void one_at_a_time() { __builtin_amdgcn_sched_barrier(0); }

// NV: 16-byte pieces of the row per thread that stay in registers (0: the row is read twice).
// MIX: the cross-entropy term takes part (beta > 0).
template <class T, int NT, int NV, bool MIX, bool GRAD>
__global__ __launch_bounds__(NT, NV <= 8 ? 8 : 4) void distill_kernel(const DistillArgs a) {
    constexpr int E = T::E, NW = NT / 64;
    typedef typename T::S S;
    extern __shared__ __attribute__((aligned(16))) char smem[];   // K entries: index, then weight
    __shared__ float red[NW][3];
    __shared__ float tred[4];
    __shared__ int cnt[2];
    int* sidx = (int*)smem;
    float* sq = (float*)(sidx + a.K);
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const float gs = a.gscale != nullptr ? *a.gscale : 1.f;
    if (a.written && gs == 1.f) return;   // the forward wrote this gradient already
    if (tid < 64) {   // the counts of the whole batch
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
    for (int row = blockIdx.x; row < a.M; row += gridDim.x) {
        const S* z = (const S*)a.logits + (int64_t)row * a.ld;
        // whole 16-byte pieces from the first boundary on; the elements before and behind them (less
        // than a piece each) are held by threads 0 and 1
        const int skew = (int)(((uintptr_t)z & 15) / sizeof(S));
        const int a0 = min(skew ? E - skew : 0, a.V), np = (a.V - a0) / E, a1 = a0 + np * E;
        const int e0 = tid == 0 ? 0 : a1, e1 = tid == 0 ? a0 : tid == 1 ? a.V : a1;   // this thread's edge elements
        auto load = [&](int p) { return *(const u32x4*)(z + a0 + (int64_t)p * E); };
        u32x4 q[NV > 0 ? NV : 1], qe;
#pragma unroll
        for (int t = 0; t < NV; ++t) {
            const int p = tid + t * NT;
            if (p < np) q[t] = load(p);
        }
        {
            float f[E];
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] = e0 + i < e1 ? T::get(z[e0 + i]) : -INFINITY;
            qe = T::pack(f);   // exact: the values come from this type
        }
        // ---- the last wave takes the teacher's entries: sum of e^(t - max), weights to LDS
        const int label = MIX ? label_of(a, row) : -1;
        if (w == NW - 1) {
            float tm = -INFINITY;
            for (int k = lane; k < a.K; k += 64) {
                const int64_t at = (int64_t)row * a.K + k;
                const int i = entry_at(a, at);
                const float t = i >= 0 ? teacher_at(a, at) : -INFINITY;
                sidx[k] = i;
                sq[k] = t;
                tm = t == t ? fmaxf(tm, t) : t;
            }
            float any = 0.f, nan = tm == tm ? 0.f : 1.f;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                nan += __shfl_xor(nan, o, 64);
                tm = fmaxf(tm, __shfl_xor(tm, o, 64));
            }
            float ts = 0.f;
            const float c = 1.f / a.tau;
            for (int k = lane; k < a.K; k += 64) {
                const float e = sq[k] == -INFINITY ? 0.f : __expf((sq[k] - tm) * c);
                any += sidx[k] >= 0 ? 1.f : 0.f;
                ts += e;
            }
            ts = wave_sum(ts);
            any = wave_sum(any);
            if (lane == 0) {
                tred[0] = tm;
                tred[1] = nan > 0.f ? __uint_as_float(0x7fc00000u) : ts;
                tred[2] = any;
            }
        }
        // ---- the row's maximum and sums of 2^((z - max) log2(e) / tau) and 2^((z - max) log2(e)); each wave
        // with its own maximum, joined through LDS
        const float L2E = 1.4426950408889634f;
        const float ct = L2E / a.tau;
        float m = -INFINITY;
        auto top = [&](const u32x4& u) {
            float f[E];
            T::unpack(u, f);
#pragma unroll
            for (int i = 0; i < E; ++i) m = fmaxf(m, f[i]);
        };
        top(qe);
        if constexpr (NV > 0) {
#pragma unroll
            for (int t = 0; t < NV; ++t) {
                if (tid + t * NT < np) top(q[t]);
                one_at_a_time();
            }
            keep_packed(q);
        } else {
            for (int p = tid; p < np; p += NT) top(load(p));
        }
        m = wave_max(m);
        const float mz = m == -INFINITY ? 0.f : m;
        float st = 0.f, s1 = 0.f;
        auto sums = [&](const u32x4& u) {
            float f[E];
            T::unpack(u, f);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float d = f[i] - mz;
                st += exp2_(d * ct);
                if (MIX) s1 += exp2_(d * L2E);
            }
        };
        if (e0 < e1) sums(qe);
        if constexpr (NV > 0) {
#pragma unroll
            for (int t = 0; t < NV; ++t) {
                if (tid + t * NT < np) sums(q[t]);
                one_at_a_time();
            }
            keep_packed(q);
        } else {
            for (int p = tid; p < np; p += NT) sums(load(p));
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
        float S_t = red[lane % NW][1] * exp2_(dw * ct), S_1 = MIX ? red[lane % NW][2] * exp2_(dw * L2E) : 0.f;
#pragma unroll
        for (int o = NW / 2; o > 0; o >>= 1) {
            S_t += __shfl_xor(S_t, o, 64);
            if (MIX) S_1 += __shfl_xor(S_1, o, 64);
        }
        const bool has = tred[2] > 0.f, lab = MIX && label >= 0;
        const float tm = tred[0], ts = tred[1];
        const float n_t = (float)max(cnt[0], 1), n_l = (float)max(cnt[1], 1);
        const float lt = logf(S_t), l1 = MIX ? logf(S_1) : 0.f;   // log sums above the maximum M
        const float qt = has && ts != 0.f ? 1.f / ts : 0.f;       // (no finite entry: nothing to learn from)
        const float live = has && ts != 0.f && a.alpha > 0.f ? 1.f : 0.f;
        const float gt = live * a.alpha * a.tau / n_t * gs, g1 = lab ? a.beta / n_l * gs : 0.f;
        const float it = 1.f / a.tau;
        // ---- loss share: the wave that holds the entries
        if (a.rows != nullptr && w == NW - 1) {
            float kd = 0.f;
            for (int k = lane; k < a.K && live != 0.f; k += 64) {
                const int i = sidx[k];
                if (i < 0 || sq[k] == -INFINITY) continue;
                const float u = (sq[k] - tm) * it;
                const float wq = __expf(u) * qt;
                const float lp = (T::get(z[i]) - M) * it - lt;
                if (wq != 0.f) kd += wq * ((u - logf(ts)) - lp);   // 0 log 0 = 0
            }
            kd = wave_sum(kd);
            if (lane == 0) {
                float v = live != 0.f ? a.alpha * a.tau * a.tau * kd / n_t : 0.f;
                if (lab) v += a.beta / n_l * (l1 - (T::get(z[label]) - M));
                a.rows[row] = v;
            }
        }
        if constexpr (GRAD) {
            // p as 2^((z - M) c - log2 S): the factors 1 / S and the means' weights multiply outside
            const float wt = gt / S_t, w1 = MIX ? g1 / S_1 : 0.f;
            const bool do_t = gt != 0.f || gt != gt, do_1 = MIX && g1 != 0.f;
            auto dz = [&](float v) {
                const float d = v - M;
                float g = do_t ? wt * exp2_(d * ct) : 0.f;
                if (MIX && do_1) g += w1 * exp2_(d * L2E);
                return g;
            };
            // this thread's special columns (entries tid, tid + NT, ...; the label as entry K): read before
            // the row is overwritten (grad may be the logits)
            constexpr int NE = (MAX_K + 1 + NT - 1) / NT;
            float zs[NE];
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                const int k = tid + e * NT;
                const int i = k < a.K ? sidx[k] : k == a.K ? label : -1;
                zs[e] = i >= 0 ? T::get(z[i]) : 0.f;
            }
            __syncthreads();
            S* g = (S*)a.grad + (int64_t)row * a.gld;
            auto store = [&](int p, const u32x4& u) {
                float f[E];
                T::unpack(u, f);
#pragma unroll
                for (int i = 0; i < E; ++i) f[i] = dz(f[i]);
                *(u32x4*)(g + a0 + (int64_t)p * E) = T::pack(f);   // (the host gives grad rows the logits' alignment)
            };
            if constexpr (NV > 0) {
#pragma unroll
                for (int t = 0; t < NV; ++t) {
                    if (tid + t * NT < np) store(tid + t * NT, q[t]);
                    one_at_a_time();
                }
            } else {
                for (int p = tid; p < np; p += NT) store(p, load(p));
            }
            if (e0 < e1) {
                float f[E];
                T::unpack(qe, f);
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (e0 + i < e1) g[e0 + i] = T::put(dz(f[i]));
            }
            for (int j = a.V + tid; j < a.W; j += NT) g[j] = T::put(0.f);
            __syncthreads();   // the special columns are written after the row
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                const int k = tid + e * NT;
                const int i = k < a.K ? sidx[k] : k == a.K ? label : -1;
                if (i < 0) continue;
                float wq = 0.f;
                bool first = true;
                for (int x = 0; x < a.K; ++x) {
                    const bool same = sidx[x] == i;
                    if (same && x < k) first = false;
                    if (same && sq[x] != -INFINITY) wq += __expf((sq[x] - tm) * it);
                }
                if (!first) continue;
                g[i] = T::put(dz(zs[e]) - gt * (wq * qt) - (i == label ? g1 : 0.f));
            }
        }
        __syncthreads();   // the next row's entries and sums replace this one's in LDS
    }
}

template <class T, int NT, int NV>
int launch(const DistillArgs& a, hipStream_t s) {
    const size_t lds = (size_t)a.K * 8;
    const bool mix = a.beta > 0.f;
    // one workgroup a row; the pass that most often has nothing to do (written) as few as fill the chip
    const int grid = a.written && a.M > 1024 ? 1024 : a.M;
    if (a.grad != nullptr) {
        if (mix) distill_kernel<T, NT, NV, true, true><<<grid, NT, lds, s>>>(a);
        else distill_kernel<T, NT, NV, false, true><<<grid, NT, lds, s>>>(a);
    } else {
        if (mix) distill_kernel<T, NT, NV, true, false><<<grid, NT, lds, s>>>(a);
        else distill_kernel<T, NT, NV, false, false><<<grid, NT, lds, s>>>(a);
    }
    return (int)hipGetLastError();
}

template <class T>
int by_length(const DistillArgs& a, hipStream_t s) {
    const int np = a.V / T::E;   // whole pieces, at most
    if (np <= 256) return launch<T, 256, 1>(a, s);
    if (np <= 1024) return launch<T, 256, 4>(a, s);
    if (np <= 4096) return launch<T, 1024, 4>(a, s);
    if (np <= 8192) return launch<T, 1024, 8>(a, s);
    if (np <= 16384) return launch<T, 1024, 16>(a, s);
    return launch<T, 1024, 0>(a, s);
}

}  // namespace

// args: DistillArgs.  rows not null: counts, loss rows, loss and (grad not null) the gradient.  rows
// null: the gradient alone, from counts that an earlier call left.
TDL_API int tdl_distill(const void* args, hipStream_t s) {
    const DistillArgs& a = *(const DistillArgs*)args;
    if (a.M <= 0 || a.V <= 0 || a.W < a.V || a.K <= 0 || a.K > MAX_K || a.G <= 0 || a.dtype < 0 || a.dtype > 2 || !(a.tau > 0.f) ||
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

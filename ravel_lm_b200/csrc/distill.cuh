// distill.cuh -- distillation from a teacher's top logits, forward and backward.
//
// A row has the student's logits s over the vocabulary and k teacher entries (id_j, t_j).  An entry
// is live when its id lies in the vocabulary and t_j is not -inf.  Over the live ones
// p = softmax(t / tau); with lse = log sum_v exp(s_v / tau):
//
//   loss  = tau^2 sum_j p_j (log p_j - s[id_j] / tau + lse)       (tau^2 KL(teacher || student))
//   d s_v = u tau (exp(s_v / tau - lse) - sum_{j: id_j = v} p_j)  (u: the row's upstream gradient)
//
// A row without a live entry has loss 0 and gradient 0 and is not counted by the mean.
//
//   k_distill_count  rows with a live entry (integers: any order gives the same sum).
//   k_distill        a block per row.  One pass over the logits keeps a running maximum and sum
//                    (base 2: exp2 of one fused multiply-add per element); with GRAD a second pass
//                    writes the gradient for upstream 1 while the row is still in L2, then the at
//                    most k entries are written once more with their p, from float32.
//   k_distill_bwd    the second pass alone, for any upstream gradient.
//   k_distill_total  the rows' losses added in a fixed order.
// Bound by HBM: one read of the logits, and one write of the gradient.
#pragma once

#include "colsum.cuh"
#include "host.cuh"
#include "norm.cuh"

namespace ravel {

struct DistillArgs {
    const void* s;            // [R, V], rows lds apart
    const void* ids;          // [R, k] int32 or int64
    const void* t;            // [R, k] teacher logits
    void* grad;               // [R, V] contiguous, or null
    float* losses;            // [R]
    float2* stat;             // [R] (m, l): m the largest s_v c, l = sum_v 2^(s_v c - m), c = log2(e) / tau
    const unsigned int* count;  // rows counted by the mean, or null (sum, none)
    const float* up;          // upstream gradient: one value (mean, sum) or [R]
    int up_rows;              // up has one value per row
    int done;                 // grad already holds the gradient of upstream 1
    int64_t R, lds;
    int V, k;
    int ids64;
    float tau, weight;
    unsigned int* err;
};

template <typename TT>
__device__ __forceinline__ bool distill_entry(const DistillArgs& a, int64_t row, int j, int& id, float& t, bool& bad) {
    const int64_t i = row * a.k + j;
    const int64_t v = a.ids64 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
    t = as_float(static_cast<const TT*>(a.t)[i]);
    bad = v >= a.V;  // negative: an empty entry; past the vocabulary: an error, taken as empty
    id = static_cast<int>(v);
    return v >= 0 && !bad && t != -INFINITY;
}

// A block per 8 rows (a warp each).
template <typename TT>
__global__ void __launch_bounds__(256) k_distill_count(const DistillArgs a, unsigned int* count) {
    __shared__ unsigned int n;
    grid_wait();
    grid_trigger();
    if (threadIdx.x == 0) n = 0u;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    const int64_t nw = static_cast<int64_t>(gridDim.x) * 8;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); row < a.R; row += nw) {
        bool any = false;
        for (int j = lane; j < a.k; j += 32) {
            int id;
            float t;
            bool bad;
            any |= distill_entry<TT>(a, row, j, id, t, bad);
        }
        if (__any_sync(0xffffffffu, any) && lane == 0) atomicAdd(&n, 1u);
    }
    __syncthreads();
    if (threadIdx.x == 0 && n != 0u) atomicAdd(count, n);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Running (maximum, sum of 2^(x - maximum)); an empty one is (-inf, 0).
struct MaxSum {
    float m, l;
};
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b) {
    const float m = fmaxf(a.m, b.m), r = finite_ref(m);
    return {m, a.l * ex2(a.m - r) + b.l * ex2(b.m - r)};
}

template <int TH>
__device__ __forceinline__ MaxSum block_join(MaxSum v, MaxSum* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        MaxSum w = {__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.l, o)};
        v = join(v, w);
    }
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < TH / 32; ++w) v = join(v, red[w]);
    return v;
}

// The row's elements as this block's threads share them: a head and a tail of single elements and
// 16-byte vectors between (rows need not start on 16 bytes).
template <typename T>
struct RowSplit {
    int head, vecs;  // elements before the first vector; vectors
    __device__ __forceinline__ RowSplit(const T* row, int n) {
        constexpr int E = 16 / sizeof(T);
        const int off = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
        head = off == 0 ? 0 : E - off;
        if (head > n) head = n;
        vecs = (n - head) / E;
    }
};

// Teacher entries into shared memory: p_j (0 for a dead entry) and ids (-1 for a dead one).  Every
// thread gets whether the row has a live entry, and (thread 0 only) the loss.
template <typename T, typename TT>
__device__ __forceinline__ bool distill_teacher(const DistillArgs& a, int64_t row, MaxSum st, bool want_loss,
                                                float* sp, int* sid, float* sred, float& loss) {
    // warp 0 alone: k is small next to the vocabulary
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        const float c = 1.4426950408889634f / a.tau;  // log2(e) / tau
        float m = -INFINITY;
        bool live = false, bad_any = false;
        for (int j = lane; j < a.k; j += 32) {
            int id;
            float t;
            bool bad;
            const bool ok = distill_entry<TT>(a, row, j, id, t, bad);
            bad_any |= bad;
            sid[j] = ok ? id : -1;
            sp[j] = ok ? t * c : -INFINITY;
            live |= ok;
            if (ok) m = fmaxf(m, t * c);
        }
        if (bad_any) atomicOr(a.err, RAVEL_DEVERR_INDEX);
        live = __any_sync(0xffffffffu, live);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        float z = 0.0f;
        for (int j = lane; j < a.k; j += 32)
            if (sid[j] >= 0) z += ex2(sp[j] - m);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
        const float lz = m + __log2f(z), iz = 1.0f / z, ll = __log2f(st.l);
        float acc = 0.0f;
        for (int j = lane; j < a.k; j += 32) {
            if (sid[j] < 0) {
                sp[j] = 0.0f;
                continue;
            }
            const float lp = sp[j] - lz, p = ex2(sp[j] - m) * iz;
            if (want_loss && p != 0.0f) {
                const float sv = as_float(static_cast<const T*>(a.s)[row * a.lds + sid[j]]);
                acc += p * (lp + ll - fmaf(sv, c, -st.m));  // base 2; p = 0 contributes nothing
            }
            sp[j] = p;
        }
        if (want_loss) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
            loss = live ? acc * 0.6931471805599453f * a.tau * a.tau * a.weight : 0.0f;
        }
        if (lane == 0) sred[0] = live ? 1.0f : 0.0f;
    }
    __syncthreads();
    return sred[0] != 0.0f;
}

// grad row = gs * (2^(s c - m) / l - p at the entries); a row without a live entry gets zeros.
template <typename T, int TH>
__device__ __forceinline__ void distill_grad_row(const DistillArgs& a, int64_t row, MaxSum st, float gs, bool live,
                                                 const float* sp, const int* sid) {
    constexpr int E = 16 / sizeof(T);
    const T* const s = static_cast<const T*>(a.s) + row * a.lds;
    T* const d = static_cast<T*>(a.grad) + row * a.V;
    const float c = 1.4426950408889634f / a.tau;
    const RowSplit<T> rs(d, a.V);
    // vectors when the logits' row is aligned like the gradient's
    const bool same = ((reinterpret_cast<uintptr_t>(s) ^ reinterpret_cast<uintptr_t>(d)) & 15u) == 0;
    if (!live) {
        const T zero = round_to<T>(0.0f);
        for (int i = threadIdx.x; i < rs.vecs; i += TH)
            *reinterpret_cast<uint4*>(d + rs.head + i * E) = make_uint4(0u, 0u, 0u, 0u);
        for (int i = threadIdx.x; i < rs.head; i += TH) d[i] = zero;
        for (int i = rs.head + rs.vecs * E + threadIdx.x; i < a.V; i += TH) d[i] = zero;
        return;
    }
    const float gl = gs / st.l;
    auto one = [&](T v) { return round_to<T>(gl * ex2(fmaf(as_float(v), c, -st.m))); };
    if (same) {
#pragma unroll 4
        for (int i = threadIdx.x; i < rs.vecs; i += TH) {
            float f[E];
            to_floats<T, E>(load_pack<T, E>(s + rs.head + i * E), f);
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = gl * ex2(fmaf(f[e], c, -st.m));
            store_pack<T, E>(d + rs.head + i * E, from_floats<T, E>(f));
        }
        for (int i = threadIdx.x; i < rs.head; i += TH) d[i] = one(s[i]);
        for (int i = rs.head + rs.vecs * E + threadIdx.x; i < a.V; i += TH) d[i] = one(s[i]);
    } else {
        for (int i = threadIdx.x; i < a.V; i += TH) d[i] = one(s[i]);
    }
    __syncthreads();  // the entries' elements are written again, by other threads
    for (int j = threadIdx.x; j < a.k; j += TH) {
        const int id = sid[j];
        if (id < 0) continue;
        float p = 0.0f;
        bool first = true;  // of the entries that name this id
        for (int i = 0; i < a.k; ++i) {
            if (sid[i] != id) continue;
            if (i < j) first = false;
            p += sp[i];
        }
        if (first) d[id] = round_to<T>(gl * ex2(fmaf(as_float(s[id]), c, -st.m)) - gs * p);
    }
}

template <typename T, typename TT, int TH, bool GRAD>
__global__ void __launch_bounds__(TH) k_distill(const DistillArgs a) {
    constexpr int E = 16 / sizeof(T);
    extern __shared__ float dyn[];  // p [k], ids [k]
    __shared__ MaxSum red[TH / 32];
    __shared__ float sred[1];
    float* const sp = dyn;
    int* const sid = reinterpret_cast<int*>(dyn + a.k);
    grid_wait();
    grid_trigger();
    const int64_t row = blockIdx.x;
    const T* const s = static_cast<const T*>(a.s) + row * a.lds;
    const float c = 1.4426950408889634f / a.tau;
    const RowSplit<T> rs(s, a.V);
    MaxSum v = {-INFINITY, 0.0f};
    auto take = [&](float x) {
        const float x2 = x * c;
        if (x2 > v.m) {
            v.l *= ex2(v.m - x2);
            v.m = x2;
        }
        v.l += ex2(fmaf(x, c, -finite_ref(v.m)));
    };
#pragma unroll 4
    for (int i = threadIdx.x; i < rs.vecs; i += TH) {
        float x[E], m = -INFINITY;
        to_floats<T, E>(load_pack<T, E>(s + rs.head + i * E), x);
#pragma unroll
        for (int e = 0; e < E; ++e) m = fmaxf(m, x[e]);
        m *= c;
        if (m > v.m) {
            v.l *= ex2(v.m - m);
            v.m = m;
        }
        const float r = finite_ref(v.m);
#pragma unroll
        for (int e = 0; e < E; ++e) v.l += ex2(fmaf(x[e], c, -r));
    }
    for (int i = threadIdx.x; i < rs.head; i += TH) take(as_float(s[i]));
    for (int i = rs.head + rs.vecs * E + threadIdx.x; i < a.V; i += TH) take(as_float(s[i]));
    v = block_join<TH>(v, red);
    float loss = 0.0f;
    const bool live = distill_teacher<T, TT>(a, row, v, true, sp, sid, sred, loss);
    if (threadIdx.x == 0) {
        a.losses[row] = loss;
        if (a.stat != nullptr) a.stat[row] = make_float2(v.m, v.l);
    }
    if constexpr (GRAD) {
        const float n = a.count != nullptr ? fmaxf(static_cast<float>(*a.count), 1.0f) : 1.0f;
        distill_grad_row<T, TH>(a, row, v, a.weight * a.tau / n, live, sp, sid);
    }
}

template <typename T, typename TT, int TH>
__global__ void __launch_bounds__(TH) k_distill_bwd(const DistillArgs a) {
    extern __shared__ float dyn[];
    __shared__ float sred[1];
    float* const sp = dyn;
    int* const sid = reinterpret_cast<int*>(dyn + a.k);
    grid_wait();
    grid_trigger();
    if (a.done && *a.up == 1.0f) return;
    const float n = a.count != nullptr ? fmaxf(static_cast<float>(*a.count), 1.0f) : 1.0f;
    for (int64_t row = blockIdx.x; row < a.R; row += gridDim.x) {
        const float2 f = a.stat[row];
        const MaxSum st = {f.x, f.y};
        float unused;
        const bool live = distill_teacher<T, TT>(a, row, st, false, sp, sid, sred, unused);
        distill_grad_row<T, TH>(a, row, st, a.up[a.up_rows ? row : 0] * a.weight * a.tau / n, live, sp, sid);
        __syncthreads();
    }
}

// out = sum of the losses (/ count): one block, a fixed order.
__global__ void __launch_bounds__(1024) k_distill_total(const float* __restrict__ losses, int64_t R,
                                                        const unsigned int* __restrict__ count,
                                                        float* __restrict__ out) {
    __shared__ float2 red[64];
    int turn = 0;
    grid_wait();
    grid_trigger();
    float s = 0.0f;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < R; i += 1024) s += losses[i];
    s = group_sum2<32>(s, 0.0f, red, turn).x;
    if (threadIdx.x == 0) out[0] = count != nullptr ? s / fmaxf(static_cast<float>(*count), 1.0f) : s;
}

}  // namespace ravel

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
//   k_distill_count  rows with a live entry, counted before a gradient of the mean is written.
//   k_distill        a block per row.  One pass over the logits keeps a running maximum and sum
//                    (base 2: exp2 of (s - max) log2(e) / tau, subtracted before it is scaled, so that a row of the
//                    type's lowest or highest values does not leave float32 and a common offset costs nothing.
//                    In pairs; one fused multiply-add an element, which fails there, was 0 to 5% faster: 8192 x 65536
//                    bf16 179 / 181 us, with the gradient 440 / 442, 16384 x 4096 85 / 89); with GRAD a second pass
//                    writes the gradient for upstream 1 while the row is still in registers (up to 8 KB)
//                    or L2, then the at most k entries are written once more with their p, from float32.
//   k_distill_bwd    the second pass alone, for any upstream gradient.
//   k_distill_total  the rows' losses added in a fixed order.
// Bound by HBM: one read of the logits, and one write of the gradient.
#pragma once

#include "colsum.cuh"
#include "host.cuh"
#include "norm.cuh"

namespace ravel {

// Rows longer than this are dropped from L2 as the second pass reads them: the rows in flight (8 or 4 an SM) then
// take more than half of it, and a third of the second reads went to memory.  With the gradient, us without and with:
// 8192 rows of 128 KB 468 / 438, 4096 of 196 KB 392 / 344, 8192 of 62 KB 230 / 217, 16384 of 32 KB 206 / 223.
constexpr int64_t DISTILL_DROP_BYTES = 48 * 1024;
constexpr int DISTILL_COUNTS = 256;  // blocks of k_distill_count

struct DistillArgs {
    const void* s;            // [R, V], rows lds apart
    const void* ids;          // [R, k] int32 or int64
    const void* t;            // [R, k] teacher logits
    void* grad;               // [R, V] contiguous, or null
    float* losses;            // [R]
    float2* stat;             // [R] (m, l): m the largest s_v, l = sum_v 2^((s_v - m) c), c = log2(e) / tau
    unsigned char* live;      // [R] the row has a live entry, or null
    const unsigned int* counts;  // [DISTILL_COUNTS] rows counted by the mean, in parts; null: sum, none
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

// counts[block] = the rows with a live entry among the block's (a warp per row).
template <typename TT>
__global__ void __launch_bounds__(256) k_distill_count(const DistillArgs a, unsigned int* counts) {
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
    if (threadIdx.x == 0) counts[blockIdx.x] = n;
}

// What the mean divides by, by one warp: all of it where a.counts is null.
__device__ __forceinline__ float distill_counted(const DistillArgs& a) {
    if (a.counts == nullptr) return 1.0f;
    unsigned int n = 0u;
    for (int i = threadIdx.x & 31; i < DISTILL_COUNTS; i += 32) n += a.counts[i];
    n = __reduce_add_sync(0xffffffffu, n);
    return fmaxf(static_cast<float>(n), 1.0f);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// x[i] = (x[i] - m) c for an even number of elements, two an instruction.
template <int E>
__device__ __forceinline__ void sub_scale(float (&x)[E], float m, float c) {
    uint64_t m2, c2;
    asm("mov.b64 %0, {%1, %1};" : "=l"(m2) : "f"(-m));
    asm("mov.b64 %0, {%1, %1};" : "=l"(c2) : "f"(c));
#pragma unroll
    for (int e = 0; e < E; e += 2)
        asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%0, %1};\n\tadd.rn.f32x2 t, t, %2;\n\tmul.rn.f32x2 t, t, %3;\n\t"
            "mov.b64 {%0, %1}, t;\n\t}"
            : "+f"(x[e]), "+f"(x[e + 1])
            : "l"(m2), "l"(c2));
}

// Running (maximum, sum of 2^((x - maximum) c)); an empty one is (-inf, 0).
struct MaxSum {
    float m, l;
};
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.0f : m; }
// The warp's (maximum, sum): the maxima first, then one rescaling of each lane's sum.
__device__ __forceinline__ MaxSum warp_join(MaxSum v, float c) {
    float m = v.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float l = v.l * ex2((v.m - finite_ref(m)) * c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    return {m, l};
}
template <int TH>
__device__ __forceinline__ MaxSum block_join(MaxSum v, float c, MaxSum* red) {
    v = warp_join(v, c);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    v = {-INFINITY, 0.0f};
    if (lane < TH / 32) v = red[lane];
    return warp_join(v, c);
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

// Teacher entries into shared memory, by one warp: ids (-1 for a dead entry), p_j (0 for a dead one); for the
// loss log2 p_j (-inf) in its place, and s[id_j].  Returns whether the row has a live entry.
template <typename T, typename TT>
__device__ __forceinline__ bool distill_teacher(const DistillArgs& a, int64_t row, bool want_loss, float* sp, int* sid,
                                                float* ss) {
    const int lane = threadIdx.x & 31;
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
        sp[j] = ok ? t : -INFINITY;
        if (want_loss) ss[j] = ok ? as_float(static_cast<const T*>(a.s)[row * a.lds + id]) : 0.0f;
        live |= ok;
        if (ok) m = fmaxf(m, t);
    }
    if (bad_any) atomicOr(a.err, RAVEL_DEVERR_INDEX);
    live = __any_sync(0xffffffffu, live);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float z = 0.0f;
    for (int j = lane; j < a.k; j += 32)
        if (sid[j] >= 0) z += ex2((sp[j] - m) * c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    const float lz = log2f(z);
    for (int j = lane; j < a.k; j += 32) {
        const float lp = sid[j] >= 0 ? fmaf(sp[j] - m, c, -lz) : -INFINITY;
        sp[j] = want_loss ? lp : ex2(lp);
    }
    return live;
}

// The row's loss from those and the student's (m, l), by the same warp; leaves p_j in the place of log2 p_j.
// An entry's term is p (log p - (s - m) / tau + log l): natural units, which hold a student's logit of the type's
// lowest value for tau >= 1.
__device__ __forceinline__ float distill_loss(const DistillArgs& a, MaxSum st, float* sp, const float* ss) {
    const float ll = log2f(st.l), it = 1.0f / a.tau;
    float acc = 0.0f;
    for (int j = threadIdx.x & 31; j < a.k; j += 32) {
        const float lp = sp[j], p = ex2(lp);
        if (p != 0.0f) acc += p * fmaf(lp + ll, 0.6931471805599453f, (st.m - ss[j]) * it);  // p = 0 contributes nothing
        sp[j] = p;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    return acc * a.tau * a.tau * a.weight;
}

// grad row = gs * (2^((s - m) c) / l - p at the entries); a row without a live entry gets zeros.  The row's vectors are
// in v (NV > 0: vector i * TH + thread in v[i]) or read again.
template <typename T, int TH, int NV>
__device__ __forceinline__ void distill_grad_row(const DistillArgs& a, int64_t row, MaxSum st, float gs, bool live,
                                                 const float* sp, const int* sid, const Pack<T, 16 / sizeof(T)>* v) {
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
    auto one = [&](T x) { return round_to<T>(gl * ex2((as_float(x) - st.m) * c)); };
    if (same) {
        auto put = [&](int i, const Pack<T, E>& x) {
            float f[E];
            to_floats<T, E>(x, f);
            sub_scale<E>(f, st.m, c);
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = gl * ex2(f[e]);
            store_pack_stream<T, E>(d + rs.head + i * E, from_floats<T, E>(f));
        };
        if constexpr (NV > 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (threadIdx.x + i * TH < rs.vecs) put(threadIdx.x + i * TH, v[i]);
        } else if (static_cast<int64_t>(a.V) * sizeof(T) > DISTILL_DROP_BYTES) {
#pragma unroll 4
            for (int i = threadIdx.x; i < rs.vecs; i += TH) put(i, load_pack_last<T, E>(s + rs.head + i * E));
        } else {
#pragma unroll 4
            for (int i = threadIdx.x; i < rs.vecs; i += TH) put(i, load_pack<T, E>(s + rs.head + i * E));
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
        if (first) d[id] = round_to<T>(gl * ex2((as_float(s[id]) - st.m) * c) - gs * p);
    }
}

// NV > 0: the row's vectors (at most NV * TH) stay in registers between the passes.
template <typename T, typename TT, int TH, int NV, bool GRAD>
__global__ void __launch_bounds__(TH) k_distill(const DistillArgs a) {
    constexpr int E = 16 / sizeof(T);
    extern __shared__ float dyn[];  // p [k], ids [k], the entries' logits [k]
    __shared__ MaxSum red[TH / 32];
    __shared__ float s_live, s_count;
    float* const sp = dyn;
    int* const sid = reinterpret_cast<int*>(dyn + a.k);
    float* const ss = dyn + 2 * a.k;
    grid_wait();
    grid_trigger();
    const int64_t row = blockIdx.x;
    const T* const s = static_cast<const T*>(a.s) + row * a.lds;
    const float c = 1.4426950408889634f / a.tau;
    const RowSplit<T> rs(s, a.V);
    Pack<T, E> held[NV > 0 ? NV : 1];
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (threadIdx.x + i * TH < rs.vecs) held[i] = load_pack<T, E>(s + rs.head + (threadIdx.x + i * TH) * E);
    }
    // the teacher's part first: its chain of loads runs under the other warps' pass over the logits
    if (threadIdx.x < 32) {
        const bool live = distill_teacher<T, TT>(a, row, true, sp, sid, ss);
        if (threadIdx.x == 0) s_live = live ? 1.0f : 0.0f;
    } else if (GRAD && threadIdx.x < 64) {
        const float n = distill_counted(a);
        if (threadIdx.x == 32) s_count = n;
    }
    MaxSum v = {-INFINITY, 0.0f};
    auto add = [&](const Pack<T, E>& p) {
        float x[E], m = -INFINITY;
        to_floats<T, E>(p, x);
#pragma unroll
        for (int e = 0; e < E; ++e) m = fmaxf(m, x[e]);
        if (m > v.m) {
            v.l *= ex2((v.m - m) * c);
            v.m = m;
        }
        sub_scale<E>(x, finite_ref(v.m), c);
#pragma unroll
        for (int e = 0; e < E; ++e) v.l += ex2(x[e]);
    };
    auto take = [&](float x) {
        if (x > v.m) {
            v.l *= ex2((v.m - x) * c);
            v.m = x;
        }
        v.l += ex2((x - finite_ref(v.m)) * c);
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (threadIdx.x + i * TH < rs.vecs) add(held[i]);
    } else {
#pragma unroll 4
        for (int i = threadIdx.x; i < rs.vecs; i += TH) add(load_pack<T, E>(s + rs.head + i * E));
    }
    for (int i = threadIdx.x; i < rs.head; i += TH) take(as_float(s[i]));
    for (int i = rs.head + rs.vecs * E + threadIdx.x; i < a.V; i += TH) take(as_float(s[i]));
    v = block_join<TH>(v, c, red);
    const bool live = s_live != 0.0f;
    if (threadIdx.x < 32) {
        const float loss = live ? distill_loss(a, v, sp, ss) : 0.0f;
        if (threadIdx.x == 0) {
            a.losses[row] = loss;
            if (a.live != nullptr) a.live[row] = live;
            if (a.stat != nullptr) a.stat[row] = make_float2(v.m, v.l);
        }
    }
    if constexpr (GRAD) distill_grad_row<T, TH, NV>(a, row, v, a.weight * a.tau / s_count, live, sp, sid, held);
}

// 32 registers, so that an SM is full: 16384 x 8192 bf16 125 us without the bound, 98 with it.
template <typename T, typename TT, int TH>
__global__ void __launch_bounds__(TH, 2048 / TH) k_distill_bwd(const DistillArgs a) {
    extern __shared__ float dyn[];
    __shared__ float s_live, s_count;
    float* const sp = dyn;
    int* const sid = reinterpret_cast<int*>(dyn + a.k);
    grid_wait();
    grid_trigger();
    if (a.done && *a.up == 1.0f) return;
    for (int64_t row = blockIdx.x; row < a.R; row += gridDim.x) {
        if (threadIdx.x < 32) {
            const bool live = distill_teacher<T, TT>(a, row, false, sp, sid, nullptr);
            if (threadIdx.x == 0) s_live = live ? 1.0f : 0.0f;
        } else if (threadIdx.x < 64) {
            const float n = distill_counted(a);
            if (threadIdx.x == 32) s_count = n;
        }
        __syncthreads();
        const float2 f = a.stat[row];
        distill_grad_row<T, TH, 0>(a, row, {f.x, f.y}, a.up[a.up_rows ? row : 0] * a.weight * a.tau / s_count,
                                   s_live != 0.0f, sp, sid, nullptr);
        __syncthreads();
    }
}

// out = sum of the losses (MEAN: / the live rows): one block, a fixed order.
template <bool MEAN>
__global__ void __launch_bounds__(1024) k_distill_total(const float* __restrict__ losses,
                                                        const unsigned char* __restrict__ live, int64_t R,
                                                        float* __restrict__ out) {
    __shared__ float2 red[64];
    int turn = 0;
    grid_wait();
    grid_trigger();
    float s = 0.0f, n = 0.0f;  // at most R / 1024 rows a thread: exact
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < R; i += 1024) {
        s += losses[i];
        if (MEAN && live[i]) n += 1.0f;
    }
    const float2 t = group_sum2<32>(s, n, red, turn);
    if (threadIdx.x == 0) out[0] = MEAN ? t.x / fmaxf(t.y, 1.0f) : t.x;
}

}  // namespace ravel

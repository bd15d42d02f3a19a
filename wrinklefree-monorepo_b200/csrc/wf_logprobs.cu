// Log probabilities of given tokens, the entropy and the most likely alternatives of rows of logits, in one pass over them, and the gradient.
//
//   m = max x,  r = m log2 e (rounded),  s = sum 2^d,  t = sum d 2^d  with d = x log2 e - r:   log2 p_j = d_j - log2 s,   H = ln 2 (log2 s - t / s)
//
// HBM bounds many rows: each logit is read once, 11.6 of them per cycle and SM in bf16 at the measured rate, next to 16 exponentials that the SM can
// compute in it and about 128 instructions, of which one logit takes 6.5: pairs of fp32 go through one instruction where there is one (fma, add).  d is
// one fma, so r may be rounded (the sums are in terms of r as it is): d of the maximum is then what the rounding left of it, at most 2^-4 up to |m| = 2^20.  It grows
// with |m| and passes what 2^d can hold from 2^31 on, so beyond 2^20, as in rows masked throughout by a constant, d is (x - m) log2 e.
// Every thread keeps its own sums over its share of the row, in terms of a reference that is renewed where an element is LP_AHEAD in front of it (with the
// maximum itself one of 32 threads nearly always has to), and at the end in terms of the largest; they are joined then.  Batches come through a ring of
// each thread's own in shared memory.
//
// Alternatives: a candidate is a 64-bit key, the value's bits in the order of whole numbers above the inverted index, so that one
// comparison says which is ahead (of equal values the lower index).  Every warp keeps its 32 best, one per lane in descending order.  A bound that k elements
// of the row reach - the k-th largest of all threads' maxima over their first values, then, whenever the elements seen have doubled, of all warps'
// lists - keeps all but about k / 4 candidates per doubling from a warp's list.
//
// Rows of up to LP_SHORT elements take a warp each, longer ones a block of four.  Where rows are few, a row is cut over a cluster of blocks, and what bounds it
// is the chain of shuffles: candidates from the first bound on go to a buffer in shared memory instead (what does not fit it goes to the warps' lists), the place
// of each among them is the number of those ahead of it, and the first block finds the places of all blocks' best by searching their sorted lists.  One row of
// 128256 with twenty alternatives 10.9 us with the lists, 9.2 so (4.4 without alternatives).
//
// Measured, bf16, none / 5 / 20 / 32 alternatives in us: 4096 x 49152 (61.5 at the measured copy rate) 63 / 87 / 104 / 115, 2048 x 128256 (80.3) 84 / 97 / 112 / 121.
// On the way there: blocks of eight warps 97 without alternatives (the joins at the end of a row), no loads ahead of the batch in hand 79, sums joined
// pair by pair 72, loads ahead into registers 68, the maximum as the reference 64.5 / 90 / 106 / 116; candidates put into the lists from code unrolled over the
// elements 245 with five (the instructions did not fit their cache), a buffer of candidates sorted by 32 153, a bound that is not renewed 113, candidates
// picked from the registers 105.  Four batches on their way instead of two: 66 / 95.
#include <cooperative_groups.h>

#include "wf_common.cuh"

namespace wf {

namespace cg = cooperative_groups;

constexpr int LP_THREADS = 128;
constexpr int LP_WARPS = LP_THREADS / 32;
constexpr int LP_UNROLL = 4;     // 16-byte loads per thread and batch
constexpr int LP_STAGES = 3;     // batches of them: one in hand, the others on their way
constexpr int LP_CLUSTER = 8;
constexpr int LP_TOP = 32;       // alternatives at most: one per lane
constexpr int LP_SHORT = 4096;   // elements of a row that one warp takes
constexpr float LP_LN2 = 0.69314718055994531f, LP_LOG2E = 1.4426950408889634f;
constexpr float LP_LOWEST = -3.402823466e38f;
constexpr float LP_AHEAD = 5.f;                   // how far elements may be ahead of what the sums are in terms of; at the end that is the maximum
constexpr float LP_FAR = 1048576.f;               // 2^20: maxima up to here are within 2^-4 of their rounded multiple of log2 e

using Key = unsigned long long;
constexpr Key LP_FLOOR = (static_cast<Key>(0x007fffffu) << 32) | 0xffffffffu;  // above every element of -inf, below all others

__device__ __forceinline__ uint32_t lp_order(float v) {
    const uint32_t u = __float_as_uint(v + 0.f);  // -0 and 0 are equal
    return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float lp_value(uint32_t o) { return __uint_as_float(o ^ (o >> 31 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ Key lp_key(float v, int index) { return (static_cast<Key>(lp_order(v)) << 32) | (0xffffffffu - static_cast<uint32_t>(index)); }
__device__ __forceinline__ float lp_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float lp_max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float lp_element(float v) { return v; }
__device__ __forceinline__ float lp_element(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float lp_element(__half v) { return __half2float(v); }

using Pair = unsigned long long;
__device__ __forceinline__ Pair lp_pair(float a, float b) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 lp_two(Pair p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ Pair lp_fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ Pair lp_add2(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// a bit for each of eight halves of masks
__device__ __forceinline__ uint32_t lp_bits(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const uint32_t m = (a & 0x00020001u) | (b & 0x00080004u) | (c & 0x00200010u) | (d & 0x00800040u);
    return (m | m >> 16) & 0xffu;
}

// 16 bytes of logits.  EMPTY: -inf throughout; most: the largest (a NaN is not looked at); get: as fp32; near: as fp32, those below -2^100 as that (a NaN
// stays one), so that 2^d is 0 and d 2^d with it; reach: a bit for each that is `least` (a value of the type) or more; LEAST: the smallest number.
template <int DT>
struct LpVec;
template <>
struct LpVec<WF_F32> {
    static constexpr int N = 4;
    static constexpr uint32_t EMPTY = 0xff800000u;
    static constexpr float LEAST = LP_LOWEST;
    static __device__ __forceinline__ uint32_t reach(const uint4& u, float least) {
        return (__uint_as_float(u.x) >= least ? 1u : 0u) | (__uint_as_float(u.y) >= least ? 2u : 0u) | (__uint_as_float(u.z) >= least ? 4u : 0u) |
               (__uint_as_float(u.w) >= least ? 8u : 0u);
    }
    using Most = float;
    static __device__ __forceinline__ Most most(const uint4& u) {
        return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
    }
    static __device__ __forceinline__ Most larger(Most a, Most b) { return fmaxf(a, b); }
    static __device__ __forceinline__ float top(Most a) { return a; }
    static __device__ __forceinline__ void get(const uint4& u, float* f) {
        f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ void near(const uint4& u, float* f) {
        get(u, f);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = lp_max_nan(f[i], -1.2676506002282294e30f);
    }
};
template <>
struct LpVec<WF_BF16> {
    static constexpr int N = 8;
    static constexpr uint32_t EMPTY = 0xff80ff80u;
    static constexpr float LEAST = -3.3895313892515355e38f;
    static __device__ __forceinline__ __nv_bfloat162 pair(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
    static __device__ __forceinline__ uint32_t reach(const uint4& u, float least) {
        const __nv_bfloat162 l = __float2bfloat162_rn(least);
        return lp_bits(__hge2_mask(pair(u.x), l), __hge2_mask(pair(u.y), l), __hge2_mask(pair(u.z), l), __hge2_mask(pair(u.w), l));
    }
    using Most = __nv_bfloat162;
    static __device__ __forceinline__ Most most(const uint4& u) { return __hmax2(__hmax2(pair(u.x), pair(u.y)), __hmax2(pair(u.z), pair(u.w))); }
    static __device__ __forceinline__ Most larger(Most a, Most b) { return __hmax2(a, b); }
    static __device__ __forceinline__ float top(Most a) { return fmaxf(__low2float(a), __high2float(a)); }
    static __device__ __forceinline__ void get(const uint4& u, float* f) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ void near(const uint4& u, float* f) {
        const __nv_bfloat162 least = pair(0xf180f180u);  // -2^100
        const __nv_bfloat162 w[4] = {__hmax2_nan(pair(u.x), least), __hmax2_nan(pair(u.y), least), __hmax2_nan(pair(u.z), least), __hmax2_nan(pair(u.w), least)};
        get(*reinterpret_cast<const uint4*>(w), f);
    }
};
template <>
struct LpVec<WF_F16> {
    static constexpr int N = 8;
    static constexpr uint32_t EMPTY = 0xfc00fc00u;
    static constexpr float LEAST = -65504.f;
    static __device__ __forceinline__ __half2 pair(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
    static __device__ __forceinline__ uint32_t reach(const uint4& u, float least) {
        const __half2 l = __float2half2_rn(least);
        return lp_bits(__hge2_mask(pair(u.x), l), __hge2_mask(pair(u.y), l), __hge2_mask(pair(u.z), l), __hge2_mask(pair(u.w), l));
    }
    using Most = __half2;
    static __device__ __forceinline__ Most most(const uint4& u) { return __hmax2(__hmax2(pair(u.x), pair(u.y)), __hmax2(pair(u.z), pair(u.w))); }
    static __device__ __forceinline__ Most larger(Most a, Most b) { return __hmax2(a, b); }
    static __device__ __forceinline__ float top(Most a) { return fmaxf(__low2float(a), __high2float(a)); }
    static __device__ __forceinline__ void get(const uint4& u, float* f) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 v = __half22float2(pair(w[i]));
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        }
    }
    static __device__ __forceinline__ void near(const uint4& u, float* f) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // -inf is the only one below
            const float2 v = __half22float2(__hmax2_nan(pair(w[i]), pair(0xfbfffbffu)));
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        }
    }
};

// -65504 in the place of -inf: in a row whose largest element is near it d would not be far below.  Rows down there go the other way.
template <int DT>
__device__ __forceinline__ bool lp_far(float m) {
    return DT == WF_F16 ? m < -32768.f : fabsf(m) > LP_FAR;
}
// d of the maximum itself: what the rounding left of m log2 e, or nothing
template <int DT>
__device__ __forceinline__ float lp_rest(float m) {
    return lp_far<DT>(m) ? 0.f : fmaf(m, LP_LOG2E, -__fmul_rn(m, LP_LOG2E));
}

// m, s and t of a part of a row, in terms of r = m log2 e as it is rounded (of m itself where that is far)
struct LpSums {
    float m, s, t;
    // the same sums in terms of a larger maximum.  (As the difference of the rounded multiples where neither is far: two branches more, up to 1% slower.)
    template <int DT>
    __device__ __forceinline__ void raise(float to) {
        const float d = fmaf(m - to, LP_LOG2E, lp_rest<DT>(to) - lp_rest<DT>(m));
        const float f = lp_exp2(d), all = t + d * s;
        s *= f;
        t = f == 0.f ? s : f * all;  // 0, and d may be -inf; a NaN in s stays one
        m = to;
    }
    // those of all lanes, in every lane
    template <int DT>
    __device__ __forceinline__ void join() {
        float to = m;
#pragma unroll
        for (int i = 16; i > 0; i >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, i));
        raise<DT>(to);
#pragma unroll
        for (int i = 16; i > 0; i >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, i);
            t += __shfl_xor_sync(0xffffffffu, t, i);
        }
    }
};

// Descending order of one value per lane.
template <class T>
__device__ __forceinline__ T lp_sort(T a, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int s = size / 2; s > 0; s >>= 1) {
            const T o = __shfl_xor_sync(0xffffffffu, a, s);
            const bool larger = ((lane & s) == 0) == ((lane & size) == 0);
            a = (a > o) == larger ? a : o;
        }
    return a;
}
// The better 32 of two descending lists of one value per lane, descending.
template <class T>
__device__ __forceinline__ T lp_merge(T a, T b, int lane) {
    const T r = __shfl_sync(0xffffffffu, b, 31 - lane);
    a = a > r ? a : r;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
        const T o = __shfl_xor_sync(0xffffffffu, a, s);
        const bool upper = lane & s;
        a = (a > o) != upper ? a : o;
    }
    return a;
}

struct LpParams {
    const void* x;           // [R, V], stride ld
    int64_t ld;
    const int64_t* tokens;   // [R]
    float* logprob;          // [R]
    float* entropy;          // [R]
    float* stats;            // [R, 2]: m, log s (nullable)
    float* top_logprob;      // [R, top]
    int64_t* top_id;
    int64_t R;
    int V, top;
};

constexpr int LP_BUFFER = 256;  // candidates of a block of a cluster; the lists' behind them
constexpr int LP_ROUNDS = 5;    // batches of a block up to which its candidates go there (about as many as alternatives are asked for from each)

// WARPS: of a row (one, or LP_WARPS).  SPLIT: of each of a cluster's blocks.
template <int DT, bool TOP, int WARPS, bool SPLIT>
__global__ void __launch_bounds__(LP_THREADS, 7) logprobs_kernel(const LpParams p) {
    constexpr int N = LpVec<DT>::N;
    constexpr int THREADS = WARPS * 32, STEP = THREADS * LP_UNROLL;
    using T = typename Elem<DT>::type;
    __shared__ __align__(16) uint4 s_ring[LP_STAGES][LP_UNROLL][LP_THREADS];
    __shared__ uint32_t s_order[2][TOP ? LP_WARPS : 1][32];
    __shared__ Key s_list[TOP && !SPLIT ? LP_WARPS : 1][32];
    __shared__ LpSums s_sums[SPLIT ? LP_CLUSTER * LP_WARPS : LP_WARPS];  // (SPLIT: of the cluster's warps, in the first block)
    __shared__ __align__(16) Key s_buffer[TOP && SPLIT ? LP_BUFFER + LP_WARPS * 32 + 8 : 1];
    __shared__ Key s_lists[TOP && SPLIT ? LP_CLUSTER : 1][32];           // the blocks' best in order, in the first block
    __shared__ float s_row[2];
    __shared__ int s_held, s_place[LP_WARPS];
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    const int tid = threadIdx.x, block_warp = tid >> 5, lane = tid & 31, warp = WARPS == 1 ? 0 : block_warp;
    cg::cluster_group cluster = cg::this_cluster();
    const int cs = SPLIT ? static_cast<int>(cluster.num_blocks()) : 1, rank = SPLIT ? static_cast<int>(cluster.block_rank()) : 0;
    if constexpr (SPLIT) {
        if constexpr (TOP) {
            if (tid == 0) s_held = 0;
            for (int i = tid; i < LP_CLUSTER * 32; i += LP_THREADS) s_lists[0][i] = 0;
        }
        cluster.barrier_arrive();  // the first block's shared memory is written to once all have come here
    }
    const int64_t row = WARPS == 1 ? static_cast<int64_t>(blockIdx.x) * LP_WARPS + block_warp : blockIdx.x / cs;
    if (WARPS == 1 && row >= p.R) return;
    const T* x = static_cast<const T*>(p.x) + row * p.ld;
    const int mis = static_cast<int>(reinterpret_cast<uintptr_t>(x) / sizeof(T) % N);
    const int head = min(mis ? N - mis : 0, p.V);   // elements in front of the first 16-byte boundary
    const int vecs = (p.V - head) / N, tail0 = head + vecs * N;
    const int v_lo = static_cast<int>(static_cast<int64_t>(vecs) * rank / cs), v_hi = static_cast<int>(static_cast<int64_t>(vecs) * (rank + 1) / cs);
    const T* body = x + head;

    int64_t tok = -1;
    float tok_logit = 0.f;
    if (rank == 0 && warp == 0 && lane == 0) {  // in front: two loads, one behind the other
        tok = p.tokens[row];
        if (tok >= 0 && tok < p.V) tok_logit = load1<DT>(x, tok);
    }
    float m = LP_LOWEST, largest = LP_LOWEST;  // what the sums are in terms of; their largest element
    float2 s2 = {0.f, 0.f}, t2 = {0.f, 0.f};
    auto raise = [&](float to) {
        LpSums a = {m, s2.x, t2.x}, b = {m, s2.y, t2.y};
        a.raise<DT>(to);
        b.raise<DT>(to);
        m = to;
        s2 = make_float2(a.s, b.s);
        t2 = make_float2(a.t, b.t);
    };
    auto add_far = [&](float v) {
        const float d = lp_max_nan((v - m) * LP_LOG2E, -200.f), e = lp_exp2(d);  // 2^-200 is 0, and 0 * -200 with it; -inf would not do
        s2.x += e;
        t2.x = fmaf(e, d, t2.x);
    };

    Key list = 0, bound = LP_FLOOR;
    // the lanes' keys, of those that have one ahead of the bound, into the list
    auto insert = [&](Key key, bool has) {
        uint32_t who = __ballot_sync(0xffffffffu, has && key > bound);
        if (!who) return;
        while (who) {
            const Key c = __shfl_sync(0xffffffffu, key, __ffs(who) - 1);
            who &= who - 1;
            const int ahead = __popc(__ballot_sync(0xffffffffu, list > c));
            const Key up = __shfl_up_sync(0xffffffffu, list, 1);
            list = lane < ahead ? list : (lane == ahead ? c : up);
        }
        const Key last = __shfl_sync(0xffffffffu, list, p.top - 1);
        bound = last > bound ? last : bound;
    };
    const bool buffered = SPLIT && v_hi - v_lo <= LP_ROUNDS * STEP;
    // Batches on their way: every thread's own, so that waiting for its own copies is enough
    uint4 raw[LP_UNROLL];
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(&s_ring[0][0][tid]));
    int slot = 0, ask_slot = 0;
    auto request = [&](int base) {
#pragma unroll
        for (int u = 0; u < LP_UNROLL; ++u) {
            const int i = base + warp * 32 + u * THREADS + lane;
            if (i < v_hi)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(ring + ask_slot + u * LP_THREADS * 16), "l"(body + static_cast<int64_t>(i) * N) : "memory");
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");  // one group per batch, also when empty: the wait counts stay uniform
        ask_slot = ask_slot == (LP_STAGES - 1) * LP_UNROLL * LP_THREADS * 16 ? 0 : ask_slot + LP_UNROLL * LP_THREADS * 16;
    };
#pragma unroll
    for (int i = 0; i < LP_STAGES - 1; ++i) request(v_lo + i * STEP);
    int round = 0;
    for (int base = v_lo; round == 0 || base < v_hi; base += STEP, ++round) {  // the same number of rounds for all warps of the row
        typename LpVec<DT>::Most most[LP_UNROLL];
        request(base + (LP_STAGES - 1) * STEP);
        asm volatile("cp.async.wait_group %0;\n" ::"n"(LP_STAGES - 1) : "memory");
        const uint4(*batch)[LP_THREADS] = s_ring[slot];
        slot = slot == LP_STAGES - 1 ? 0 : slot + 1;
        if (base + STEP <= v_hi) {
#pragma unroll
            for (int u = 0; u < LP_UNROLL; ++u) raw[u] = batch[u][tid];
        } else {
#pragma unroll
            for (int u = 0; u < LP_UNROLL; ++u) {
                raw[u] = make_uint4(LpVec<DT>::EMPTY, LpVec<DT>::EMPTY, LpVec<DT>::EMPTY, LpVec<DT>::EMPTY);
                if (base + warp * 32 + u * THREADS + lane < v_hi) raw[u] = batch[u][tid];
            }
        }
#pragma unroll
        for (int u = 0; u < LP_UNROLL; ++u) most[u] = LpVec<DT>::most(raw[u]);
        static_assert(LP_UNROLL == 4, "the four maxima of a batch");
        const float top = LpVec<DT>::top(LpVec<DT>::larger(LpVec<DT>::larger(most[0], most[1]), LpVec<DT>::larger(most[2], most[3])));
        largest = fmaxf(largest, top);
        if (top > m + LP_AHEAD) raise(top);
        if (lp_far<DT>(m)) {
#pragma unroll 1
            for (int u = 0; u < LP_UNROLL; ++u) {
                uint4 one = raw[0];
#pragma unroll
                for (int w = 1; w < LP_UNROLL; ++w)
                    if (u == w) one = raw[w];
                float f[N];
                LpVec<DT>::get(one, f);
#pragma unroll
                for (int e = 0; e < N; ++e) add_far(f[e]);
            }
        } else {
            const float r = -__fmul_rn(m, LP_LOG2E);
            const Pair l2 = lp_pair(LP_LOG2E, LP_LOG2E), r2 = lp_pair(r, r);
            Pair s = lp_pair(s2.x, s2.y), t = lp_pair(t2.x, t2.y);
#pragma unroll
            for (int u = 0; u < LP_UNROLL; ++u) {
                float f[N];
                LpVec<DT>::near(raw[u], f);
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    const Pair d = lp_fma2(lp_pair(f[e], f[e + 1]), l2, r2);
                    const float2 dd = lp_two(d);
                    const Pair x2 = lp_pair(lp_exp2(dd.x), lp_exp2(dd.y));
                    s = lp_add2(s, x2);
                    t = lp_fma2(x2, d, t);
                }
            }
            s2 = lp_two(s);
            t2 = lp_two(t);
        }
        if constexpr (TOP) {
            // A new bound for all warps of the row whenever the elements seen have doubled: at first the k-th largest of the threads' maxima, then of what
            // the lists hold; k elements are at least that.
            if (round == 0 || (WARPS > 1 && !buffered && (round & (round - 1)) == 0)) {
                uint32_t o = round ? static_cast<uint32_t>(list >> 32) : lp_sort(lp_order(fmaxf(top, -INFINITY)), lane);
                if constexpr (WARPS > 1) {
#pragma unroll
                    for (int half = 1; half < WARPS; half <<= 1) {  // after these steps every warp has the best 32 of all
                        s_order[half & 1][warp][lane] = o;
                        __syncthreads();
                        o = lp_merge(o, s_order[half & 1][warp ^ half][lane], lane);
                    }
                }
                const Key start = static_cast<Key>(__shfl_sync(0xffffffffu, o, p.top - 1)) << 32;
                bound = start > bound ? start : bound;
            }
            const float least = fmaxf(lp_value(static_cast<uint32_t>(bound >> 32)), LpVec<DT>::LEAST);
            if (__any_sync(0xffffffffu, top >= least)) {
                uint32_t bits = 0;  // this lane's candidates of the batch
#pragma unroll
                for (int u = 0; u < LP_UNROLL; ++u)
                    if (__any_sync(0xffffffffu, LpVec<DT>::top(most[u]) >= least)) bits |= LpVec<DT>::reach(raw[u], least) << (u * N);
                const auto first = [&] {  // of them, read again: picked from the registers they took longer
                    const int u = (__ffs(bits) - 1) / N, e = (__ffs(bits) - 1) % N;
                    return lp_key(lp_element(reinterpret_cast<const T*>(&batch[u][tid])[e]), head + (base + warp * 32 + u * THREADS + lane) * N + e);
                };
                if (buffered && bits) {  // every lane by itself
                    for (int to = atomicAdd(&s_held, __popc(bits)); bits && to < LP_BUFFER; ++to, bits &= bits - 1) s_buffer[to] = first();
                }
#pragma unroll 1
                while (__any_sync(0xffffffffu, bits != 0)) {  // one per lane and round
                    insert(bits ? first() : 0, bits != 0);
                    bits &= bits - 1;
                }
            }
        }
    }
    if (largest > m) raise(largest);
    if (rank == 0 && warp == 0) {  // what lies in front of the first boundary and behind the last one: at most one element per lane
        const int i = lane < 16 ? lane : tail0 + lane - 16;
        const bool there = lane < 16 ? lane < head : i < p.V;
        const float v = there ? load1<DT>(x, i) : -INFINITY;
        if (v > m) raise(v);
        if (lp_far<DT>(m)) {
            add_far(v);
        } else {
            const float d = lp_max_nan(fmaf(v, LP_LOG2E, -__fmul_rn(m, LP_LOG2E)), -200.f), e = lp_exp2(d);
            s2.x += e;
            t2.x = fmaf(e, d, t2.x);
        }
        if constexpr (TOP) insert(lp_key(v, i), v > -INFINITY);
    }

    // the row's own results, by one warp whose lanes hold the sums of the whole row
    float row_m = 0.f, row_log = 0.f;
    auto finish = [&](const LpSums& a) {
        const bool empty = a.s == 0.f;  // every element is -inf
        const float log2_s = log2f(a.s);
        row_m = a.m;
        // neither is below 0 but by rounding, as where one element has all of the row: a logarithm of more than 1 or an entropy of less than nothing is no answer
        row_log = empty ? -INFINITY : lp_max_nan(LP_LN2 * (log2_s - lp_rest<DT>(a.m)), 0.f);
        if (lane == 0) {
            float lp = 0.f;
            if (tok >= p.V) lp = __uint_as_float(0x7fc00000u);
            else if (tok >= 0) lp = empty ? -INFINITY : (tok_logit - row_m) - row_log;
            p.logprob[row] = lp;
            p.entropy[row] = empty ? 0.f : lp_max_nan(LP_LN2 * (log2_s - a.t / a.s), 0.f);
            if (p.stats) {
                p.stats[2 * row] = row_m;
                p.stats[2 * row + 1] = row_log;
            }
            if (SPLIT) {
                s_row[0] = row_m;
                s_row[1] = row_log;
            }
        }
    };

    // ---- join the lanes, the warps, the blocks
    const LpSums none = {LP_LOWEST, 0.f, 0.f};
    LpSums a = {m, s2.x + s2.y, t2.x + t2.y};
    a.join<DT>();
    if constexpr (SPLIT) {
        cluster.barrier_wait();
        if (lane == 0) cluster.map_shared_rank(s_sums, 0)[rank * WARPS + warp] = a;
        if constexpr (TOP) {
            __syncthreads();
            int n = min(s_held, LP_BUFFER);
            const Key* keys = s_buffer;
            if (!buffered) {
                s_buffer[tid] = list;
                n = LP_WARPS * 32;
            } else {
                // behind the buffer's the lists' (of few elements; empty but for the edges of the row and for what did not fit the buffer)
                uint32_t in = __ballot_sync(0xffffffffu, list != 0);
                if (lane == 0) s_place[warp] = __popc(in);
                __syncthreads();
                int before = n;
                for (int w = 0; w < LP_WARPS; ++w) {
                    if (w < warp) before += s_place[w];
                    n += s_place[w];
                }
                if (list) s_buffer[before + lane] = list;  // the first lanes have them
                if (tid < 8) s_buffer[n + tid] = 0;        // up to a whole number of eight
            }
            __syncthreads();
            Key* best = cluster.map_shared_rank(&s_lists[rank][0], 0);
            for (int i = tid; i < n; i += LP_THREADS) {
                const Key key = keys[i];
                int ahead = 0;
                for (int j = 0; j < n; j += 8) {
                    ulonglong2 o[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) o[k] = *reinterpret_cast<const ulonglong2*>(keys + j + 2 * k);
#pragma unroll
                    for (int k = 0; k < 4; ++k) ahead += (o[k].x > key) + (o[k].y > key);
                }
                if (key && ahead < 32) best[ahead] = key;
            }
        }
        cluster.sync();
        if (rank != 0) return;
        if (warp == 0) {
            a = lane < cs * WARPS ? s_sums[lane] : none;
            a.join<DT>();
        }
    } else if constexpr (WARPS > 1) {
        if (lane == 0) s_sums[warp] = a;
        if constexpr (TOP) s_list[warp][lane] = list;
        __syncthreads();
        if constexpr (TOP) {
#pragma unroll
            for (int half = WARPS / 2; half > 0; half >>= 1) {
                if (warp < half) s_list[warp][lane] = list = lp_merge(list, s_list[warp + half][lane], lane);
                if (half > 1) __syncthreads();
            }
        }
        if (warp != 0) return;
        a = lane < WARPS ? s_sums[lane] : none;
        a.join<DT>();
    }
    if (!SPLIT || warp == 0) finish(a);
    if constexpr (TOP && SPLIT) {
        __syncthreads();
        // place of a key among all blocks' best: how many of each list, which descend, are ahead of it
        auto place = [&](Key key) {
            int at[LP_CLUSTER], all = 0;
#pragma unroll
            for (int r = 0; r < LP_CLUSTER; ++r) at[r] = 0;
#pragma unroll
            for (int step = 16; step > 0; step >>= 1)
#pragma unroll
                for (int r = 0; r < LP_CLUSTER; ++r) at[r] += s_lists[r][at[r] + step - 1] > key ? step : 0;
#pragma unroll
            for (int r = 0; r < LP_CLUSTER; ++r) all += at[r] + (s_lists[r][at[r]] > key);
            return all;
        };
        auto give = [&](int at, Key key) {
            p.top_id[row * p.top + at] = key ? static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(key)) : -1;
            p.top_logprob[row * p.top + at] = key ? (lp_value(static_cast<uint32_t>(key >> 32)) - s_row[0]) - s_row[1] : -INFINITY;
        };
        for (int i = tid; i < cs * 32; i += LP_THREADS) {
            const Key key = s_lists[0][i];
            if (key && i % 32 < p.top) {
                const int at = place(key);
                if (at < p.top) give(at, key);
            }
        }
        bool enough = false;
#pragma unroll
        for (int r = 0; r < LP_CLUSTER; ++r) enough = enough || s_lists[r][p.top - 1];
        if (!enough && tid < p.top && tid >= place(0)) give(tid, 0);
    } else if constexpr (TOP) {
        if (lane < p.top) {
            const bool there = list != 0;
            p.top_id[row * p.top + lane] = there ? static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(list)) : -1;
            p.top_logprob[row * p.top + lane] = there ? (lp_value(static_cast<uint32_t>(list >> 32)) - row_m) - row_log : -INFINITY;
        }
    }
}

struct LpGradParams {
    const void* x;
    int64_t ld;
    const int64_t* tokens;
    const float* stats;
    const float* entropy;
    const int64_t* top_id;
    const float *g_logprob, *g_entropy, *g_top;  // [R], [R], [R, top]; nullable
    void* dx;                // [R, V] contiguous, the type of x
    int V, top;
};
constexpr int LG_BYTES = 32768;  // of logits per block (2048 x 128256: bf16 167 us, f32 319, of 160 and 321 at the measured copy rate; 16 KB 174 and 313, one load at a time 180 and 323)

// d x_j = sum_i g_i ([j = id_i] - p_j) - g_H p_j (log p_j + H) over the token and the alternatives as id_i.  The row's part without the
// brackets' ones is written first; then the block's few elements that have some are computed again, all of them by one thread each.
template <int DT>
__global__ void __launch_bounds__(LP_THREADS) logprobs_grad_kernel(const LpGradParams p) {
    constexpr int N = LpVec<DT>::N;
    using T = typename Elem<DT>::type;
    __shared__ int64_t s_id[LP_TOP + 1];
    __shared__ float s_g[LP_TOP + 1];
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    constexpr int CHUNK = LG_BYTES / static_cast<int>(sizeof(T));
    const int chunks = (p.V - 1) / CHUNK + 1;
    const int64_t row = blockIdx.x / chunks;
    const int lo = static_cast<int>(blockIdx.x % chunks) * CHUNK, hi = min(lo + CHUNK, p.V);
    const int tid = threadIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.ld;
    T* dx = static_cast<T*>(p.dx) + row * p.V;
    const float m = p.stats[2 * row], log_s = p.stats[2 * row + 1], h = p.entropy[row], g_h = p.g_entropy ? p.g_entropy[row] : 0.f;
    if (tid <= p.top) {
        int64_t id = tid == 0 ? p.tokens[row] : p.top_id[row * p.top + tid - 1];
        if (id >= p.V) id = -1;
        const float* g = tid == 0 ? p.g_logprob : p.g_top;
        s_id[tid] = id;
        s_g[tid] = id < 0 || !g ? 0.f : (tid == 0 ? g[row] : g[row * p.top + tid - 1]);
    }
    __syncthreads();
    float total = 0.f;
    for (int i = 0; i <= p.top; ++i) total += s_g[i];
    const bool empty = log_s == -INFINITY;  // nothing to learn from
    auto one = [&](float v) {
        const float lp = lp_max_nan((v - m) - log_s, -200.f), pr = lp_exp2(lp * LP_LOG2E);
        return empty ? 0.f : -pr * (total + g_h * (lp + h));
    };
    auto put = [&](int j, float v) {
        if constexpr (DT == WF_F32) dx[j] = v;
        else if constexpr (DT == WF_BF16) dx[j] = __float2bfloat16_rn(v);
        else dx[j] = __float2half_rn(v);
    };
    const int mx = static_cast<int>(reinterpret_cast<uintptr_t>(x + lo) / sizeof(T) % N), md = static_cast<int>(reinterpret_cast<uintptr_t>(dx + lo) / sizeof(T) % N);
    const int v_lo = mx == md ? min(lo + (mx ? N - mx : 0), hi) : hi, vecs = (hi - v_lo) / N;  // whole vectors where both are aligned alike
    for (int j = lo + tid; j < v_lo; j += LP_THREADS) put(j, one(load1<DT>(x, j)));
    for (int base = tid; base < vecs; base += LP_THREADS * LP_UNROLL) {
        uint4 raw[LP_UNROLL];
#pragma unroll
        for (int u = 0; u < LP_UNROLL; ++u)
            if (base + u * LP_THREADS < vecs) raw[u] = ld16_chained(x + v_lo + (base + u * LP_THREADS) * N);
#pragma unroll
        for (int u = 0; u < LP_UNROLL; ++u) {
            const int i = base + u * LP_THREADS;
            if (i >= vecs) break;
            float f[N];
            LpVec<DT>::get(raw[u], f);
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = one(f[e]);
            uint4 w;
            if constexpr (DT == WF_F32) {
                w = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
            } else {
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (DT == WF_BF16) {
                        const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
                        o[e] = *reinterpret_cast<const uint32_t*>(&v);
                    } else {
                        const __half2 v = __floats2half2_rn(f[2 * e], f[2 * e + 1]);
                        o[e] = *reinterpret_cast<const uint32_t*>(&v);
                    }
                }
                w = make_uint4(o[0], o[1], o[2], o[3]);
            }
            *reinterpret_cast<uint4*>(dx + v_lo + i * N) = w;
        }
    }
    for (int j = v_lo + vecs * N + tid; j < hi; j += LP_THREADS) put(j, one(load1<DT>(x, j)));
    __syncthreads();
    if (tid <= p.top && !empty) {
        const int64_t id = s_id[tid];
        if (id >= lo && id < hi) {
            float g = 0.f;
            bool mine = true;  // of several entries with one index the first one writes
            for (int i = 0; i <= p.top; ++i)
                if (s_id[i] == id) {
                    g += s_g[i];
                    mine = mine && i >= tid;
                }
            if (mine) put(static_cast<int>(id), g + one(load1<DT>(x, id)));
        }
    }
}

template <int DT>
static void (*lp_kernel(int top, bool warps, bool split))(LpParams) {
    if (warps) return top ? logprobs_kernel<DT, true, 1, false> : logprobs_kernel<DT, false, 1, false>;
    if (split) return top ? logprobs_kernel<DT, true, LP_WARPS, true> : logprobs_kernel<DT, false, LP_WARPS, true>;
    return top ? logprobs_kernel<DT, true, LP_WARPS, false> : logprobs_kernel<DT, false, LP_WARPS, false>;
}

// Blocks per row: up to six per SM (seven fit; 300 rows of 49152 10.8 us, with four 14.3), at least 8 KB of a row each
static int lp_cluster(int64_t R, int64_t row_bytes) {
    int cs = 1;
    while (cs < LP_CLUSTER && R * cs * 2 <= 6LL * num_sms() && row_bytes / (cs * 2) >= 8192) cs *= 2;
    return cs;
}

}  // namespace wf

using namespace wf;

extern "C" int wf_token_logprobs(const void* x, int dtype, int64_t ld, const int64_t* tokens, float* logprob, float* entropy, float* stats, float* top_logprob, int64_t* top_id,
                                 int top, int64_t R, int64_t V, unsigned flags, void* stream) {
    WF_REQUIRE(x && tokens && logprob && entropy && (top == 0 || (top_logprob && top_id)), "wf_token_logprobs: null pointer");
    WF_REQUIRE(is_float_dtype(dtype), "wf_token_logprobs: logits must be f32, bf16 or f16");
    WF_REQUIRE(R > 0 && V > 0 && V <= 0x7fff0000LL && ld >= V && R < (1LL << 31) / LP_CLUSTER, "wf_token_logprobs: bad dimensions");
    WF_REQUIRE(top >= 0 && top <= LP_TOP, "wf_token_logprobs: 0 to %d alternatives (got %d)", LP_TOP, top);
    WF_REQUIRE(reinterpret_cast<uintptr_t>(x) % dtype_size(dtype) == 0, "wf_token_logprobs: misaligned logits");
    if (int rc = require_device()) return rc;
    LpParams p;
    p.x = x; p.ld = ld; p.tokens = tokens; p.logprob = logprob; p.entropy = entropy; p.stats = stats; p.top_logprob = top_logprob; p.top_id = top_id;
    p.R = R; p.V = static_cast<int>(V); p.top = top;
    const bool warps = V <= LP_SHORT;
    const int cs = warps ? 1 : lp_cluster(R, V * static_cast<int64_t>(dtype_size(dtype)));
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(static_cast<unsigned>(warps ? (R + LP_WARPS - 1) / LP_WARPS : R * cs));
    lc.blockDim = dim3(LP_THREADS);
    lc.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = attr;
    // Clusters are one wave: placed beside the CTAs of a predecessor that still runs they load the SMs unevenly (200 rows of 128256: 14.4 us, chained 20.5)
    lc.numAttrs = (flags & WF_FLAG_PDL) && cs == 1 ? 2 : 1;
    auto* kern = dtype == WF_F32 ? lp_kernel<WF_F32>(top, warps, cs > 1) : (dtype == WF_BF16 ? lp_kernel<WF_BF16>(top, warps, cs > 1) : lp_kernel<WF_F16>(top, warps, cs > 1));
    WF_CUDA(cudaLaunchKernelEx(&lc, kern, p));
    return WF_OK;
}

extern "C" int wf_token_logprobs_grad(const void* x, int dtype, int64_t ld, const int64_t* tokens, const float* stats, const float* entropy, const int64_t* top_id, int top,
                                      const float* g_logprob, const float* g_entropy, const float* g_top, void* dx, int64_t R, int64_t V, unsigned flags, void* stream) {
    WF_REQUIRE(x && tokens && stats && entropy && dx && (top == 0 || top_id), "wf_token_logprobs_grad: null pointer");
    WF_REQUIRE(is_float_dtype(dtype), "wf_token_logprobs_grad: logits must be f32, bf16 or f16");
    WF_REQUIRE(R > 0 && V > 0 && V <= 0x7fff0000LL && ld >= V && top >= 0 && top <= LP_TOP, "wf_token_logprobs_grad: bad dimensions");
    const int64_t chunk = LG_BYTES / static_cast<int64_t>(dtype_size(dtype)), chunks = (V + chunk - 1) / chunk;
    WF_REQUIRE(R < (1LL << 31) / chunks, "wf_token_logprobs_grad: oversized problem");
    WF_REQUIRE(reinterpret_cast<uintptr_t>(x) % dtype_size(dtype) == 0 && reinterpret_cast<uintptr_t>(dx) % dtype_size(dtype) == 0, "wf_token_logprobs_grad: misaligned logits");
    if (int rc = require_device()) return rc;
    LpGradParams p;
    p.x = x; p.ld = ld; p.tokens = tokens; p.stats = stats; p.entropy = entropy; p.top_id = top_id;
    p.g_logprob = g_logprob; p.g_entropy = g_entropy; p.g_top = g_top; p.dx = dx; p.V = static_cast<int>(V); p.top = top;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(static_cast<unsigned>(R * chunks));
    lc.blockDim = dim3(LP_THREADS);
    lc.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = attr;
    lc.numAttrs = (flags & WF_FLAG_PDL) ? 1 : 0;
    auto* kern = dtype == WF_F32 ? logprobs_grad_kernel<WF_F32> : (dtype == WF_BF16 ? logprobs_grad_kernel<WF_BF16> : logprobs_grad_kernel<WF_F16>);
    WF_CUDA(cudaLaunchKernelEx(&lc, kern, p));
    return WF_OK;
}

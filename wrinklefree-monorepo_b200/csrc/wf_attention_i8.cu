// Decode-step attention over the int8 cache: one new token per sequence, grouped-query heads, sequences of different lengths.
//
//   s[t] = scale * (q . k_codes[t]) * k_step[t]        out = softmax_t(s) @ (v_codes[t] * v_step[t])        t <= pos[b]
//
// Every code and step of the context is read once per launch and sixteen query heads of a KV head, half the bytes of a bf16 cache: HBM bounds it, as long as the SM's instructions keep
// up: 730 cycles for the 16.9 KB of 64 positions at the measured rate.  The steps never touch the codes: k_step multiplies a score, v_step a probability.
//
// Scores: q as three signed 8-bit digits of 2^23 steps of its row's maximum, so that the codes of the keys go into mma.sync.m16n8k32 as they lie in memory
// and the sums are exact.  An instruction has sixteen rows and a group of query heads at most eight: rows 0..7 hold the first digit and rows 8..15 the
// second, a second instruction the third.
// Values: p * v_step as a sum of two f16 numbers, 22 bits, in rows 0..7 and 8..15 of mma.sync.m16n8k16; the codes as f16, two at a time: byte ^ 0x80 in the
// low bits of 1024.0, less 1152.  Range: p is taken relative to 2^8 to 2^9 times its row's largest, and that is renewed when a score is ahead of it; p * v_step
// relative to the row's largest so far, at 2^3 to 2^5 of the range, and renewed when one may be 2^10 ahead.  The sum stays below 2^15 and resolves 2^-28 of the
// largest p * v_step of the row, of which half is what its position's codes cannot tell apart; p below 2^-117 of the largest is 0.  Whether to renew is asked of scores
// and steps alone, before the exponents: a row's limit for scores allows for the largest step of the tile that renewed last.  (Relative to the largest step, whatever
// its weight, other positions lost 0.4 % beside a step 2^20 ahead of theirs and everything beside one 2^28 ahead; that took 36.2 us for 32 sequences of 2048, this 36.7, and asked
// of the weights themselves it was 37.8.)
// The order of the summed axis is free as long as both operands share it: a thread reads 16 or 32 neighbouring codes of a key (q is laid out to
// match), and 8 or 16 neighbouring codes of four values, whose bytes it exchanges by pairs; no ldmatrix, which cannot split bytes.
// (Codes to bf16 by two masks and an addition for both products, and a maximum renewed for every tile: 54 us for 32 sequences of 2048, 755 instructions per
// warp and tile.)
//
// Measured (32 query and 8 KV heads of 128): 2 sequences of 65536 positions 57.8 us = 4.79 TB/s, the loops over the tiles 6.2; 32 of 2048 36.7 us (21 at the
// measured copy rate: the ranges are found in 1.3 us, the loops take 27, the joins 4); 1 of 2048 10.9 us.  A tile takes a warp 475 instructions, issued in 44% of
// the cycles: most of the waiting is for results of the instruction before.  Requests further ahead in L2, queries asked for ahead, and whole units for a CTA
// without joins were no faster.
//
// Work split: a unit is one (sequence, KV head, up to 16 of its query heads).  Where units are many, the 64-position tiles of all form one sequence that
// is cut into equal ranges, one per persistent CTA; where they are few, each is cut into pieces of its own.  Lengths are read on the device, every CTA finds its
// range by itself.  In a CTA every warp takes 16 positions of a tile through a ring of its own.  A unit that several CTAs share is joined by the last of them
// to finish (a ticket that is zero between launches): a CTA leaves at most two partial results, so the workspace depends on the device and the heads alone.
#include "wf_common.cuh"

namespace wf {

constexpr int A8_WARPS = 4;
constexpr int A8_THREADS = A8_WARPS * 32;
constexpr int A8_PART = 16;       // positions per stage of a warp's ring
constexpr int A8_TILE = A8_WARPS * A8_PART;
constexpr int A8_STAGES = 3;
constexpr int A8_SPLITS = 320;    // CTAs that a unit is cut into at most (one more where it begins inside a range)
constexpr int A8_TICKETS = 1024;  // one per CTA, and one more for the first step of a merge in two
constexpr int A8_GROUP = 12;      // partial results that are merged in that step
constexpr float A8_AHEAD = 8.f;   // log2 of how far a score may be ahead of the largest when the reference was taken
constexpr float A8_ROOM = 10.f;   // log2 of how far p * v_step may be ahead of the largest when its reference was taken
constexpr float A8_DIGITS = 127.f * 65536.f;  // the largest number of three digits whose first one is at most 127

__device__ __forceinline__ uint32_t a8_smem(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void a8_copy16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void a8_copy4(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void a8_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void a8_wait() {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}
__device__ __forceinline__ void a8_mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void a8_mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float a8_max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float a8_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
    return r;
}
// codes in bytes 0 and 2 of w as a pair of f16
__device__ __forceinline__ uint32_t a8_codes(uint32_t w) {
    const uint32_t a = (w & 0x00ff00ffu) ^ 0x64806480u, b = 0xe480e480u;  // 1152 + code, -1152
    const __half2 s = __hadd2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&s);
}
// (x, y) as a pair of f16, and what that leaves of them as another
__device__ __forceinline__ void a8_split(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}
// The three signed digits of four numbers, four to a register each
__device__ __forceinline__ void a8_digits(const float* f, float to, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = (static_cast<uint32_t>(__float2int_rn(f[i] * to)) + 0x808080u) ^ 0x808080u;  // digits from -128 on
    const uint32_t a = __byte_perm(u[0], u[1], 0x5140), b = __byte_perm(u[2], u[3], 0x5140);
    lo = __byte_perm(a, b, 0x5410);
    mid = __byte_perm(a, b, 0x7632);
    hi = __byte_perm(__byte_perm(u[0], u[1], 0x0062), __byte_perm(u[2], u[3], 0x0062), 0x5410);
}
// Byte offset of the 16-byte chunk c of row r in a tile of codes.  The eight threads of one shared-memory access read two rows and four chunks
// of keys, or four rows two apart and two neighbouring chunks of values: distinct banks in both.
template <int D>
__device__ __forceinline__ uint32_t a8_off(int r, int c) {
    if constexpr (D == 128) return static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4));
    return static_cast<uint32_t>((r >> 1) * 128 + ((((r & 1) * 4 + c) ^ (((r >> 1) & 3) * 2)) << 4));
}

// bytes of a stage: keys, values, their steps, and what the tile is
__host__ __device__ constexpr int a8_stage(int D) { return 2 * A8_PART * D + 2 * A8_PART * 4 + 16; }

struct AttnI8Params {
    const void* q;          // [B, nq * D], stride ldq
    const int8_t *k, *v;    // [B, nkv, T, D]
    const float *ks, *vs;   // [B, nkv, T]
    const int64_t* pos;     // nullable: all T positions
    void* out;              // [B, nq * D]
    float* part_o;          // [2 * CTAs, rows, D]  partial outputs, not yet divided
    float* part_ml;         // [2 * CTAs, rows, 2]  running maximum (log2 domain) and sum
    int* tickets;           // [CTAs]
    int64_t ldq;
    int pos_stride, B, nq, nkv, T;
    int G, blocks;          // query heads per KV head; units that they make
    int pieces;             // few units: a CTA's tiles are of one unit
    float scale_log2;       // softmax scale * log2(e)
};

__device__ __forceinline__ int a8_length(const AttnI8Params& p, int b) {
    if (!p.pos) return p.T;
    int64_t last;
    asm volatile("ld.global.s64 %0, [%1];\n" : "=l"(last) : "l"(p.pos + static_cast<int64_t>(b) * p.pos_stride) : "memory");
    return last < 0 ? 0 : (last < p.T ? static_cast<int>(last) + 1 : p.T);
}

// A place in the sequence of tiles: which unit, which of its tiles.
struct A8Cursor {
    int b, unit, tile, n, tiles;  // sequence, unit within it, tile within that; the sequence's positions and tiles
    __device__ bool next(const AttnI8Params& p, int units) {  // whether another unit begins
        if (++tile < tiles) return false;
        tile = 0;
        if (++unit < units) return true;
        unit = 0;
        do {  // another sequence with positions follows: callers stop at the end of their range
            if (++b >= p.B) return true;
            if (p.pos_stride) n = a8_length(p, b);
        } while (n == 0);
        tiles = (n + A8_TILE - 1) / A8_TILE;
        return true;
    }
};

// A unit that `count` CTAs from `first` on share; in the first one it may be the second of its partial results
struct A8Join {
    int b, unit, first, count, second;
};

// Four neighbouring places of row r in the order of the merge buffer, values NT apart in the head
template <int DT, int D>
__device__ __forceinline__ void a8_give(const AttnI8Params& p, int64_t out0, int r, int at, float4 v) {
    constexpr int NT = D / 8;
    const float x[4] = {v.x, v.y, v.z, v.w};
    const int64_t to = out0 + r * D + (at & 7) * NT + (at >> 3);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == WF_BF16) static_cast<__nv_bfloat16*>(p.out)[to + i * NT] = __float2bfloat16_rn(x[i]);
        else static_cast<__half*>(p.out)[to + i * NT] = __float2half_rn(x[i]);
    }
}

// `count` partial results of a unit, `step` CTAs apart from `first` on, into one: the unit's output, or the first one's place.  BATCH at a time, all their
// loads in flight.  (One value per load and weights in shared memory first: 14 us for 28 results of 4 rows, 65 for 128 of 16.)
template <int DT, int D, int MT, bool LAST, int BATCH>
__device__ __forceinline__ void a8_merge(const AttnI8Params& p, const A8Join& j, int first, int step, int count) {
    constexpr int ROWS = 8 * MT;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvh = j.unit / p.blocks, h0 = (j.unit - kvh * p.blocks) * ROWS, slots = min(ROWS, p.G - h0) * (D / 4);
    const int64_t out0 = static_cast<int64_t>(j.b) * p.nq * D + (static_cast<int64_t>(kvh) * p.G + h0) * D;
    const int64_t part0 = 2 * static_cast<int64_t>(first) * ROWS, stride = 2 * step * ROWS, late0 = j.second && first == j.first ? ROWS : 0;
    for (int base = warp * 32; base < slots; base += A8_THREADS) {  // a row's values are one warp's, or half of one
        const bool live = base + lane < slots;
        const int slot = live ? base + lane : 0, r = slot / (D / 4), at = slot % (D / 4) * 4;
        float4 acc = {0.f, 0.f, 0.f, 0.f};
        float top = -INFINITY, l = 0.f;
#pragma unroll 1
        for (int sp = 0; sp < count; sp += BATCH) {
            float4 v[BATCH];
            float2 ml[BATCH];
            float to = top;
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                const int64_t from = part0 + (sp + k ? min(sp + k, count - 1) * stride : late0) + r;
                ml[k] = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + from);
                v[k] = __ldcg(reinterpret_cast<const float4*>(p.part_o + from * D + at));
            }
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                if (sp + k >= count) ml[k] = make_float2(-INFINITY, 0.f);
                to = fmaxf(to, ml[k].x);
            }
            const float corr = top == -INFINITY ? 0.f : a8_exp2(top - to);
            top = to;
            l *= corr;
            acc.x *= corr; acc.y *= corr; acc.z *= corr; acc.w *= corr;
#pragma unroll
            for (int k = 0; k < BATCH; ++k) {
                if (ml[k].y != 0.f) {  // no NaN is left out: a part of nothing else has a sum of that beside a maximum of -inf
                    const float f = ml[k].x == -INFINITY ? 0.f : a8_exp2(ml[k].x - to);
                    l += ml[k].y * f;
                    acc.x += v[k].x * f; acc.y += v[k].y * f; acc.z += v[k].z * f; acc.w += v[k].w * f;
                }
            }
        }
        __syncwarp();  // the first one's maximum and sum are overwritten
        if (!live) continue;
        if constexpr (LAST) {
            a8_give<DT, D>(p, out0, r, at, make_float4(acc.x / l, acc.y / l, acc.z / l, acc.w / l));
        } else {
            *reinterpret_cast<float4*>(p.part_o + (part0 + late0 + r) * D + at) = acc;
            if (at == 0) *reinterpret_cast<float2*>(p.part_ml + (part0 + late0 + r) * 2) = make_float2(top, l);
        }
    }
}

// The units that this CTA shares with others, two at most: the last of each unit's CTAs to come here merges their results.  Where a thread would load more
// than 32, groups of CTAs merge theirs first.
template <int DT, int D, int MT>
__device__ __forceinline__ void a8_join(const AttnI8Params& p, const A8Join* joins, int n, volatile int* s_last) {
    constexpr int ROWS = 8 * MT;
    const int tid = threadIdx.x, cta = static_cast<int>(blockIdx.x);
    auto two = [&](const A8Join& j) { return j.count > A8_GROUP && j.count * max(min(ROWS, p.G) * (D / 4), A8_THREADS) > 32 * A8_THREADS; };
    // Whether this is the last of `count` CTAs.  A shared unit is the last one of its first CTA's range: no other has that number, nor one of those up to
    // its last CTA.
    auto last = [&](int ticket, int count) {
        const bool is = atomicAdd(p.tickets + ticket, 1) == count - 1;
        if (is) p.tickets[ticket] = 0;
        return is;
    };
    int out = 0;  // units whose group is not complete yet, a bit each
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        const A8Join j = joins[i];
        if (!two(j)) continue;
        const int group = (cta - j.first) / A8_GROUP, first = j.first + group * A8_GROUP, count = min(A8_GROUP, j.count - group * A8_GROUP);
        if (count == 1) continue;  // one CTA left over: where it is the next unit's first, the ticket is that unit's
        __threadfence();
        __syncthreads();
        if (tid == 0) s_last[0] = last(A8_TICKETS + first, count);
        __syncthreads();
        if (s_last[0]) {
            __threadfence();
            a8_merge<DT, D, MT, false, A8_GROUP>(p, j, first, 1, count);
        } else {
            out |= 1 << i;
        }
    }
    __threadfence();
    __syncthreads();
    if (tid < n) {  // both at once: one after the other 38.5 us for 32 sequences of 2048
        const A8Join j = joins[tid];
        s_last[tid] = !(out >> tid & 1) && last(j.first, two(j) ? (j.count + A8_GROUP - 1) / A8_GROUP : j.count);
    }
    __syncthreads();
    __threadfence();
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        const A8Join j = joins[i];
        const int step = two(j) ? A8_GROUP : 1;
        if (s_last[i]) {
            const int count = (j.count + step - 1) / step;
            // batches of few or of all: with eight always 37.0 us for 32 sequences of 2048 (two or three results each) instead of 36.5, 8 of 20000 with 16 query
            // heads 32.6 instead of 29.3
            if (count <= 4) a8_merge<DT, D, MT, true, 4>(p, j, j.first, step, count);
            else if (count <= 8) a8_merge<DT, D, MT, true, 8>(p, j, j.first, step, count);
            else a8_merge<DT, D, MT, true, 16>(p, j, j.first, step, count);
        }
    }
}

// DT: type of q and out.  MT: groups of eight query heads per unit.
template <int DT, int D, int MT>
__global__ void __launch_bounds__(A8_THREADS, MT == 1 ? 3 : 2) attn_decode_i8_kernel(const __grid_constant__ AttnI8Params p) {
    constexpr int ROWS = 8 * MT, CHUNKS = D / 16, PART_BYTES = A8_PART * D, STEPS = D / 32, NT = D / 8, STAGE_BYTES = a8_stage(D);
    constexpr int RED = D + 8;  // floats from one row of the merge buffer to the next
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* ring = smem + (threadIdx.x >> 5) * A8_STAGES * STAGE_BYTES;  // this warp's: [A8_STAGES][keys | values | key steps | value steps]
    float* red_o = reinterpret_cast<float*>(smem + A8_WARPS * A8_STAGES * STAGE_BYTES);  // [A8_WARPS][ROWS][RED]
    float* red_ml = red_o + A8_WARPS * ROWS * RED;                            // [A8_WARPS][ROWS][2]
    __shared__ int s_scan[2][A8_WARPS], s_most[A8_WARPS], s_at[3], s_plan[3], s_last[2], s_joins;
    __shared__ A8Join s_join[2];
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const int units = p.nkv * p.blocks;

    // ---- this CTA's range of tiles
    const int ctas = static_cast<int>(gridDim.x);
    int R, total, sought = static_cast<int>(blockIdx.x), piece;
    A8Cursor use;
    // sequences without positions: zeros, by whichever CTA
    auto clear = [&](int b) {
        for (int i = tid; i < p.nq * D; i += A8_THREADS) static_cast<uint16_t*>(p.out)[static_cast<int64_t>(b) * p.nq * D + i] = 0;
    };
    // Few units: pieces of R tiles each, which begin with their unit, one per CTA; at most 16 of a unit while that makes them no longer than four tiles (the
    // merge of more takes longer than the shorter pieces save: one sequence of 2048, 8 KV heads, 32 pieces 12.6 us, 16 10.6).  Many: ranges of R tiles.
    if (p.pos_stride == 0) {  // sequences of one length: no scan over them, which takes 1 to 2 us
        use.n = a8_length(p, 0);
        use.tiles = (use.n + A8_TILE - 1) / A8_TILE;
        if (use.tiles == 0) {
            for (int b = blockIdx.x; b < p.B; b += ctas) clear(b);
            return;
        }
        const int all = p.B * units;
        total = all * use.tiles;  // < 2^30 (checked on the host)
        R = p.pieces ? (use.tiles - 1) / (ctas / all) + 1 : (total - 1) / ctas + 1;
        R = max(max(R, (use.tiles + A8_SPLITS - 1) / A8_SPLITS), p.pieces ? min(4, (use.tiles + 15) / 16) : 1);
        const int per_unit = p.pieces ? (use.tiles + R - 1) / R : use.tiles;
        if (p.pieces) total = all * per_unit;
        else sought *= R;  // < 2^31 on the same grounds as total
        if (sought >= total) return;
        const int unit = sought / per_unit;
        piece = sought - unit * per_unit;
        use.b = unit / units;
        use.unit = unit - use.b * units;
    } else {
        const int per = (p.B + A8_THREADS - 1) / A8_THREADS, b_lo = min(tid * per, p.B), b_hi = min(b_lo + per, p.B);
        int sum = 0, most = 0;
        for (int b = b_lo; b < b_hi; ++b) {
            const int t = (a8_length(p, b) + A8_TILE - 1) / A8_TILE;
            sum += t;
            most = max(most, t);
        }
        // the values in front of this thread's, and all of them
        auto scan = [&](int v, int* room, int& all) {
            int incl = v;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, incl, s);
                if (lane >= s) incl += o;
            }
            if (lane == 31) room[warp] = incl;
            __syncthreads();
            int front = incl - v;
            all = 0;
#pragma unroll
            for (int w = 0; w < A8_WARPS; ++w) {
                if (w < warp) front += room[w];
                all += room[w];
            }
            return front;
        };
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) s_most[warp] = most;
        int before = scan(sum, s_scan[0], total);
        most = max(max(s_most[0], s_most[1]), max(s_most[2], s_most[3]));
        total *= units;  // < 2^30 (checked on the host)
        for (int b = blockIdx.x; b < p.B; b += ctas)
            if (a8_length(p, b) == 0) clear(b);
        R = max((most + A8_SPLITS - 1) / A8_SPLITS, p.pieces ? max((total - 1) / (ctas - p.B * units) + 1, min(4, (most + 15) / 16)) : (total + ctas - 1) / ctas);
        R = max(R, 1);
        int mine = sum;
        if (p.pieces) {
            mine = 0;
            for (int b = b_lo; b < b_hi; ++b) mine += ((a8_length(p, b) + A8_TILE - 1) / A8_TILE + R - 1) / R;
            before = scan(mine, s_scan[1], total);
            total *= units;
        } else {
            sought *= R;  // < 2^31 on the same grounds as total
        }
        if (sought >= total) return;
        if (mine > 0 && before * units <= sought && sought < (before + mine) * units) {
            int at = before * units, b = b_lo;
            for (;; ++b) {
                int t = (a8_length(p, b) + A8_TILE - 1) / A8_TILE;
                if (p.pieces) t = (t + R - 1) / R;
                if (sought < at + t * units) {
                    s_at[0] = b;
                    s_at[1] = (sought - at) / t;
                    s_at[2] = (sought - at) % t;
                    break;
                }
                at += t * units;
            }
        }
        __syncthreads();
        use.b = s_at[0];
        use.n = a8_length(p, use.b);
        use.tiles = (use.n + A8_TILE - 1) / A8_TILE;
        use.unit = s_at[1];
        piece = s_at[2];
    }
    use.tile = piece * (p.pieces ? R : 1);
    if (tid == 0) {  // for the merges; the loop over the tiles needs the registers
        s_plan[0] = R;
        s_plan[1] = piece;
        s_plan[2] = sought;
        s_joins = 0;
    }
    const int gt1 = p.pieces ? min(R, use.tiles - use.tile) : min(sought + R, total);  // the tiles end, by number among all or within the piece
    int gt = p.pieces ? 0 : sought;

    // Every warp copies its own 16 positions of a tile and waits for nobody else's: between the units no barrier holds the warps together.
    constexpr int STRIDE = 32 / CHUNKS;  // rows that a warp copies in one go
    const int my_row = lane / CHUNKS, my_chunk = lane % CHUNKS;
    const uint32_t ring_s = a8_smem(ring), off0 = ring_s + a8_off<D>(my_row, my_chunk), off1 = ring_s + a8_off<D>(my_row + STRIDE, my_chunk) - STRIDE * D;
    const int64_t v_from_k = p.v - p.k;
    int ask_stage = 0;                // byte offset of the stage of the next tile to request, which `use` stands at
    const int8_t* ask_k = nullptr;    // this lane's first chunk of keys in it
    const float* ask_step = nullptr;  // and its step: of a key (lanes 0..15) or of a value
    bool ask_unit = true;
    auto request = [&](int number) {
        if (number < gt1) {
            if (ask_unit) {
                const int64_t row = (static_cast<int64_t>(use.b) * p.nkv + use.unit / p.blocks) * p.T + use.tile * A8_TILE + warp * A8_PART;
                ask_k = p.k + (row + my_row) * D + my_chunk * 16;
                ask_step = (lane < A8_PART ? p.ks : p.vs) + row + (lane & (A8_PART - 1));
            }
            const int left = use.n - use.tile * A8_TILE - warp * A8_PART;
            if (left >= A8_PART) {
#pragma unroll
                for (int j = 0; j < A8_PART / STRIDE; ++j) {
                    const uint32_t to = (j & 1 ? off1 : off0) + ask_stage + j * STRIDE * D;
                    a8_copy16(to, ask_k + j * STRIDE * D, true);
                    a8_copy16(to + PART_BYTES, ask_k + v_from_k + j * STRIDE * D, true);
                }
                a8_copy4(ring_s + ask_stage + 2 * PART_BYTES + lane * 4, ask_step, true);
            } else if (left > 0) {  // nothing is read beyond the length
#pragma unroll
                for (int j = 0; j < A8_PART / STRIDE; ++j) {
                    const uint32_t to = (j & 1 ? off1 : off0) + ask_stage + j * STRIDE * D;
                    const bool ok = my_row + j * STRIDE < left;
                    a8_copy16(to, ok ? ask_k + j * STRIDE * D : p.k, ok);
                    a8_copy16(to + PART_BYTES, ok ? ask_k + v_from_k + j * STRIDE * D : p.v, ok);
                }
                const bool ok = (lane & (A8_PART - 1)) < left;
                a8_copy4(ring_s + ask_stage + 2 * PART_BYTES + lane * 4, ok ? ask_step : p.ks, ok);
            }
            ask_k += A8_TILE * D;
            ask_step += A8_TILE;
            if (lane == 0) *reinterpret_cast<int4*>(ring + ask_stage + 2 * PART_BYTES + 2 * A8_PART * 4) = make_int4(min(max(left, 0), A8_PART) + use.tiles * 32, use.tile * 2 + (use.tile == use.tiles - 1), use.b, use.unit);
            ask_unit = use.next(p, units);
            ask_stage = ask_stage == (A8_STAGES - 1) * STAGE_BYTES ? 0 : ask_stage + STAGE_BYTES;
        }
        a8_commit();  // one group per slot, also when empty: the wait counts stay uniform
    };
#pragma unroll
    for (int s = 0; s < A8_STAGES - 1; ++s) request(gt + s);

    uint32_t qa[MT][STEPS][6];  // first digits, second digits, third digits of a step's 4 + 4 values
    float o[MT][NT][4], m_run[MT], l_run[MT], q_step[MT];
    float s_end[MT], w_to[MT];  // how large a score may get before the references are renewed; 2^15 over how large p * v_step may get
    float v_end = 0.f;          // how large a value's step may get
    int stage = 0;
    bool fresh = true;
    for (; gt < gt1; ++gt) {
        request(gt + A8_STAGES - 1);
        a8_wait<A8_STAGES - 1>();
        __syncwarp();
        const uint8_t* ks = ring + stage;
        const uint8_t* vs = ks + PART_BYTES;
        const float* k_step = reinterpret_cast<const float*>(vs + PART_BYTES);
        const float* v_step = k_step + A8_PART;
        const int4 what = *reinterpret_cast<const int4*>(v_step + A8_PART);  // positions for this warp, the unit's tiles (below 2^24); the tile's number in its unit, whether it is the last; sequence, unit
        stage = stage == (A8_STAGES - 1) * STAGE_BYTES ? 0 : stage + STAGE_BYTES;
        if (fresh) {
            // ---- a new unit: this thread's D / 4 values of query row g as digits
            fresh = false;
            const int kvh = what.w / p.blocks, h0 = (what.w - kvh * p.blocks) * ROWS;
            const int64_t q_at = static_cast<int64_t>(what.z) * p.ldq + (static_cast<int64_t>(kvh) * p.G + h0) * D;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const bool there = h0 + m * 8 + g < p.G;
                const uint16_t* row = static_cast<const uint16_t*>(p.q) + q_at + (there ? (m * 8 + g) * D : 0) + t4 * (D / 4);
                uint4 raw[STEPS];
#pragma unroll
                for (int s = 0; s < STEPS; ++s) raw[s] = ld16_chained(row + s * 8);
                auto get = [&](int s, float (&f)[8]) {
                    const uint4 x = there ? raw[s] : make_uint4(0, 0, 0, 0);
                    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (DT == WF_BF16) {
                            f[2 * i] = __uint_as_float(w[i] << 16);
                            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
                        } else {
                            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                            f[2 * i] = v.x;
                            f[2 * i + 1] = v.y;
                        }
                    }
                };
                float top = 7.8886090522101181e-31f;  // 2^-100
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    float f[8];
                    get(s, f);
#pragma unroll
                    for (int i = 0; i < 8; ++i) top = a8_max_nan(top, fabsf(f[i]));
                }
                top = a8_max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = a8_max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float to = A8_DIGITS / top;  // an infinity or a NaN: digits of 0, and a step that makes every score a NaN
                q_step[m] = top * (1.f / A8_DIGITS) * p.scale_log2;
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    float f[8];
                    get(s, f);
                    a8_digits(f, to, qa[m][s][0], qa[m][s][2], qa[m][s][4]);
                    a8_digits(f + 4, to, qa[m][s][1], qa[m][s][3], qa[m][s][5]);
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) o[m][j][0] = o[m][j][1] = o[m][j][2] = o[m][j][3] = 0.f;
                m_run[m] = -INFINITY;
                l_run[m] = 0.f;
                s_end[m] = -INFINITY;
                w_to[m] = 1.f;
            }
        }
        const int left = what.x & 31;
        if (left > 0) {
            // ---- scores of two times eight positions: this thread gets those of query row g at 2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9
            float s[MT][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t w[2 * STEPS];
#pragma unroll
                for (int c = 0; c < STEPS / 2; ++c) {
                    const uint4 x = *reinterpret_cast<const uint4*>(ks + a8_off<D>(h * 8 + g, t4 * (STEPS / 2) + c));
                    w[4 * c] = x.x; w[4 * c + 1] = x.y; w[4 * c + 2] = x.z; w[4 * c + 3] = x.w;
                }
                const float2 kk = *reinterpret_cast<const float2*>(k_step + h * 8 + 2 * t4);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    int a[4] = {0, 0, 0, 0}, b[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < STEPS; ++i) {
                        a8_mma_s8(a, qa[m][i][0], qa[m][i][2], qa[m][i][1], qa[m][i][3], w[2 * i], w[2 * i + 1]);
                        a8_mma_s8(b, qa[m][i][4], 0u, qa[m][i][5], 0u, w[2 * i], w[2 * i + 1]);
                    }
                    s[m][2 * h] = fmaf(static_cast<float>(a[0]), 65536.f, static_cast<float>(a[2] * 256 + b[0])) * (kk.x * q_step[m]);
                    s[m][2 * h + 1] = fmaf(static_cast<float>(a[1]), 65536.f, static_cast<float>(a[3] * 256 + b[1])) * (kk.y * q_step[m]);
                }
            }
            const float2 va = *reinterpret_cast<const float2*>(v_step + 2 * t4), vb = *reinterpret_cast<const float2*>(v_step + 8 + 2 * t4);
            if (left < 16) {
                const int at[4] = {2 * t4, 2 * t4 + 1, 2 * t4 + 8, 2 * t4 + 9};
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (at[i] >= left) s[m][i] = -INFINITY;
            }
            // ---- other references for the scores or for p * v_step: rare behind the first tiles
            const auto largest = [](float x, float y, float z, float w) { return fmaxf(fmaxf(x, y), fmaxf(z, w)); };
            float top_v = largest(fabsf(va.x), fabsf(va.y), fabsf(vb.x), fabsf(vb.y));
            bool renew = top_v > v_end;
#pragma unroll
            for (int m = 0; m < MT; ++m) renew = renew || largest(s[m][0], s[m][1], s[m][2], s[m][3]) > s_end[m];
            if (__any_sync(0xffffffffu, renew)) {
                const auto above = [](float v) { return static_cast<float>(static_cast<int>(__float_as_uint(v) >> 23 & 255u) - 126); };  // log2 of a power of two above |v|
                const float lv[4] = {above(va.x), above(va.y), above(vb.x), above(vb.y)};
                top_v = fmaxf(top_v, __shfl_xor_sync(0xffffffffu, top_v, 1));
                top_v = fmaxf(top_v, __shfl_xor_sync(0xffffffffu, top_v, 2));  // the same positions in all rows
                v_end = __uint_as_float((__float_as_uint(top_v) + 0x7fffffu) & 0x7f800000u);  // of this tile: one that was larger without weight is behind
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    float mx = largest(s[m][0], s[m][1], s[m][2], s[m][3]), end = static_cast<float>(127 + 15 - static_cast<int>(__float_as_uint(w_to[m]) >> 23));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    if (mx > m_run[m]) {  // whole numbers: powers of two exactly
                        mx = ceilf(mx) + A8_AHEAD;
                        l_run[m] *= a8_exp2(m_run[m] - mx);
                        end += m_run[m] - mx;
                        m_run[m] = mx;
                    }
                    float wx = largest(s[m][0] - m_run[m] + lv[0], s[m][1] - m_run[m] + lv[1], s[m][2] - m_run[m] + lv[2], s[m][3] - m_run[m] + lv[3]);
                    wx = fmaxf(wx, __shfl_xor_sync(0xffffffffu, wx, 1));
                    wx = fmaxf(wx, __shfl_xor_sync(0xffffffffu, wx, 2));
                    const float w_end = fmaxf(fmaxf(end, ceilf(wx) + A8_ROOM), -111.f), both = a8_exp2(end - w_end);
                    w_to[m] = __int_as_float((127 + 15 - static_cast<int>(w_end)) << 23);
                    s_end[m] = __fadd_rd(m_run[m], fminf(0.f, w_end - above(top_v)));
#pragma unroll
                    for (int j = 0; j < NT; ++j) { o[m][j][0] *= both; o[m][j][1] *= both; o[m][j][2] *= both; o[m][j][3] *= both; }
                }
            }
            uint32_t pa[MT][4];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const float base = m_run[m] == -INFINITY ? 0.f : m_run[m];  // every score so far has overflowed to -inf: weights of zero, not inf - inf
                float pe[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) pe[i] = a8_exp2(s[m][i] - base);
                l_run[m] += (pe[0] + pe[1]) + (pe[2] + pe[3]);  // this thread's positions; the four threads of a row are summed at the end
                a8_split(pe[0] * va.x * w_to[m], pe[1] * va.y * w_to[m], pa[m][0], pa[m][1]);
                a8_split(pe[2] * vb.x * w_to[m], pe[3] * vb.y * w_to[m], pa[m][2], pa[m][3]);
            }
            // ---- O += P V: this thread's D / 8 neighbouring codes (from g * D / 8 on) of positions 2 t4, + 1, + 8, + 9
            uint32_t w[4][NT / 4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 2 * t4 + (i & 1) + (i >> 1) * 8;
                if constexpr (D == 128) {
                    const uint4 x = *reinterpret_cast<const uint4*>(vs + a8_off<D>(r, g));
                    w[i][0] = x.x; w[i][1] = x.y; w[i][2] = x.z; w[i][3] = x.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2*>(vs + a8_off<D>(r, g >> 1) + (g & 1) * 8);
                    w[i][0] = x.x; w[i][1] = x.y;
                }
            }
#pragma unroll
            for (int c = 0; c < NT / 4; ++c) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {  // codes 4 c + 2 u and the next: bytes (first, next) of one position, then of the other
                    const uint32_t pick = u ? 0x7632 : 0x5410;
                    const uint32_t x = __byte_perm(w[0][c], w[1][c], pick), y = __byte_perm(w[2][c], w[3][c], pick);
                    const uint32_t x0 = a8_codes(x), y0 = a8_codes(y), x1 = a8_codes(x >> 8), y1 = a8_codes(y >> 8);
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        a8_mma_f16(o[m][4 * c + 2 * u], pa[m], x0, y0);
                        a8_mma_f16(o[m][4 * c + 2 * u + 1], pa[m], x1, y1);
                    }
                }
            }
        }
        __syncwarp();  // every lane is done with this stage before it is refilled
        if (!(what.y & 1) && gt != gt1 - 1) continue;

        // ---- this CTA's share of the unit is complete: merge the warps, each of which saw a quarter of every tile's positions
        const int kvh = what.w / p.blocks, h0 = (what.w - kvh * p.blocks) * ROWS, rows = min(ROWS, p.G - h0);
        const int64_t out0 = static_cast<int64_t>(what.z) * p.nq * D + (static_cast<int64_t>(kvh) * p.G + h0) * D;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const float w_of = __uint_as_float(0x7f000000u - __float_as_uint(w_to[m]));  // 1 over a power of two
            float l = l_run[m];
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            if (t4 == 0) *reinterpret_cast<float2*>(red_ml + (warp * ROWS + m * 8 + g) * 2) = make_float2(m_run[m], l);
#pragma unroll
            for (int j = 0; j < NT; ++j)  // column 2 t4 + e of instruction j is value (2 t4 + e) * NT + j of the head: kept at 8 j + 2 t4 + e
                *reinterpret_cast<float2*>(red_o + (warp * ROWS + m * 8 + g) * RED + 8 * j + 2 * t4) = make_float2((o[m][j][0] + o[m][j][2]) * w_of, (o[m][j][1] + o[m][j][3]) * w_of);
        }
        __syncthreads();
        const int plan_r = s_plan[0], tiles = what.x >> 5, unit_start = gt - (what.y >> 1);  // the number of the unit's first tile
        const int cta = static_cast<int>(blockIdx.x), first_cta = p.pieces ? cta - s_plan[1] : unit_start / plan_r;
        const int expected = p.pieces ? (tiles + plan_r - 1) / plan_r : (unit_start + tiles - 1) / plan_r - first_cta + 1;
        const int64_t part = 2 * cta + (!p.pieces && unit_start >= s_plan[2] ? 1 : 0);  // the second of a CTA's two where the unit begins in its range
        for (int i = tid; i < rows * (D / 4); i += A8_THREADS) {
            const int r = i / (D / 4), at = i % (D / 4) * 4;
            float2 ml[A8_WARPS];
            float mstar = -INFINITY, l = 0.f;
#pragma unroll
            for (int w = 0; w < A8_WARPS; ++w) {
                ml[w] = *reinterpret_cast<const float2*>(red_ml + (w * ROWS + r) * 2);
                mstar = fmaxf(mstar, ml[w].x);
            }
            float4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < A8_WARPS; ++w) {
                const float f = ml[w].x == -INFINITY ? 0.f : a8_exp2(ml[w].x - mstar);
                const float4 v = *reinterpret_cast<const float4*>(red_o + (w * ROWS + r) * RED + at);
                acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
                l += ml[w].y * f;
            }
            if (expected == 1) {
                a8_give<DT, D>(p, out0, r, at, make_float4(acc.x / l, acc.y / l, acc.z / l, acc.w / l));
            } else {
                *reinterpret_cast<float4*>(p.part_o + (part * ROWS + r) * D + at) = acc;
                if (at == 0) *reinterpret_cast<float2*>(p.part_ml + (part * ROWS + r) * 2) = make_float2(mstar, l);
            }
        }
        if (expected > 1 && tid == 0) s_join[s_joins++] = {what.z, what.w, first_cta, expected, !p.pieces && unit_start >= first_cta * plan_r};
        __syncthreads();  // the merge buffer is free again
        fresh = true;
    }
    a8_wait<0>();
    __syncthreads();
    // Behind the loop: in it the merge's registers were taken from those of the tiles (32 sequences of 2048: 37 -> 66 us).
    if (s_joins) a8_join<DT, D, MT>(p, s_join, s_joins, s_last);
}

static int a8_rows(int G) { return G <= 8 ? 8 : 16; }
static int a8_ctas(int G) { return (G <= 8 ? 3 : 2) * num_sms(); }  // that an SM holds at once
static int a8_grid(int64_t units, int64_t T, int G) {
    const int64_t tiles = units * ((T + A8_TILE - 1) / A8_TILE), most = a8_ctas(G);
    return static_cast<int>(tiles < most ? tiles : most);
}

template <int DT, int D, int MT>
static int launch_attn_i8(const AttnI8Params& p, int grid, unsigned flags, cudaStream_t st) {
    constexpr size_t smem = A8_WARPS * A8_STAGES * a8_stage(D) + A8_WARPS * 8 * MT * (D + 8 + 2) * 4;
    static_assert((MT == 1 ? 3 : 2) * (smem + 1024 + 256) <= 228 * 1024, "CTAs per SM");
    static PerDeviceOnce configured;
    const int dev = current_device();
    if (configured.needs(dev)) {
        WF_CUDA(cudaFuncSetAttribute(attn_decode_i8_kernel<DT, D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
        configured.mark(dev);
    }
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(grid);
    lc.blockDim = dim3(A8_THREADS);
    lc.dynamicSmemBytes = smem;
    lc.stream = st;
    cudaLaunchAttribute attr[1];
    if (flags & WF_FLAG_PDL) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        lc.attrs = attr;
        lc.numAttrs = 1;
    }
    WF_CUDA(cudaLaunchKernelEx(&lc, attn_decode_i8_kernel<DT, D, MT>, p));
    return WF_OK;
}
template <int DT>
static int launch_attn_i8_of(const AttnI8Params& p, int D, int grid, unsigned flags, cudaStream_t st) {
    const bool one = a8_rows(p.G) == 8;
    if (D == 64) return one ? launch_attn_i8<DT, 64, 1>(p, grid, flags, st) : launch_attn_i8<DT, 64, 2>(p, grid, flags, st);
    return one ? launch_attn_i8<DT, 128, 1>(p, grid, flags, st) : launch_attn_i8<DT, 128, 2>(p, grid, flags, st);
}

}  // namespace wf

using namespace wf;

// workspace: [tickets: two times A8_TICKETS ints] [partial outputs] [partial maxima and sums], two partial results of a unit's rows per CTA
extern "C" size_t wf_attn_decode_i8_workspace_bytes(int nq, int nkv, int D) {
    if (nq <= 0 || nkv <= 0 || D <= 0 || nq % nkv) return 0;
    return 2 * A8_TICKETS * sizeof(int) + static_cast<size_t>(a8_ctas(nq / nkv)) * 2 * a8_rows(nq / nkv) * (D + 2) * sizeof(float);
}

extern "C" int wf_attn_decode_i8(const void* q, int dtype, int64_t ldq, const int8_t* kcache, const int8_t* vcache, const float* kscale, const float* vscale,
                                 const int64_t* pos, int pos_stride, void* out, int64_t B, int nq, int nkv, int D, int64_t T, float scale, void* workspace,
                                 size_t workspace_bytes, unsigned flags, void* stream) {
    WF_REQUIRE(q && kcache && vcache && kscale && vscale && out, "wf_attn_decode_i8: null pointer");
    WF_REQUIRE(dtype == WF_BF16 || dtype == WF_F16, "wf_attn_decode_i8: q and out must be bf16 or f16");
    WF_REQUIRE(D == 64 || D == 128, "wf_attn_decode_i8: head dimension must be 64 or 128 (got %d)", D);
    WF_REQUIRE(B > 0 && B < (1LL << 30) && nq > 0 && nkv > 0 && nq % nkv == 0 && T > 0 && T < (1LL << 30) && (pos_stride == 0 || pos_stride == 1),
               "wf_attn_decode_i8: bad dimensions (query heads must be a multiple of the KV heads)");
    const int G = nq / nkv, blocks = (G + a8_rows(G) - 1) / a8_rows(G);
    const int64_t tiles = (T + A8_TILE - 1) / A8_TILE;
    WF_REQUIRE(B <= (1LL << 30) / tiles && B * tiles <= (1LL << 30) / (static_cast<int64_t>(nkv) * blocks), "wf_attn_decode_i8: oversized problem");
    WF_REQUIRE(ldq >= static_cast<int64_t>(nq) * D && ldq % 8 == 0, "wf_attn_decode_i8: the row stride of q must cover the heads and be a multiple of 8");
    WF_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kcache) | reinterpret_cast<uintptr_t>(vcache)) & 15) == 0,
               "wf_attn_decode_i8: q and the caches must be 16-byte aligned");
    const size_t need = wf_attn_decode_i8_workspace_bytes(nq, nkv, D);
    if (!workspace || workspace_bytes < need) return fail(WF_E_SCRATCH, "wf_attn_decode_i8: workspace of %zu bytes, need %zu", workspace ? workspace_bytes : 0, need);
    WF_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 256 == 0, "wf_attn_decode_i8: workspace must be 256-byte aligned");
    const auto from = reinterpret_cast<uintptr_t>(q), to = reinterpret_cast<uintptr_t>(out);
    WF_REQUIRE(to >= from + 2 * ((B - 1) * ldq + static_cast<int64_t>(nq) * D) || from >= to + 2 * B * nq * D,
               "wf_attn_decode_i8: out must not overlap q, which parts of a sequence that run later still read");
    if (int rc = require_device()) return rc;
    AttnI8Params p;
    p.q = q; p.k = kcache; p.v = vcache; p.ks = kscale; p.vs = vscale; p.pos = pos; p.out = out;
    p.ldq = ldq; p.pos_stride = pos_stride; p.B = static_cast<int>(B); p.nq = nq; p.nkv = nkv; p.T = static_cast<int>(T);
    p.G = G; p.blocks = blocks;
    p.scale_log2 = scale * 1.4426950408889634f;
    int grid = a8_grid(B * nkv * blocks, T, G);
    // at least four pieces of a unit: 7 sequences of 2048 with 8 KV heads 14.9 us, in ranges 18.1, 12 of them 18.5 and 20.9; with three 16 of them 21.7 and 24.4, but
    // 16 of 8192 59.2 and 57.3, 16 of different lengths up to that 45.8 and 40.7
    p.pieces = 4 * B * nkv * blocks <= a8_ctas(G);
    if (p.pieces) grid = a8_ctas(G);  // pieces are rounded up unit by unit
    WF_REQUIRE(grid <= A8_TICKETS, "wf_attn_decode_i8: more CTAs than tickets");
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    p.tickets = reinterpret_cast<int*>(ws);
    p.part_o = reinterpret_cast<float*>(ws + 2 * A8_TICKETS * sizeof(int));
    p.part_ml = p.part_o + static_cast<size_t>(a8_ctas(G)) * 2 * a8_rows(G) * D;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == WF_BF16 ? launch_attn_i8_of<WF_BF16>(p, D, grid, flags, st) : launch_attn_i8_of<WF_F16>(p, D, grid, flags, st);
}

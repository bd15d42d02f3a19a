// Rows in 8 bits: the quantizing write of new keys and values into an int8 cache (with the rotary embedding in front of it), the reading
// back, and the quantization of plain rows (weights per output channel, activations per token).
//
//   a = max |r| of the row (at least 2^-100),  code = rint(r * (127 / a)),  step = a / 127,  value = code * step
//
// Every operation is an fp32 operation rounded by itself, 127 / a and a / 127 with it, so that codes and steps are defined to the bit.  A row that
// holds an infinity or a NaN gets codes of zero and that as its step: it reads back as NaN, not as a number.  All three kernels move each
// element once; HBM bounds them on many rows, the launch on few.
#include <initializer_list>

#include "wf_common.cuh"

namespace wf {

constexpr float Q8_LEAST = 7.8886090522101181e-31f;  // 2^-100: below it a row counts as zeros and 127 / a stays finite

__device__ __forceinline__ float max_nan(float a, float b) {  // a NaN on either side is the result
    float r;
    asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// rint(v * inv) in the low byte: beside 1.5 * 2^23 the sum's last place is 1.  (The conversion instruction runs at an eighth of the rate.)
__device__ __forceinline__ uint32_t code_of(float v, float inv) { return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.f)); }
// codes of four values; `keep` is 0 for a row that holds an infinity or a NaN
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inv, uint32_t keep) {
    return __byte_perm(__byte_perm(code_of(a, inv), code_of(b, inv), 0x0040), __byte_perm(code_of(c, inv), code_of(d, inv), 0x0040), 0x5410) & keep;
}
__device__ __forceinline__ uint32_t keep_row(float most) { return most < __uint_as_float(0x7f800000u) ? 0xffffffffu : 0u; }
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (DT == WF_BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}
template <int DT>
__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
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
}
template <int DT>
__device__ __forceinline__ void store8(void* base, int64_t off, const float (&f)[8]) {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + off) = make_uint4(pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3]), pack2<DT>(f[4], f[5]), pack2<DT>(f[6], f[7]));
}

struct RopeI8Params {
    const void* q;         // row b * S + s, stride ldq: [nq * D]
    const void* k;         // the same with nkv heads, stride ldkv
    const void* v;
    void* q_out;           // stride ldo; may be q
    const float* cos;      // [T, D / 2]
    const float* sin;
    const int64_t* pos;    // position of a sequence's first new token, pos_stride (0 or 1) apart
    int8_t *kc, *vc;       // [B, nkv, T, D]
    float *ks, *vs;        // [B, nkv, T]
    int64_t ldq, ldkv, ldo, rows;
    int pos_stride, S, T, nq, nkv;
    int groups, block_rows;  // threads per 8 + 8 values of a token's heads; tokens per block
};

// D / 16 neighbouring threads share a head, 8 + 8 values each (the two halves that rotate into each other), and find its maximum together.  A thread takes the
// same values of ROPE_HEADS heads at a time: their loads are in flight together, in front of the position and the rotation that is found by it (read
// once for them).  A token outside the cache's positions writes nothing and gets a query of zeros.
// 8192 tokens of 20 + 2 x 5 heads of 128: 24.2 us = 4.8 TB/s (17.7 us at the measured copy rate); a thread per head, the position first, 30.9.
constexpr int ROPE_THREADS = 256;
constexpr int ROPE_HEADS = 4;
template <int DT, int D>
__global__ void __launch_bounds__(ROPE_THREADS, 3) rope_kv_i8_kernel(const RopeI8Params p) {
    constexpr int PARTS = D / 16, HALF = D / 2;
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    const int per_row = PARTS * p.groups, here = static_cast<int>(threadIdx.x) / per_row, rest = static_cast<int>(threadIdx.x) - here * per_row;
    const int part = rest % PARTS, group = rest / PARTS, heads = p.nq + 2 * p.nkv;
    const int64_t row_at = static_cast<int64_t>(blockIdx.x) * p.block_rows + here;
    const bool live = here < p.block_rows && row_at < p.rows;  // whole heads: the threads of one are all live or all not
    const int64_t row = live ? row_at : 0;
    uint4 raw[ROPE_HEADS][2];
    auto load = [&](int base) {
#pragma unroll
        for (int j = 0; j < ROPE_HEADS; ++j) {
            const int head = base + j * p.groups;
            if (head < heads) {
                const bool is_q = head < p.nq, is_v = head >= p.nq + p.nkv;
                const void* src = is_q ? p.q : (is_v ? p.v : p.k);
                const int hk = is_v ? head - p.nq - p.nkv : head - p.nq;
                const uint16_t* from = static_cast<const uint16_t*>(src) + (is_q ? row * p.ldq + static_cast<int64_t>(head) * D : row * p.ldkv + static_cast<int64_t>(hk) * D) + part * 8;
                raw[j][0] = ld16_chained(from);
                raw[j][1] = ld16_chained(from + HALF);
            }
        }
    };
    load(group);  // in front of the position and of the rotation that is found by it
    const int64_t b = row / p.S, at = p.pos[b * p.pos_stride] + (row - b * p.S);
    const bool in = at >= 0 && at < p.T;
    float cs[8], sn[8];
    {
        const int64_t from = (in ? at : 0) * HALF + part * 8;
        const uint4 c0 = ld16_chained(p.cos + from), c1 = ld16_chained(p.cos + from + 4), s0 = ld16_chained(p.sin + from), s1 = ld16_chained(p.sin + from + 4);
        const uint32_t cu[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, su[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            cs[e] = __uint_as_float(cu[e]);
            sn[e] = __uint_as_float(su[e]);
        }
    }
    for (int base = group; base - group < heads; base += p.groups * ROPE_HEADS) {
        if (base != group) load(base);
#pragma unroll
        for (int j = 0; j < ROPE_HEADS; ++j) {
            const int head = base + j * p.groups;
            const bool is_q = head < p.nq, is_v = head >= p.nq + p.nkv;
            float lo[8], hi[8];
            unpack8<DT>(raw[j][0], lo);
            unpack8<DT>(raw[j][1], hi);
            if (!is_v) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x1 = lo[e], x2 = hi[e];
                    lo[e] = __fsub_rn(__fmul_rn(x1, cs[e]), __fmul_rn(x2, sn[e]));
                    hi[e] = __fadd_rn(__fmul_rn(x2, cs[e]), __fmul_rn(x1, sn[e]));
                }
            }
            float most = Q8_LEAST;
            if (__any_sync(0xffffffffu, !is_q)) {  // queries are not quantized
#pragma unroll
                for (int e = 0; e < 8; ++e) most = max_nan(most, max_nan(fabsf(lo[e]), fabsf(hi[e])));
#pragma unroll
                for (int s = PARTS / 2; s > 0; s >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, s));
            }
            if (!live || head >= heads) continue;
            if (is_q) {
                if (!in) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) lo[e] = hi[e] = 0.f;
                }
                const int64_t to = row * p.ldo + static_cast<int64_t>(head) * D + part * 8;
                store8<DT>(p.q_out, to, lo);
                store8<DT>(p.q_out, to + HALF, hi);
            } else if (in) {
                const float inv = __fdiv_rn(127.0f, most);
                const uint32_t keep = keep_row(most);
                const int64_t slot = (b * p.nkv + (is_v ? head - p.nq - p.nkv : head - p.nq)) * p.T + at;
                int8_t* dst = (is_v ? p.vc : p.kc) + slot * D + part * 8;
                *reinterpret_cast<uint2*>(dst) = make_uint2(codes4(lo[0], lo[1], lo[2], lo[3], inv, keep), codes4(lo[4], lo[5], lo[6], lo[7], inv, keep));
                *reinterpret_cast<uint2*>(dst + HALF) = make_uint2(codes4(hi[0], hi[1], hi[2], hi[3], inv, keep), codes4(hi[4], hi[5], hi[6], hi[7], inv, keep));
                if (part == 0) (is_v ? p.vs : p.ks)[slot] = __fdiv_rn(most, 127.0f);
            }
        }
    }
}

struct ReadI8Params {
    const int8_t *kc, *vc;
    const float *ks, *vs;
    void *k, *v;           // [B * nkv, S, D]
    int64_t total;         // threads for one of the two
    int T, start, S;
};
template <int DT, int D>
__global__ void __launch_bounds__(256) kv_read_i8_kernel(const ReadI8Params p) {
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    const bool is_v = i >= p.total;
    if (is_v) i -= p.total;
    if (i >= p.total) return;
    const int part = static_cast<int>(i % (D / 16));
    const int64_t r = i / (D / 16), unit = r / p.S, at = unit * p.T + p.start + (r - unit * p.S);
    const uint4 c = ld16_chained((is_v ? p.vc : p.kc) + at * D + part * 16);
    const float step = *static_cast<const volatile float*>((is_v ? p.vs : p.ks) + at);
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    float f[2][8];
#pragma unroll
    for (int e = 0; e < 16; ++e) f[e / 8][e % 8] = __fmul_rn(static_cast<float>(static_cast<int8_t>(w[e / 4] >> (8 * (e % 4)))), step);
    void* out = is_v ? p.v : p.k;
    store8<DT>(out, r * D + part * 16, f[0]);
    store8<DT>(out, r * D + part * 16 + 8, f[1]);
}

// One block per row; what fits stays in registers between the maximum and the codes, the rest is read again (from L2).
constexpr int QR_THREADS = 256;
constexpr int QR_KEEP = 2;  // chunks of 16 values that a thread keeps: rows up to 8192 values
template <int DT, bool VEC>
__global__ void __launch_bounds__(QR_THREADS) quant_rows_kernel(const void* x, int64_t ldx, int8_t* q, int64_t ldq, float* step, int64_t K) {
    __shared__ float sh[QR_THREADS / 32];
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");  // not in front: the product that follows reads its weights without a wait of its own
    const int64_t row = blockIdx.x, x0 = row * ldx;
    const int tid = threadIdx.x;
    const int64_t chunks = VEC ? K / 16 : 0;
    float keep[QR_KEEP][2][8];
    float most = 0.f;
    auto take = [&](const float (&f)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) most = max_nan(most, fabsf(f[e]));
    };
#pragma unroll
    for (int c = 0; c < QR_KEEP; ++c) {
        const int64_t i = tid + c * QR_THREADS;
        if (i < chunks) {
            load8<DT>(x, x0 + i * 16, keep[c][0]);
            load8<DT>(x, x0 + i * 16 + 8, keep[c][1]);
        }
    }
#pragma unroll
    for (int c = 0; c < QR_KEEP; ++c)
        if (tid + c * QR_THREADS < chunks) {
            take(keep[c][0]);
            take(keep[c][1]);
        }
    for (int64_t i = tid + QR_KEEP * QR_THREADS; i < chunks; i += QR_THREADS) {
        float f[8];
        load8<DT>(x, x0 + i * 16, f);
        take(f);
        load8<DT>(x, x0 + i * 16 + 8, f);
        take(f);
    }
    for (int64_t i = chunks * 16 + tid; i < K; i += QR_THREADS) most = max_nan(most, fabsf(load1<DT>(x, x0 + i)));
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, s));
    if ((tid & 31) == 0) sh[tid >> 5] = most;
    __syncthreads();
    most = Q8_LEAST;
#pragma unroll
    for (int w = 0; w < QR_THREADS / 32; ++w) most = max_nan(most, sh[w]);
    const float inv = __fdiv_rn(127.0f, most);
    const uint32_t whole = keep_row(most);
    int8_t* out = q + row * ldq;
    auto give = [&](int64_t i, const float (&a)[8], const float (&b)[8]) {
        *reinterpret_cast<uint4*>(out + i * 16) = make_uint4(codes4(a[0], a[1], a[2], a[3], inv, whole), codes4(a[4], a[5], a[6], a[7], inv, whole),
                                                             codes4(b[0], b[1], b[2], b[3], inv, whole), codes4(b[4], b[5], b[6], b[7], inv, whole));
    };
#pragma unroll
    for (int c = 0; c < QR_KEEP; ++c)
        if (tid + c * QR_THREADS < chunks) give(tid + c * QR_THREADS, keep[c][0], keep[c][1]);
    for (int64_t i = tid + QR_KEEP * QR_THREADS; i < chunks; i += QR_THREADS) {
        float a[8], b[8];
        load8<DT>(x, x0 + i * 16, a);
        load8<DT>(x, x0 + i * 16 + 8, b);
        give(i, a, b);
    }
    for (int64_t i = chunks * 16 + tid; i < K; i += QR_THREADS) out[i] = static_cast<int8_t>(code_of(load1<DT>(x, x0 + i), inv) & whole);
    if (tid == 0) step[row] = __fdiv_rn(most, 127.0f);
}

// Many rows: one warp per row, which stays in registers up to 32 * QW_KEEP chunks (4096 values of 16 bits).
template <int DT>
__global__ void __launch_bounds__(QR_THREADS) quant_rows_warp_kernel(const void* x, int64_t ldx, int8_t* q, int64_t ldq, float* step, int64_t M, int64_t K) {
    constexpr int KEEP = DT == WF_F32 ? 4 : 8, WORDS = DT == WF_F32 ? 4 : 2, SIZE = DT == WF_F32 ? 4 : 2;  // chunks kept; 16-byte words of one
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");  // not in front: the product that follows reads its weights without a wait of its own
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (QR_THREADS / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= M) return;
    const uint8_t* from = static_cast<const uint8_t*>(x) + row * ldx * SIZE;
    const int chunks = static_cast<int>(K / 16);
    uint4 raw[KEEP][WORDS];
#pragma unroll
    for (int c = 0; c < KEEP; ++c) {
        const int i = lane + c * 32;
        if (i < chunks) {
#pragma unroll
            for (int w = 0; w < WORDS; ++w) raw[c][w] = ld16_chained(from + (static_cast<int64_t>(i) * WORDS + w) * 16);
        }
    }
    auto get = [&](const uint4 (&r)[WORDS], float (&f)[16]) {
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
            const uint32_t u[4] = {r[w].x, r[w].y, r[w].z, r[w].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (DT == WF_F32) {
                    f[4 * w + e] = __uint_as_float(u[e]);
                } else if constexpr (DT == WF_BF16) {
                    f[8 * w + 2 * e] = __uint_as_float(u[e] << 16);
                    f[8 * w + 2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
                } else {
                    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&u[e]));
                    f[8 * w + 2 * e] = v.x;
                    f[8 * w + 2 * e + 1] = v.y;
                }
            }
        }
    };
    float most = Q8_LEAST;
    auto take = [&](const uint4 (&r)[WORDS]) {
        float f[16];
        get(r, f);
#pragma unroll
        for (int e = 0; e < 16; ++e) most = max_nan(most, fabsf(f[e]));
    };
    int8_t* out = q + row * ldq;
    auto give = [&](int i, const uint4 (&r)[WORDS], float inv, uint32_t keep) {
        float f[16];
        get(r, f);
        *reinterpret_cast<uint4*>(out + static_cast<int64_t>(i) * 16) =
            make_uint4(codes4(f[0], f[1], f[2], f[3], inv, keep), codes4(f[4], f[5], f[6], f[7], inv, keep), codes4(f[8], f[9], f[10], f[11], inv, keep),
                       codes4(f[12], f[13], f[14], f[15], inv, keep));
    };
    auto again = [&](int i, uint4 (&r)[WORDS]) {
#pragma unroll
        for (int w = 0; w < WORDS; ++w) r[w] = ld16_chained(from + (static_cast<int64_t>(i) * WORDS + w) * 16);
    };
#pragma unroll
    for (int c = 0; c < KEEP; ++c)
        if (lane + c * 32 < chunks) take(raw[c]);
    for (int i = lane + KEEP * 32; i < chunks; i += 32) {
        uint4 r[WORDS];
        again(i, r);
        take(r);
    }
    for (int64_t i = static_cast<int64_t>(chunks) * 16 + lane; i < K; i += 32) most = max_nan(most, fabsf(load1<DT>(from, i)));
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, s));
    const float inv = __fdiv_rn(127.0f, most);
    const uint32_t keep = keep_row(most);
#pragma unroll
    for (int c = 0; c < KEEP; ++c)
        if (lane + c * 32 < chunks) give(lane + c * 32, raw[c], inv, keep);
    for (int i = lane + KEEP * 32; i < chunks; i += 32) {
        uint4 r[WORDS];
        again(i, r);
        give(i, r, inv, keep);
    }
    for (int64_t i = static_cast<int64_t>(chunks) * 16 + lane; i < K; i += 32) out[i] = static_cast<int8_t>(code_of(load1<DT>(from, i), inv) & keep);
    if (lane == 0) step[row] = __fdiv_rn(most, 127.0f);
}

template <class... KArgs, class... Args>
static cudaError_t launch(void (*kernel)(KArgs...), unsigned grid, unsigned block, unsigned flags, void* stream, Args... args) {
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(grid);
    lc.blockDim = dim3(block);
    lc.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    if (flags & WF_FLAG_PDL) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        lc.attrs = attr;
        lc.numAttrs = 1;
    }
    return cudaLaunchKernelEx(&lc, kernel, args...);
}
static bool aligned16(std::initializer_list<const void*> ps) {
    for (const void* q : ps)
        if (reinterpret_cast<uintptr_t>(q) & 15) return false;
    return true;
}
// Whether one of `rows` rows of a (wa bytes each, lda apart) shares a byte with one of as many of b.  Rows equally far apart may lie between each other, like columns of
// one tensor; of others whose ranges meet it is taken to be so.
static bool rows_meet(const void* a, int64_t wa, int64_t lda, const void* b, int64_t wb, int64_t ldb, int64_t rows) {
    const int64_t from_a_to_b = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b)) - static_cast<int64_t>(reinterpret_cast<uintptr_t>(a));
    if (from_a_to_b >= (rows - 1) * lda + wa || -from_a_to_b >= (rows - 1) * ldb + wb) return false;
    if (rows == 1 || lda != ldb) return true;
    // the first row of b, counted from one of a's, that ends behind that one's beginning
    int64_t first = (-wb - from_a_to_b) / lda;
    while (from_a_to_b + first * lda + wb <= 0) ++first;
    while (first > -(rows - 1) && from_a_to_b + (first - 1) * lda + wb > 0) --first;
    if (first < -(rows - 1)) first = -(rows - 1);
    return first < rows && from_a_to_b + first * lda < wa;
}

}  // namespace wf

using namespace wf;

extern "C" int wf_rope_kv_i8(const void* q, int64_t ldq, const void* k, const void* v, int64_t ldkv, int dtype, const float* cos, const float* sin, const int64_t* pos,
                             int pos_stride, void* q_out, int64_t ldo, int8_t* kcache, int8_t* vcache, float* kscale, float* vscale, int64_t B, int64_t S, int nq, int nkv,
                             int D, int64_t T, unsigned flags, void* stream) {
    WF_REQUIRE(q && k && v && cos && sin && pos && q_out && kcache && vcache && kscale && vscale, "wf_rope_kv_i8: null pointer");
    WF_REQUIRE(dtype == WF_BF16 || dtype == WF_F16, "wf_rope_kv_i8: q, k and v must be bf16 or f16");
    WF_REQUIRE(D == 64 || D == 128, "wf_rope_kv_i8: head dimension must be 64 or 128 (got %d)", D);
    WF_REQUIRE(B > 0 && S > 0 && T > 0 && T < (1LL << 31) && nq > 0 && nkv > 0 && (pos_stride == 0 || pos_stride == 1), "wf_rope_kv_i8: bad dimensions");
    WF_REQUIRE(B <= (1LL << 40) / S / (nq + 2LL * nkv), "wf_rope_kv_i8: oversized problem");
    WF_REQUIRE(ldq >= static_cast<int64_t>(nq) * D && ldo >= static_cast<int64_t>(nq) * D && ldkv >= static_cast<int64_t>(nkv) * D && ((ldq | ldo | ldkv) & 7) == 0,
               "wf_rope_kv_i8: row strides must cover the heads and be multiples of 8");
    WF_REQUIRE(aligned16({q, k, v, cos, sin, q_out, kcache, vcache}), "wf_rope_kv_i8: tensors must be 16-byte aligned");
    WF_REQUIRE(B * S < (1LL << 31), "wf_rope_kv_i8: oversized problem");
    const int64_t wq = 2LL * nq * D, wk = 2LL * nkv * D, rows_all = B * S;
    const bool in_place = q_out == q && (ldo == ldq || rows_all == 1);
    WF_REQUIRE((in_place || !rows_meet(q_out, wq, 2 * ldo, q, wq, 2 * ldq, rows_all)) && !rows_meet(q_out, wq, 2 * ldo, k, wk, 2 * ldkv, rows_all) &&
                   !rows_meet(q_out, wq, 2 * ldo, v, wk, 2 * ldkv, rows_all),
               "wf_rope_kv_i8: q_out must be q itself or share nothing with q, k and v, which other threads still read");
    if (int rc = require_device()) return rc;
    RopeI8Params p;
    p.q = q; p.k = k; p.v = v; p.q_out = q_out; p.cos = cos; p.sin = sin; p.pos = pos;
    p.kc = kcache; p.vc = vcache; p.ks = kscale; p.vs = vscale;
    p.ldq = ldq; p.ldkv = ldkv; p.ldo = ldo; p.rows = B * S;
    p.pos_stride = pos_stride; p.S = static_cast<int>(S); p.T = static_cast<int>(T); p.nq = nq; p.nkv = nkv;
    const int parts = D / 16, heads = nq + 2 * nkv, most = ROPE_THREADS / parts;
    // tokens that fill the card: four heads per thread; fewer: a thread for each
    const bool many = p.rows * heads * parts >= 2LL * ROPE_THREADS * num_sms() * ROPE_HEADS;
    const int wanted = many ? (heads + ROPE_HEADS - 1) / ROPE_HEADS : heads;
    p.groups = wanted < most ? wanted : most;
    p.block_rows = ROPE_THREADS / (parts * p.groups);
    const unsigned grid = static_cast<unsigned>((p.rows + p.block_rows - 1) / p.block_rows);
    auto* kern = dtype == WF_BF16 ? (D == 64 ? rope_kv_i8_kernel<WF_BF16, 64> : rope_kv_i8_kernel<WF_BF16, 128>)
                                  : (D == 64 ? rope_kv_i8_kernel<WF_F16, 64> : rope_kv_i8_kernel<WF_F16, 128>);
    WF_CUDA(launch(kern, grid, ROPE_THREADS, flags, stream, p));
    return WF_OK;
}

extern "C" int wf_kv_read_i8(const int8_t* kcache, const int8_t* vcache, const float* kscale, const float* vscale, void* k, void* v, int dtype, int64_t units, int64_t T,
                             int64_t start, int64_t S, int D, unsigned flags, void* stream) {
    WF_REQUIRE(kcache && vcache && kscale && vscale && k && v, "wf_kv_read_i8: null pointer");
    WF_REQUIRE(dtype == WF_BF16 || dtype == WF_F16, "wf_kv_read_i8: keys and values are read back as bf16 or f16");
    WF_REQUIRE(D == 64 || D == 128, "wf_kv_read_i8: head dimension must be 64 or 128 (got %d)", D);
    WF_REQUIRE(units > 0 && T > 0 && T < (1LL << 31) && S > 0 && start >= 0 && start <= T - S, "wf_kv_read_i8: positions outside the cache");
    WF_REQUIRE(units < (1LL << 40) / S, "wf_kv_read_i8: oversized problem");
    WF_REQUIRE(aligned16({kcache, vcache, k, v}), "wf_kv_read_i8: tensors must be 16-byte aligned");
    const int64_t total = units * S * (D / 16), blocks = (2 * total + 255) / 256;
    WF_REQUIRE(blocks < (1LL << 31), "wf_kv_read_i8: oversized problem");
    if (int rc = require_device()) return rc;
    ReadI8Params p;
    p.kc = kcache; p.vc = vcache; p.ks = kscale; p.vs = vscale; p.k = k; p.v = v;
    p.total = total; p.T = static_cast<int>(T); p.start = static_cast<int>(start); p.S = static_cast<int>(S);
    auto* kern = dtype == WF_BF16 ? (D == 64 ? kv_read_i8_kernel<WF_BF16, 64> : kv_read_i8_kernel<WF_BF16, 128>)
                                  : (D == 64 ? kv_read_i8_kernel<WF_F16, 64> : kv_read_i8_kernel<WF_F16, 128>);
    WF_CUDA(launch(kern, static_cast<unsigned>(blocks), 256, flags, stream, p));
    return WF_OK;
}

extern "C" int wf_quantize_rows_i8(const void* x, int dtype, int64_t ldx, int8_t* q, int64_t ldq, float* step, int64_t M, int64_t K, unsigned flags, void* stream) {
    WF_REQUIRE(x && q && step, "wf_quantize_rows_i8: null pointer");
    WF_REQUIRE(is_float_dtype(dtype), "wf_quantize_rows_i8: x must be f32, f16 or bf16");
    WF_REQUIRE(M > 0 && M < (1LL << 31) && K > 0 && K < (1LL << 31) && ldx >= K && ldq >= K, "wf_quantize_rows_i8: bad dimensions");
    if (int rc = require_device()) return rc;
    const int64_t size = static_cast<int64_t>(dtype_size(dtype));
    const bool vec = aligned16({x, q}) && (ldx * size) % 16 == 0 && ldq % 16 == 0;
    // a warp per row where rows fill the card so (8192 rows of 2560 in bf16: 12.0 us, a block per row 18) and a
    // lane's registers hold its part (8192 of 6912, read twice: 45, a block per row 36)
    if (vec && M >= 8LL * num_sms() && K <= (dtype == WF_F32 ? 2048 : 4096)) {
        auto* kern = dtype == WF_F32 ? quant_rows_warp_kernel<WF_F32> : (dtype == WF_BF16 ? quant_rows_warp_kernel<WF_BF16> : quant_rows_warp_kernel<WF_F16>);
        WF_CUDA(launch(kern, static_cast<unsigned>((M + QR_THREADS / 32 - 1) / (QR_THREADS / 32)), QR_THREADS, flags, stream, x, ldx, q, ldq, step, M, K));
        return WF_OK;
    }
    auto go = [&](auto* kern) { return launch(kern, static_cast<unsigned>(M), QR_THREADS, flags, stream, x, ldx, q, ldq, step, K); };
    if (dtype == WF_F32) WF_CUDA(go(vec ? quant_rows_kernel<WF_F32, true> : quant_rows_kernel<WF_F32, false>));
    else if (dtype == WF_BF16) WF_CUDA(go(vec ? quant_rows_kernel<WF_BF16, true> : quant_rows_kernel<WF_BF16, false>));
    else WF_CUDA(go(vec ? quant_rows_kernel<WF_F16, true> : quant_rows_kernel<WF_F16, false>));
    return WF_OK;
}

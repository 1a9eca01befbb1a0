// pe_mixer.cuh - what the recurrent-mixer kernels share: element types, packed
// sequences, the activations and warp reductions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "pe_common.cuh"

namespace pe {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// One element. Not __ldg of the 16-bit types: CUDA's headers write that as assembly
// without "volatile", which the compiler may move out of the condition that guards it,
// to addresses that are not there.
__device__ __forceinline__ float load_one(const float* p) { return __ldg(p); }
__device__ __forceinline__ __half load_one(const __half* p) {
    return __ushort_as_half(__ldg(reinterpret_cast<const unsigned short*>(p)));
}
__device__ __forceinline__ __nv_bfloat16 load_one(const __nv_bfloat16* p) {
    return __ushort_as_bfloat16(__ldg(reinterpret_cast<const unsigned short*>(p)));
}

// V elements that one load moves (V * sizeof(T) is 16 or 8 bytes, or V is 1).
template <typename T, int V>
struct alignas(V * sizeof(T)) Vec {
    T v[V];
};
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
    if constexpr (V * sizeof(T) == 16) {
        const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
        return *reinterpret_cast<const Vec<T, V>*>(&r);
    } else if constexpr (V * sizeof(T) == 8) {
        const uint2 r = __ldg(reinterpret_cast<const uint2*>(p));
        return *reinterpret_cast<const Vec<T, V>*>(&r);
    } else {
        static_assert(V == 1, "16 or 8 bytes, or one element");
        Vec<T, V> r;
        r.v[0] = load_one(p);
        return r;
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, V>& r) {
    *reinterpret_cast<Vec<T, V>*>(p) = r;
}
template <typename T, int V>
__device__ __forceinline__ void unpack(const Vec<T, V>& r, float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_float(r.v[i]);
}

// 2^x and 1/x of one instruction each (relative errors of 2^-22 and 2^-23; denormal
// arguments and results count as zero).
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// 1 / (1 + exp(-x)); 0, its limit, where exp(-x) overflows.
__device__ __forceinline__ float sigmoidf(float x) { return rcp_fast(1.0f + exp2_fast(-kLog2e * x)); }
// d silu(x) / dx with s = sigmoid(x).
__device__ __forceinline__ float silu_slope(float x, float s) { return s * (1.0f + x * (1.0f - s)); }

// log(1 + exp(x)) = max(x, 0) + log1p(e), e = exp(-|x|) in (0, 1]. log1p(e) =
// 2 artanh(s) with s = e / (2 + e) <= 1/3, whose odd power series through s^13
// leaves a relative error below (1/9)^7 / 15 = 1.4e-8. A logarithm of the
// rounded 1 + e would lose the small step sizes (e = 1e-3 keeps 13 bits).
__device__ __forceinline__ float softplusf(float x) {
    // the product -|x| log2(e) in two parts: rounded to one, small step sizes (x = -7) would
    // be off by 4e-7, more than all that follows
    const float a = fmaxf(-fabsf(x), -150.0f), hi = a * kLog2e;   // finite: exp(-150) is 0 here
    const float lo = fmaf(a, kLog2e, -hi) + a * 1.925963033500011e-8f;   // log2(e) - kLog2e
    float e = exp2_fast(hi);
    e = fmaf(e, lo * kLn2, e);
    const float s = e * rcp_fast(2.0f + e);
    const float q = s * s;
    float r = fmaf(q, 1.0f / 13, 1.0f / 11);
    r = fmaf(r, q, 1.0f / 9);
    r = fmaf(r, q, 1.0f / 7);
    r = fmaf(r, q, 1.0f / 5);
    r = fmaf(r, q, 1.0f / 3);
    r = fmaf(r, q, 1.0f);
    return (x < 0.0f ? 0.0f : x) + 2.0f * s * r;   // NaN stays NaN
}

// ---- packed pairs --------------------------------------------------------------
// Two fp32 lanes in one 64-bit register, one instruction for both.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 exp2_2(f32x2 x) {
    float lo, hi;
    unpack2(x, lo, hi);
    return pack2(exp2_fast(lo), exp2_fast(hi));
}

// V elements as V / 2 pairs (V even).
template <typename T, int V>
__device__ __forceinline__ void unpack_pairs(const Vec<T, V>& r, f32x2 (&f)[V / 2]) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) f[i] = pack2(to_float(r.v[2 * i]), to_float(r.v[2 * i + 1]));
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> pack_pairs(const f32x2 (&f)[V / 2]) {
    Vec<T, V> r;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        float lo, hi;
        unpack2(f[i], lo, hi);
        if constexpr (sizeof(T) == 2) {
            if constexpr (std::is_same<T, __half>::value)
                *reinterpret_cast<__half2*>(&r.v[2 * i]) = __floats2half2_rn(lo, hi);
            else
                *reinterpret_cast<__nv_bfloat162*>(&r.v[2 * i]) = __floats2bfloat162_rn(lo, hi);
        } else {
            r.v[2 * i] = from_float<T>(lo);
            r.v[2 * i + 1] = from_float<T>(hi);
        }
    }
    return r;
}

// V channels as pairs; a single channel is a pair whose other half stays zero.
template <int V>
constexpr int kPairs = (V + 1) / 2;
template <typename T, int V>
__device__ __forceinline__ void widen(const Vec<T, V>& r, f32x2 (&f)[kPairs<V>]) {
    if constexpr (V == 1)
        f[0] = pack2(to_float(r.v[0]), 0.0f);
    else
        unpack_pairs(r, f);
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> narrow(const f32x2 (&f)[kPairs<V>]) {
    if constexpr (V == 1) {
        float lo, hi;
        unpack2(f[0], lo, hi);
        Vec<T, 1> r;
        r.v[0] = from_float<T>(lo);
        return r;
    } else {
        return pack_pairs<T, V>(f);
    }
}
__device__ __forceinline__ f32x2 both(float x) { return pack2(x, x); }
// A value a channel: 0 in the idle half of a single channel's pair.
template <int V>
__device__ __forceinline__ f32x2 each(float x) { return pack2(x, V == 1 ? 0.0f : x); }
__device__ __forceinline__ float halves(f32x2 v) {
    float lo, hi;
    unpack2(v, lo, hi);
    return lo + hi;
}
__device__ __forceinline__ f32x2 sigmoid2(f32x2 x) {
    float lo, hi;
    unpack2(x, lo, hi);
    return pack2(sigmoidf(lo), sigmoidf(hi));
}

// d silu(x) / dx with s = sigmoid(x), in pairs.
__device__ __forceinline__ f32x2 silu_slope2(f32x2 x, f32x2 s) {
    return mul2(s, fma2(x, fma2(s, both(-1.0f), both(1.0f)), both(1.0f)));
}

// ---- asynchronous copies ------------------------------------------------------------
template <int BYTES>
__device__ __forceinline__ void cp_async(void* dst, const void* src, int valid) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(valid) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(valid), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void cp_wait() { cp_wait_but<0>(); }

// A thread's own queue of vectors in shared memory: what it copies only it reads, so the
// copies need no barrier, and DEPTH of them are under way without holding registers.
// Slots of a block's threads lie side by side. A 2-byte element comes as the aligned
// 4-byte word that holds it (its own half alone where that is the first).
template <typename T, int V, int DEPTH>
struct Ring {
    static_assert((DEPTH & (DEPTH - 1)) == 0, "a power of two");
    using Elem = Vec<T, V>;
    static constexpr bool kHalf = sizeof(Elem) == 2;
    using Slot = typename std::conditional<kHalf, uint32_t, Elem>::type;
    Slot* at;
    int stride;
    __device__ __forceinline__ Ring(void* block, int threads)
        : at(reinterpret_cast<Slot*>(block) + threadIdx.x), stride(threads) {}
    __device__ __forceinline__ void fetch(int slot, const T* src, bool on) {
        Slot* dst = at + (slot & (DEPTH - 1)) * stride;
        if constexpr (kHalf) {
            const uintptr_t a = reinterpret_cast<uintptr_t>(src);
            if (on) cp_async<4>(dst, reinterpret_cast<const void*>(a & ~(uintptr_t)3), a & 2 ? 4 : 2);
        } else {
            if (on) cp_async<sizeof(Elem)>(dst, src, sizeof(Elem));
        }
    }
    // src: the address that the slot was filled from
    __device__ __forceinline__ Elem get(int slot, const T* src) const {
        const Slot s = at[(slot & (DEPTH - 1)) * stride];
        if constexpr (kHalf) {
            const unsigned short h = (unsigned short)(reinterpret_cast<uintptr_t>(src) & 2 ? s >> 16 : s);
            return *reinterpret_cast<const Elem*>(&h);
        } else {
            return s;
        }
    }
};
template <typename T, int V>
constexpr int kSlotBytes = V * sizeof(T) < 4 ? 4 : V * (int)sizeof(T);

// ---- sequences ----------------------------------------------------------------
// Uniform batches (cu == nullptr): nseq rows of `tokens` tokens. Packed: one row of
// `tokens` tokens that holds nseq sequences, the s-th from cu[s] to cu[s + 1].
struct Seqs {
    const int32_t* cu;
    int64_t tokens;
    int32_t nseq;
};
struct Span {
    int64_t row;    // batch row of the sequence's tokens
    int64_t start;  // its first token in that row
    int64_t len;
};

// Offsets read from the device are clamped, so that a wrong table cannot lead out
// of the tensors; check_offsets reports it.
__device__ __forceinline__ int64_t seq_offset(const Seqs& q, int s) {
    const int64_t c = __ldg(q.cu + s);
    return c < 0 ? 0 : (c > q.tokens ? q.tokens : c);
}
__device__ __forceinline__ Span seq_span(const Seqs& q, int s) {
    if (!q.cu) return Span{s, 0, q.tokens};
    const int64_t a = seq_offset(q, s), b = seq_offset(q, s + 1);
    return Span{0, a, b > a ? b - a : 0};
}

// Pieces of `size` tokens, counted from each sequence's own start, are numbered so
// that a number can be found and inverted without a table: piece j of sequence s is
// piece_base(s) + j with piece_base(s) = cu[s] / size + s. Since
// floor(a + b) - floor(a) + 1 >= ceil(b), the numbers of a sequence end before the
// next one's begin; an empty sequence owns one number, and numbers without tokens
// are skipped. Uniform batches use s * ceil(tokens / size).
__host__ __device__ __forceinline__ int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
__device__ __forceinline__ int64_t piece_base(const Seqs& q, int s, int64_t size) {
    if (!q.cu) return (int64_t)s * (q.tokens > size ? ceil_div(q.tokens, size) : 1);
    return seq_offset(q, s) / size + s;
}
__host__ __device__ __forceinline__ int64_t piece_count(const Seqs& q, int64_t size) {
    const int64_t n = q.tokens > size ? ceil_div(q.tokens, size) : 1;
    return q.cu ? n + q.nseq : n * q.nseq;
}
// Sequence and index of a piece number.
__device__ __forceinline__ void piece_find(const Seqs& q, int64_t piece, int64_t size, int& s, int64_t& j) {
    if (!q.cu) {
        const int64_t n = q.tokens > size ? ceil_div(q.tokens, size) : 1;
        s = (int)(piece / n);
        j = piece - s * n;
        return;
    }
    int lo = 0, hi = q.nseq;  // the last s with piece_base(s) <= piece
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (piece_base(q, mid, size) <= piece) lo = mid; else hi = mid;
    }
    s = lo;
    j = piece - piece_base(q, s, size);
    if (j < 0) j = 0;
}
// Last sequence that starts at or before token t of a packed row.
__device__ __forceinline__ int seq_of_token(const Seqs& q, int64_t t) {
    int lo = 0, hi = q.nseq;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (seq_offset(q, mid) <= t) lo = mid; else hi = mid;
    }
    return lo;
}
// One warp of the grid looks the offsets over: 0 first, `tokens` last, never falling.
__device__ __forceinline__ void check_offsets(const Seqs& q, int lane, int site) {
    if (!q.cu) return;
    bool bad = __ldg(q.cu) != 0 || __ldg(q.cu + q.nseq) != q.tokens;
    for (int s = lane; s < q.nseq; s += 32) bad |= __ldg(q.cu + s) > __ldg(q.cu + s + 1);
    if (bad) record_error(PE_ERR_INVALID | (site << 8));
}

// ---- warp reduction --------------------------------------------------------------
// R values a lane, summed over the R lanes that differ in the bits STEP .. STEP * R / 2
// of the lane number: lane bit pattern i of those bits ends with the sum of value i.
// Each level halves the values (R - 1 shuffles in all, against R log2 R for R sums
// that every lane keeps).
template <int R, int STEP>
__device__ __forceinline__ float reduce_scatter(float (&v)[R], int lane) {
#pragma unroll
    for (int m = R / 2; m >= 1; m /= 2) {
        const bool hi = lane & (m * STEP);
#pragma unroll
        for (int i = 0; i < m; ++i) {
            const float send = hi ? v[i] : v[i + m];
            const float keep = hi ? v[i + m] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, m * STEP);
        }
    }
    return v[0];
}

}  // namespace pe

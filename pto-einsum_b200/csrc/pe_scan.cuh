// pe_scan.cuh - what the forward and the backward scan share: parameters, the
// placement of blocks, staging, and the host's checks.
#pragma once

#include "pe_mixer.cuh"

namespace pe {

namespace {

constexpr int kThreads = 128;
constexpr int TS = 16;       // tokens a tile, and between two checkpoints
constexpr int LD = TS + 4;   // row of a [channel][token] tile: 16-byte rows whose float4 reads by
                             // neighbouring channels fall on different banks
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kSiteOffsets = 32, kSiteSlot = 33;

template <typename T>
struct ScanP {
    Seqs seqs;
    int D, N, G, Dg;      // channels, states, groups, channels a group
    int ntile;            // channel tiles a group
    int softplus;
    const T *u, *delta, *z, *B, *C;
    const float *A, *Dw, *bias, *h0;
    int64_t u_sb, u_st, d_sb, d_st, z_sb, z_st, B_sb, B_st, B_sg, C_sb, C_st, C_sg;
    T* out;
    float *state, *ckpt;
    int64_t piece;        // tokens a piece (a multiple of TS, or more than any sequence has)
    float *hloc, *dtsum;  // ws of a split scan: each piece's own last state and sum of dt
};

// Where a block works: channel tile, group and piece.
struct Place {
    int g, c0, nch;        // group, first channel, valid channels
    int s;                 // sequence
    int64_t j;             // piece of the sequence
    int64_t number;        // piece number
    Span sp;
    int64_t t0, t1;        // its tokens, counted from the sequence's start
    bool any;              // false: a number that stands for no piece
};

template <int CH, typename P>
__device__ __forceinline__ Place place_of(const P& p) {
    Place w;
    int64_t b = blockIdx.x;
    const int tile = (int)(b % p.ntile);
    b /= p.ntile;
    w.g = (int)(b % p.G);
    w.number = b / p.G;
    piece_find(p.seqs, w.number, p.piece, w.s, w.j);
    w.sp = seq_span(p.seqs, w.s);
    w.t0 = w.j * p.piece;
    w.t1 = min(w.sp.len, w.t0 + p.piece);
    w.any = w.t0 < w.sp.len || w.j == 0;
    w.c0 = w.g * p.Dg + tile * CH;
    w.nch = min(CH, p.Dg - tile * CH);
    return w;
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
__device__ __forceinline__ f32x2 exp2_2(f32x2 x) {
    float lo, hi;
    unpack2(x, lo, hi);
    return pack2(exp2_fast(lo), exp2_fast(hi));
}

// ---- host -------------------------------------------------------------------------
inline int lanes_for(int64_t states) {
    int l = 1;
    while (4 * l < states) l *= 2;
    return l;
}

inline int check_scan(const pe_scan_args* a) {
    if (!a || a->dtype < PE_F32 || a->dtype > PE_BF16) return PE_ERR_INVALID;
    if (a->batch < 0 || a->tokens < 0 || a->channels < 1 || a->groups < 1 || a->nseq < 0 || a->states < 1)
        return PE_ERR_INVALID;
    if (a->channels % a->groups || (a->cu ? a->batch != 1 : a->nseq != a->batch)) return PE_ERR_INVALID;
    if (a->states > 128 || a->channels > (1 << 24) || a->nseq > (1 << 24)) return PE_ERR_UNSUPPORTED;
    // an empty tensor may have no address
    if (!a->A || (a->tokens && a->batch && (!a->u || !a->delta || !a->B || !a->C))) return PE_ERR_INVALID;
    return PE_OK;
}

inline Seqs seqs_of(const pe_scan_args* a) { return Seqs{a->cu, a->tokens, (int32_t)a->nseq}; }

template <typename T>
ScanP<T> scan_params(const pe_scan_args* a, int ch) {
    ScanP<T> p;
    p.seqs = seqs_of(a);
    p.D = (int)a->channels; p.N = (int)a->states; p.G = (int)a->groups; p.Dg = p.D / p.G;
    p.ntile = (p.Dg + ch - 1) / ch;
    p.softplus = a->softplus != 0;
    p.u = (const T*)a->u; p.delta = (const T*)a->delta; p.z = (const T*)a->z;
    p.B = (const T*)a->B; p.C = (const T*)a->C;
    p.A = a->A; p.Dw = a->D; p.bias = a->delta_bias; p.h0 = a->h0;
    p.u_sb = a->u_sb; p.u_st = a->u_st; p.d_sb = a->delta_sb; p.d_st = a->delta_st;
    p.z_sb = a->z_sb; p.z_st = a->z_st;
    p.B_sb = a->B_sb; p.B_st = a->B_st; p.B_sg = a->B_sg;
    p.C_sb = a->C_sb; p.C_st = a->C_st; p.C_sg = a->C_sg;
    p.out = (T*)a->out; p.state = a->state; p.ckpt = a->ckpt;
    p.piece = (a->tokens / TS + 1) * TS;   // longer than any sequence: one piece each, numbered like it
    p.hloc = p.dtsum = nullptr;
    return p;
}

inline int grid_of(int64_t blocks, unsigned* grid) {
    if (blocks > 0x7fffffffll) return PE_ERR_UNSUPPORTED;
    *grid = (unsigned)blocks;
    return PE_OK;
}

template <typename K, typename P>
int launch(K kernel, const P& p, unsigned grid, int smem, cudaStream_t s) {
    if (smem > 48 * 1024 &&
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return PE_ERR_CUDA;
    kernel<<<grid, kThreads, smem, s>>>(p);
    count_launch();
    return cudaGetLastError() == cudaSuccess ? PE_OK : PE_ERR_CUDA;
}

#define PE_LANES(F, l, ...)                    \
    switch (l) {                               \
        case 1: return F<T, 1>(__VA_ARGS__);   \
        case 2: return F<T, 2>(__VA_ARGS__);   \
        case 4: return F<T, 4>(__VA_ARGS__);   \
        case 8: return F<T, 8>(__VA_ARGS__);   \
        case 16: return F<T, 16>(__VA_ARGS__); \
        default: return F<T, 32>(__VA_ARGS__); \
    }

#define PE_TYPES(F, dtype, ...)                            \
    switch (dtype) {                                       \
        case PE_F32: return F<float>(__VA_ARGS__);         \
        case PE_F16: return F<__half>(__VA_ARGS__);        \
        default: return F<__nv_bfloat16>(__VA_ARGS__);     \
    }

}  // namespace

}  // namespace pe

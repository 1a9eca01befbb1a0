// pe_scan.cuh - what the forward and the backward scan share: parameters, the
// placement of blocks, tiles and staging, and the host's checks.
#pragma once

#include <cfloat>
#include <initializer_list>

#include "pe_mixer.cuh"

namespace pe {

namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int KCK = 64;      // tokens between two checkpoints
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
    // copies to shared memory: rows of these tensors in chunks (see chunk_of), 0 = element by element
    int u_cb, d_cb, z_cb, B_cb, C_cb;
    bool fast, chunks;    // all of them in chunks of 16; of 8 or 16
    bool pairs;           // the results' rows take aligned pairs of elements
    bool longest_first;   // packed sequences are taken in the order of their lengths
    int64_t piece;        // tokens a piece (a multiple of KCK, or more than any sequence has)
    float *hloc, *dtsum;  // ws of a split scan: each piece's own last state and sum of dt

    void split(int64_t tokens) {   // pieces have about one length, and a place of their own in the order
        piece = tokens;
        longest_first = false;
    }
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

// The sequence with `rank` longer ones (equal lengths in order), for up to kThreads of
// them: blocks that take whole sequences of very different lengths start with the longest,
// or the last one to start would end long after the others (17 sequences in 8192 tokens,
// 4096 channels: 253 us, 368 in the order of the table; 60 sequences 306 and 312).
__device__ __forceinline__ int seq_of_rank(const Seqs& q, int rank) {
    __shared__ int found;
    __shared__ int64_t lens[kThreads];
    const int i = threadIdx.x;
    const int64_t len = i < q.nseq ? seq_span(q, i).len : -1;
    if (i < kThreads) lens[i] = len;
    __syncthreads();
    if (i < q.nseq) {
        int longer = 0;
#pragma unroll 8
        for (int j = 0; j < q.nseq; ++j) longer += lens[j] > len || (lens[j] == len && j < i);
        if (longer == rank) found = i;
    }
    __syncthreads();
    return found;
}

template <int CH, typename P>
__device__ __forceinline__ Place place_of(const P& p) {
    Place w;
    int64_t b = blockIdx.x;
    const int tile = (int)(b % p.ntile);
    b /= p.ntile;
    w.g = (int)(b % p.G);
    w.number = b / p.G;
    if (p.longest_first && w.number < p.seqs.nseq) w.number = seq_of_rank(p.seqs, (int)w.number);
    piece_find(p.seqs, w.number, p.piece, w.s, w.j);
    w.sp = seq_span(p.seqs, w.s);
    w.t0 = w.j * p.piece;
    w.t1 = min(w.sp.len, w.t0 + p.piece);
    w.any = w.t0 < w.sp.len || w.j == 0;
    w.c0 = w.g * p.Dg + tile * CH;
    w.nch = min(CH, p.Dg - tile * CH);
    return w;
}

// exp(dt A) with A in units of log2(e). The instruction behind exp2_fast comes out low, by
// 5e-9 of the value on average at arguments down to -0.002, by 2e-8 from there to -1
// (measured against 64 bits); a state that remembers a thousand tokens adds that up a
// thousand times. kLow in the argument takes half of it away, for no instruction more.
constexpr float kLow = 1.7e-8f;
__device__ __forceinline__ f32x2 decay2(f32x2 dt, f32x2 A) { return exp2_2(fma2(dt, A, both(kLow))); }
__device__ __forceinline__ float decay(float dt, float A) { return exp2_fast(fmaf(dt, A, kLow)); }
// A in those units, and finite: where A is -inf the state forgets everything, but a token past the
// end, with dt = 0, has to leave it as it is, and 0 times infinity is neither.
__device__ __forceinline__ float rate(float A) {
    const float a = A * kLog2e;
    return a < -FLT_MAX ? -FLT_MAX : a;
}

// ---- copies to shared memory ------------------------------------------------------
// By the NT threads of the block: cnt (at most ROWS) rows of `width` (at most W) elements
// into rows of W, in chunks of `cb` bytes that arrive asynchronously where the rows are
// aligned for them. Nothing past the width or the count is read; there the tile stays as
// it was.
template <int ROWS, int W, int BYTES, int NT, typename T>
__device__ __forceinline__ void stage_chunks(T* dst, const T* src, int64_t st, int cnt, int width) {
    constexpr int E = BYTES / (int)sizeof(T), PER = W / E;
    static_assert(W % E == 0, "rows of whole chunks");
#pragma unroll 4
    for (int i = threadIdx.x; i < ROWS * PER; i += NT) {
        const int t = i / PER, k = i % PER * E;
        if (t < cnt && k < width)
            cp_async<BYTES>(dst + t * W + k, src + t * st + k, min(BYTES, (width - k) * (int)sizeof(T)));
    }
}
template <int ROWS, int W, int NT = kThreads, typename T>
__device__ __forceinline__ void stage(T* dst, const T* src, int64_t st, int cnt, int width, int cb) {
    constexpr int ROW = W * (int)sizeof(T);
    static_assert(ROW % 8 == 0, "rows of whole chunks");
    if constexpr (ROW % 16 == 0) {
        if (cb == 16) {
            stage_chunks<ROWS, W, 16, NT>(dst, src, st, cnt, width);
            return;
        }
    }
    if (cb >= 8) {
        stage_chunks<ROWS, W, 8, NT>(dst, src, st, cnt, width);
    } else {
#pragma unroll 4
        for (int i = threadIdx.x; i < ROWS * W; i += NT) {
            const int t = i / W, k = i % W;
            if (t < cnt && k < width) dst[i] = load_one(src + t * st + k);
        }
    }
}

// Rows that no chunk fits, element by element in two halves, so that the loads of all
// tensors are on their way together: load() before other work, store() after it.
template <int ROWS, int W, int NT, typename T>
struct Elements {
    static constexpr int J = (ROWS * W + NT - 1) / NT;
    T r[J];
    __device__ __forceinline__ void load(const T* src, int64_t st, int cnt, int width) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int i = threadIdx.x + j * NT, t = i / W, k = i % W;
            if (t < cnt && k < width) r[j] = load_one(src + t * st + k);
        }
    }
    __device__ __forceinline__ void store(T* dst) const {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int i = threadIdx.x + j * NT;
            if (i < ROWS * W) dst[i] = r[j];
        }
    }
};

// ---- host -------------------------------------------------------------------------
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

// Bytes a copy of rows of `width` elements moves at once: the largest of 16 and 8 that a
// row of the tile holds and that divides the base address, the strides and `step` (what
// a block's first element may be a multiple of); 0 where none does.
inline int chunk_of(const void* p, int es, int64_t row_bytes, std::initializer_list<int64_t> strides, int64_t step) {
    for (int cb : {16, 8}) {
        bool ok = row_bytes >= cb && (uintptr_t)p % cb == 0 && step * es % cb == 0;
        for (int64_t s : strides) ok = ok && s * es % cb == 0;
        if (ok) return cb;
    }
    return 0;
}

template <typename T>
ScanP<T> scan_params(const pe_scan_args* a, int ch, int nc) {
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
    p.piece = (a->tokens / KCK + 1) * KCK;   // longer than any sequence: one piece each, numbered like it
    p.longest_first = a->cu && a->nseq > 1 && a->nseq <= kThreads;
    p.hloc = p.dtsum = nullptr;
    const int es = sizeof(T);
    const int64_t step = p.G > 1 ? p.Dg : ch, row = (int64_t)ch * es;   // of a block's first channel
    const int64_t cols = (int64_t)nc * es;
    p.u_cb = chunk_of(p.u, es, row, {p.u_sb, p.u_st, (int64_t)ch}, step);
    p.d_cb = chunk_of(p.delta, es, row, {p.d_sb, p.d_st, (int64_t)ch}, step);
    p.z_cb = p.z ? chunk_of(p.z, es, row, {p.z_sb, p.z_st, (int64_t)ch}, step) : 0;
    p.B_cb = chunk_of(p.B, es, cols, {p.B_sb, p.B_st, p.B_sg}, nc);
    p.C_cb = chunk_of(p.C, es, cols, {p.C_sb, p.C_st, p.C_sg}, nc);
    p.fast = p.u_cb == 16 && p.d_cb == 16 && (!p.z || p.z_cb == 16) && p.B_cb == 16 && p.C_cb == 16;
    p.chunks = p.u_cb && p.d_cb && (!p.z || p.z_cb) && p.B_cb && p.C_cb;
    p.pairs = p.Dg % 2 == 0 && (uintptr_t)p.out % (2 * es) == 0;
    return p;
}

inline int grid_of(int64_t blocks, unsigned* grid) {
    if (blocks > 0x7fffffffll) return PE_ERR_UNSUPPORTED;
    *grid = (unsigned)blocks;
    return PE_OK;
}

template <typename K, typename P>
int launch(K kernel, const P& p, unsigned grid, int smem, cudaStream_t s, int threads = kThreads) {
    if (smem > 40 * 1024 &&   // of the 48 KB that a block has without asking, some are the kernels' static ones
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return PE_ERR_CUDA;
    kernel<<<grid, threads, smem, s>>>(p);
    count_launch();
    return cudaGetLastError() == cudaSuccess ? PE_OK : PE_ERR_CUDA;
}

#define PE_TYPES(F, dtype, ...)                            \
    switch (dtype) {                                       \
        case PE_F32: return F<float>(__VA_ARGS__);         \
        case PE_F16: return F<__half>(__VA_ARGS__);        \
        default: return F<__nv_bfloat16>(__VA_ARGS__);     \
    }

}  // namespace

}  // namespace pe

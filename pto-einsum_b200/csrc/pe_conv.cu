// pe_conv.cu - short causal convolution along the tokens (channels last), its
// gradients and its single-token form, for sm_100a.
//
//   p[t] = bias + sum_k w[k] x[t - (W - 1) + k],   out = p or silu(p)
//   g = dout act'(p),  dx[i] = sum_j w[W - 1 - j] g[i + j],  dw[k] = sum_t g[t] x[t - (W - 1) + k]
//
// All of it is bound by memory: two FMAs a tap against 2 (forward) or 3 (backward)
// elements moved (and, with silu, two special-function operations an element, which is
// three quarters of the memory's time). Times are of a B200, by replays of a captured
// call. A thread owns 16 bytes of channels and walks a
// tile of tokens with the last W - 1 inputs in registers and the next seven on their
// way to its own slots of shared memory, so that each input is read once apart from
// the W - 1 tokens before (after) a tile.
#include "pe_mixer.cuh"

namespace pe {

namespace {

constexpr int DEPTH = 8;      // slots of a thread's queue: seven tokens on their way
constexpr int kBlock = 256;
constexpr int kSiteOffsets = 34, kSiteSlot = 35;

template <typename T>
struct ConvP {
    Seqs seqs;
    int64_t C, CV;            // channels, channel vectors
    int64_t tiles, tile;      // token tiles in all, tokens a tile
    int silu;
    const T *x, *w, *bias, *init;
    int64_t x_sb, x_st;
    T *out, *state;
};

template <typename T, int W, int V>
struct Filter {
    static constexpr int Q = kPairs<V>;
    f32x2 w[W][Q], b[Q];
    // weight [C][W]: the V channels' taps are V W consecutive elements, W loads
    __device__ __forceinline__ void load(const T* weight, const T* bias, int64_t c) {
        Vec<T, V> r[W], rb;
#pragma unroll
        for (int k = 0; k < W; ++k) r[k] = load_vec<T, V>(weight + c * W + k * V);
        if (bias) rb = load_vec<T, V>(bias + c);
#pragma unroll
        for (int k = 0; k < W; ++k) {
            Vec<T, V> tap;
#pragma unroll
            for (int v = 0; v < V; ++v) tap.v[v] = r[(v * W + k) / V].v[(v * W + k) % V];
            widen<T, V>(tap, w[k]);
        }
#pragma unroll
        for (int q = 0; q < Q; ++q) b[q] = 0;
        if (bias) widen<T, V>(rb, b);
    }
    __device__ __forceinline__ void apply(const f32x2 (&win)[W][Q], f32x2 (&p)[Q]) const {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            p[q] = b[q];
#pragma unroll
            for (int k = 0; k < W; ++k) p[q] = fma2(w[k][q], win[k][q], p[q]);
        }
    }
};
template <int W, int Q>
__device__ __forceinline__ void shift(f32x2 (&win)[W][Q]) {
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
#pragma unroll
        for (int q = 0; q < Q; ++q) win[k][q] = win[k + 1][q];
}

// Inputs before token `pos` (counted from the sequence's start): win[j] = x[pos - (W - 1) + j].
template <typename T, int W, int V>
__device__ __forceinline__ void load_before(const ConvP<T>& p, const T* xs, int64_t pos, int s, int64_t c,
                                            f32x2 (&win)[W][kPairs<V>]) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
        const int64_t i = pos - (W - 1) + j;
#pragma unroll
        for (int q = 0; q < kPairs<V>; ++q) win[j][q] = 0;
        if (i >= 0)
            widen<T, V>(load_vec<T, V>(xs + i * p.x_st + c), win[j]);
        else if (p.init)
            widen<T, V>(load_vec<T, V>(p.init + ((int64_t)s * (W - 1) + (W - 1) + i) * p.C + c), win[j]);
    }
}

// 16384 x 4352 bf16 with silu: 56 us, 5.1 TB/s. The copies need no barrier and no register
// while under way: seven inputs in flight a thread at two blocks an SM; loads into
// registers, as many as fit, took 78 us. V = 16 bytes of channels where all rows allow
// it, else one element: 8000 x 2048 and x 2049 bf16 17 and 41 us.
template <typename T, int W, int V>
__global__ void __launch_bounds__(kBlock, 2) conv_fwd(const __grid_constant__ ConvP<T> p) {
    constexpr int Q = kPairs<V>;
    __shared__ __align__(16) unsigned char queue[DEPTH * kBlock * kSlotBytes<T, V>];
    if (blockIdx.x == 0 && threadIdx.x < 32) check_offsets(p.seqs, threadIdx.x, kSiteOffsets);
    int64_t id = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    const int64_t tile = id / p.CV, c = (id - tile * p.CV) * V;
    if (tile >= p.tiles) {
        // the sequences' last W - 1 inputs
        const int64_t s = tile - p.tiles;
        if (!p.state || s >= p.seqs.nseq) return;
        const Span sp = seq_span(p.seqs, (int)s);
        const T* xs = p.x + sp.row * p.x_sb + sp.start * p.x_st;
        f32x2 win[W][Q];
        load_before<T, W, V>(p, xs, sp.len, (int)s, c, win);
#pragma unroll
        for (int j = 0; j < W - 1; ++j) store_vec(p.state + (s * (W - 1) + j) * p.C + c, narrow<T, V>(win[j]));
        return;
    }
    const int64_t per = ceil_div(p.seqs.tokens, p.tile);   // tiles a row
    int64_t t = tile % per * p.tile;
    const int64_t end = min(p.seqs.tokens, t + p.tile);
    const T* xr = p.x + (p.seqs.cu ? 0 : tile / per) * p.x_sb + c;
    // the tile's inputs, DEPTH - 1 tokens ahead: a slot is filled again one token after it was read
    Ring<T, V, DEPTH> ring(queue, kBlock);
    const T* ahead = xr + t * p.x_st;
    int left = (int)(end - t);   // tokens not yet on their way
#pragma unroll
    for (int i = 0; i < DEPTH - 1; ++i, ahead += p.x_st, --left) {
        ring.fetch(i, ahead, left > 0);
        cp_commit();
    }
    Filter<T, W, V> f;
    f.load(p.w, p.bias, c);
    int slot = 0;
    int s = p.seqs.cu ? seq_of_token(p.seqs, t) : (int)(tile / per);
    for (; t < end && s < p.seqs.nseq; ++s) {
        const Span sp = seq_span(p.seqs, s);
        const int64_t stop = min(end, sp.start + sp.len);   // of the tile's tokens in this sequence
        if (stop <= t || sp.start > t) continue;
        T* o = p.out + (sp.row * p.seqs.tokens + t) * p.C + c;
        f32x2 win[W][Q];
        load_before<T, W, V>(p, xr - c + sp.start * p.x_st, t - sp.start, s, c, win);
#pragma unroll 4
        for (; t < stop; ++t, ++slot, o += p.C) {
            cp_wait_but<DEPTH - 2>();
            widen<T, V>(ring.get(slot, xr + t * p.x_st), win[W - 1]);
            ring.fetch(slot + DEPTH - 1, ahead, left > 0);
            cp_commit();
            ahead += p.x_st;
            --left;
            f32x2 y[Q];
            f.apply(win, y);
            if (p.silu) {
#pragma unroll
                for (int q = 0; q < Q; ++q) y[q] = mul2(y[q], sigmoid2(y[q]));
            }
            shift(win);
            store_vec(o, narrow<T, V>(y));
        }
    }
    cp_wait();
}

// ---- backward -------------------------------------------------------------------
template <typename T>
struct ConvGradP {
    ConvP<T> f;
    const T *dout, *dstate;
    int64_t o_sb, o_st;
    T *dx, *dinit;
    float *pw, *pb;     // [blocks along the tokens][C W] and [..][C]
    int bx;             // channel vectors a block (power of two <= 32)
};

// One thread does for its channels and tokens what each of the three results needs: the slope of
// silu from the recomputed sum, dx from the window of g, the sums of dw and dbias in registers to
// the end of the walk, then over the block's threads in order, and over blocks by sum_rows. Bound
// by instructions at few warps: 4 x 2048 x 2048 f16 31 us, 3.2 TB/s; 16384 x 4352 bf16 102 us, 4.2
// TB/s. Eight channels a thread and one block an SM beat four channels and two (51 us against 34,
// both before the loop below had its form without edges): what a token costs beside its channels is
// paid half as often. The tokens inside a tile have a loop without the ends' conditions: 194 us
// with them for 16384 x 4352 and its forward pass, 179 without. Elements (V = 1), forward and
// backward of 8000 x 2049 bf16: 124 us, 50 for x 2048 in 16-byte accesses.
// Blocks an SM holds: by the registers of V channels' taps, sums and windows.
__host__ __device__ constexpr int bwd_blocks(int v) { return v <= 4 ? 2 : 1; }

template <typename T, int W, int V>
__global__ void __launch_bounds__(kBlock, bwd_blocks(V)) conv_bwd(const __grid_constant__ ConvGradP<T> p) {
    constexpr int Q = kPairs<V>;
    // the queues, and once they are empty the block's sums
    extern __shared__ __align__(16) unsigned char shared[];
    const ConvP<T>& f = p.f;
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < 32) check_offsets(f.seqs, threadIdx.x, kSiteOffsets);
    const int by = kBlock / p.bx, x = threadIdx.x % p.bx, y = threadIdx.x / p.bx;
    const int64_t cv = (int64_t)blockIdx.y * p.bx + x, c = cv * V;
    const int64_t tile = (int64_t)blockIdx.x * by + y;
    f32x2 dw[W][Q], db[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        db[q] = 0;
#pragma unroll
        for (int k = 0; k < W; ++k) dw[k][q] = 0;
    }
    if (cv < f.CV && tile < f.tiles) {
        const int64_t per = ceil_div(f.seqs.tokens, f.tile);
        int64_t t = tile % per * f.tile;
        const int64_t end = min(f.seqs.tokens, t + f.tile), row = f.seqs.cu ? 0 : tile / per;
        const T* xr = f.x + row * f.x_sb + c;
        const T* dor = p.dout + row * p.o_sb + c;
        Ring<T, V, DEPTH> rx(shared, kBlock), ro(shared + DEPTH * kBlock * kSlotBytes<T, V>, kBlock);
        Filter<T, W, V> flt;
        flt.load(f.w, f.bias, c);
        int s = f.seqs.cu ? seq_of_token(f.seqs, t) : (int)row;
        for (; t < end && s < f.seqs.nseq; ++s) {
            const Span sp = seq_span(f.seqs, s);
            const int64_t fin = sp.start + sp.len, stop = min(end, fin);
            if (stop <= t || sp.start > t) continue;
            T* dx = p.dx + sp.row * f.seqs.tokens * f.C + c;
            // g of the tokens t .. stop + W - 2 gives dx of t .. stop - 1 (and of the
            // inputs before the sequence where t starts it)
            const int64_t last = stop + W - 1, have = min(last, fin);
            int64_t ahead = t;
#pragma unroll
            for (int i = 0; i < DEPTH - 1; ++i, ++ahead) {
                rx.fetch(i, xr + ahead * f.x_st, ahead < have);
                ro.fetch(i, dor + ahead * p.o_st, ahead < have);
                cp_commit();
            }
            f32x2 win[W][Q], g[W][Q];   // inputs and g of the tokens up to the current one
            load_before<T, W, V>(f, xr - c + sp.start * f.x_st, t - sp.start, s, c, win);
#pragma unroll
            for (int k = 0; k < W; ++k)
#pragma unroll
                for (int q = 0; q < Q; ++q) g[k][q] = 0;
            int slot = 0;
            // EDGE false: a token of the tile and of the sequence whose g completes the dx of an
            // input of the tile, which is none of the last state's
            auto token = [&](int64_t k, auto edge) {
                constexpr bool EDGE = decltype(edge)::value;
                cp_wait_but<DEPTH - 2>();
                widen<T, V>(rx.get(slot, xr + k * f.x_st), win[W - 1]);
                widen<T, V>(ro.get(slot, dor + k * p.o_st), g[W - 1]);
                rx.fetch(slot + DEPTH - 1, xr + ahead * f.x_st, ahead < have);
                ro.fetch(slot + DEPTH - 1, dor + ahead * p.o_st, ahead < have);
                cp_commit();
                ++slot;
                ++ahead;
                if (!EDGE || k < fin) {
                    if (f.silu) {
                        f32x2 a[Q];
                        flt.apply(win, a);
#pragma unroll
                        for (int q = 0; q < Q; ++q)
                            g[W - 1][q] = mul2(g[W - 1][q], silu_slope2(a[q], sigmoid2(a[q])));
                    }
                    if (!EDGE || k < stop) {   // the tile's own: into the sums
#pragma unroll
                        for (int q = 0; q < Q; ++q) {
                            db[q] = add2(db[q], g[W - 1][q]);
#pragma unroll
                            for (int j = 0; j < W; ++j) dw[j][q] = fma2(g[W - 1][q], win[j][q], dw[j][q]);
                        }
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < Q; ++q) g[W - 1][q] = 0;
                }
                shift(win);
                // dx of the input W - 1 tokens back, whose sum this completes
                f32x2 d[Q];
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    d[q] = mul2(flt.w[W - 1][q], g[0][q]);
#pragma unroll
                    for (int j = 1; j < W; ++j) d[q] = fma2(flt.w[W - 1 - j][q], g[j][q], d[q]);
                }
                shift(g);
                const int64_t i0 = k - (W - 1);
                T* to = dx + i0 * f.C;
                if constexpr (EDGE) {
                    const int64_t pos = i0 - sp.start;
                    const bool first = pos < 0 && t == sp.start && p.dinit;   // an input before the sequence
                    if (i0 < t && !first) return;
                    const int64_t j = pos + W - 1 - sp.len;                    // its place in the last state
                    if (p.dstate && j >= 0) {
                        f32x2 e[Q];
                        widen<T, V>(load_vec<T, V>(p.dstate + ((int64_t)s * (W - 1) + j) * f.C + c), e);
#pragma unroll
                        for (int q = 0; q < Q; ++q) d[q] = add2(d[q], e[q]);
                    }
                    if (first) to = p.dinit + ((int64_t)s * (W - 1) + W - 1 + pos) * f.C + c;
                }
                store_vec(to, narrow<T, V>(d));
            };
            int64_t k = t;
#pragma unroll 1
            for (const int64_t head = min(stop, t + W - 1); k < head; ++k) token(k, std::true_type());
#pragma unroll(V == 1 ? 4 : 2)
            for (; k < stop; ++k) token(k, std::false_type());
#pragma unroll 1
            for (; k < last; ++k) token(k, std::true_type());
            cp_wait();
            t = stop;
        }
    }
    // the block's tiles, in order
    __syncthreads();
    float* red = reinterpret_cast<float*>(shared);   // [(W + 1) V][kBlock]
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int k = 0; k <= W; ++k) {
            float h[2];
            unpack2(k < W ? dw[k < W ? k : 0][v / 2] : db[v / 2], h[0], h[1]);
            red[(k * V + v) * kBlock + threadIdx.x] = h[v % 2];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < (W + 1) * V * p.bx; i += kBlock) {
        const int xi = i % p.bx, kv = i / p.bx, k = kv / V, v = kv % V;
        const int64_t ci = ((int64_t)blockIdx.y * p.bx + xi) * V + v;
        if (ci >= f.C) continue;
        float a = 0.0f;
        for (int r = 0; r < by; ++r) a += red[kv * kBlock + r * p.bx + xi];
        if (k < W)
            p.pw[(int64_t)blockIdx.x * f.C * W + ci * W + k] = a;
        else
            p.pb[(int64_t)blockIdx.x * f.C + ci] = a;
    }
}

// dinit of the sequences without tokens: their last state is their first.
template <typename T>
__global__ void __launch_bounds__(kBlock) conv_empty(Seqs q, int64_t n, const T* dstate, T* dinit) {
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (i >= n * q.nseq || seq_span(q, (int)(i / n)).len) return;
    dinit[i] = dstate ? dstate[i] : from_float<T>(0.0f);
}

// ---- one token --------------------------------------------------------------------
template <typename T>
struct ConvStepP {
    int64_t C, CV, batch, slots, x_sb;
    const int32_t* s32;
    const int64_t* s64;
    int silu;
    const T *x, *w, *bias;
    T *state, *out;
};

// One thread a request's V channels, all its loads on their way at once. Bound by memory
// (the state, read and written, and x) and at few requests by latency: 512 x 4352 f16 in
// slots 8.4 us, 4.2 TB/s.
template <typename T, int W, int V>
__global__ void __launch_bounds__(128) conv_step(const __grid_constant__ ConvStepP<T> p) {
    constexpr int Q = kPairs<V>;
    const int64_t id = (int64_t)blockIdx.x * 128 + threadIdx.x;
    const int64_t b = id / p.CV, c = (id - b * p.CV) * V;
    if (b >= p.batch) return;
    int64_t slot = b;
    if (p.s32) slot = __ldg(p.s32 + b);
    if (p.s64) slot = __ldg(p.s64 + b);
    f32x2 y[Q];
    if (slot < 0 || slot >= p.slots) {
        if (slot >= 0 && c == 0) record_error(PE_ERR_INVALID | (kSiteSlot << 8));
#pragma unroll
        for (int q = 0; q < Q; ++q) y[q] = 0;
        store_vec(p.out + b * p.C + c, narrow<T, V>(y));
        return;
    }
    T* st = p.state + slot * (W - 1) * p.C + c;
    Vec<T, V> raw[W];
#pragma unroll
    for (int k = 0; k < W - 1; ++k) raw[k] = *reinterpret_cast<const Vec<T, V>*>(st + k * p.C);
    raw[W - 1] = load_vec<T, V>(p.x + b * p.x_sb + c);
    Filter<T, W, V> f;
    f.load(p.w, p.bias, c);
    f32x2 win[W][Q];
#pragma unroll
    for (int k = 0; k < W; ++k) widen<T, V>(raw[k], win[k]);
    f.apply(win, y);
    if (p.silu) {
#pragma unroll
        for (int q = 0; q < Q; ++q) y[q] = mul2(y[q], sigmoid2(y[q]));
    }
#pragma unroll
    for (int k = 0; k < W - 1; ++k) store_vec(st + k * p.C, raw[k + 1]);
    store_vec(p.out + b * p.C + c, narrow<T, V>(y));
}

// ---- host -------------------------------------------------------------------------
int check_conv(const pe_conv_args* a) {
    if (!a || a->dtype < PE_F32 || a->dtype > PE_BF16 || a->width < 2 || a->width > 4) return PE_ERR_INVALID;
    if (a->batch < 0 || a->tokens < 0 || a->channels < 1 || a->nseq < 0) return PE_ERR_INVALID;
    if (a->cu ? a->batch != 1 : a->nseq != a->batch) return PE_ERR_INVALID;
    if (a->channels > (1 << 24) || a->nseq > (1 << 24)) return PE_ERR_UNSUPPORTED;
    if (!a->weight || (a->tokens && a->batch && !a->x)) return PE_ERR_INVALID;
    return PE_OK;
}

int elem_bytes(int64_t dtype) { return dtype == PE_F32 ? 4 : 2; }

// 16-byte accesses: every row of every tensor starts on a 16-byte boundary.
bool wide(int64_t dtype, int64_t channels, std::initializer_list<const void*> ptrs,
          std::initializer_list<int64_t> strides) {
    const int64_t v = 16 / elem_bytes(dtype);
    if (channels % v) return false;
    for (const void* q : ptrs)
        if ((uintptr_t)q % 16) return false;
    for (int64_t st : strides)
        if (st % v) return false;
    return true;
}

template <typename T>
ConvP<T> conv_params(const pe_conv_args* a, int v, int64_t tile) {
    ConvP<T> p;
    p.seqs = Seqs{a->cu, a->tokens, (int32_t)a->nseq};
    p.C = a->channels; p.CV = a->channels / v;
    p.tile = tile;
    p.tiles = ceil_div(a->tokens, tile) * a->batch;
    p.silu = a->silu != 0;
    p.x = (const T*)a->x; p.w = (const T*)a->weight; p.bias = (const T*)a->bias; p.init = (const T*)a->init;
    p.x_sb = a->x_sb; p.x_st = a->x_st;
    p.out = (T*)a->out; p.state = (T*)a->state;
    return p;
}

// Tokens a thread walks: whole waves of the blocks an SM holds, at most `most` tokens each
// (the W - 1 tokens read again, the filter and the filling of the queue weigh less on a
// longer walk, the backward pass's sums too; a last wave that is not full costs as much as
// one that is), at least 4. by: a block's threads along the tokens, where the block is laid
// out by channels. Forward, bf16, by this rule (at most 64), by 8, 64 and 256 tokens:
// 300 x 1024 6, 6, 17, 43 us; 8192 x 2048 17, 23, 21, 55; 16384 x 4352 56, 93, 58, 62. With the
// backward pass (at most 256): 17, 19, 46, 109; 50, 99, 55, 155; 158, 388, 183, 165.
int64_t tile_of(const pe_conv_args* a, int64_t columns, int resident, int by, int64_t most) {
    const int64_t rows = a->batch, slots = (int64_t)num_sms() * resident, threads = slots * kBlock;
    const int64_t cells = a->tokens * rows * columns, waves = ceil_div(cells, most * threads);
    if (!waves) return 4;
    int64_t tile = ceil_div(cells, waves * threads);
    if (by > 1) {   // blocks are whole: lengthen the walk until they fit
        const int64_t per = ceil_div(columns, kBlock / by);
        while (tile < most && ceil_div(ceil_div(a->tokens, tile) * rows, by) * per > waves * slots) ++tile;
    }
    return tile < 4 ? 4 : tile;
}

template <typename T, int W, int V>
int conv_run(const pe_conv_args* a, cudaStream_t s) {
    const ConvP<T> p = conv_params<T>(a, V, tile_of(a, a->channels / V, 2, 1, 64));
    const int64_t ids = (p.tiles + (p.state ? a->nseq : 0)) * p.CV, blocks = ceil_div(ids, kBlock);
    if (blocks > 0x7fffffffll) return PE_ERR_UNSUPPORTED;
    if (!blocks) return PE_OK;
    conv_fwd<T, W, V><<<(unsigned)blocks, kBlock, 0, s>>>(p);
    count_launch();
    return cudaGetLastError() == cudaSuccess ? PE_OK : PE_ERR_CUDA;
}

struct ConvGradShape {
    int bx;
    int64_t tile, rows;   // tokens a thread, blocks along the tokens
};
ConvGradShape grad_shape(const pe_conv_args* a, int v) {
    const int64_t cv = a->channels / v;
    ConvGradShape g{1, 4, 0};
    while (g.bx < 32 && g.bx < cv) g.bx *= 2;
    g.tile = tile_of(a, cv, bwd_blocks(v), kBlock / g.bx, 256);
    g.rows = ceil_div(ceil_div(a->tokens, g.tile) * a->batch, kBlock / g.bx);
    return g;
}

template <typename T, int W, int V>
int conv_grad_run(const pe_conv_grad_args* g, cudaStream_t s) {
    const pe_conv_args* a = &g->fwd;
    const ConvGradShape sh = grad_shape(a, V);
    ConvGradP<T> p;
    p.f = conv_params<T>(a, V, sh.tile);
    p.dout = (const T*)g->dout; p.dstate = (const T*)g->dstate;
    p.o_sb = g->dout_sb; p.o_st = g->dout_st;
    p.dx = (T*)g->dx; p.dinit = (T*)g->dinit;
    p.pw = (float*)g->ws;
    p.pb = p.pw + sh.rows * a->channels * W;
    p.bx = sh.bx;
    const int64_t cblocks = ceil_div(p.f.CV, sh.bx);
    if (sh.rows > 0x7fffffffll || cblocks > 65535) return PE_ERR_UNSUPPORTED;
    if (sh.rows) {
        const int queues = 2 * DEPTH * kBlock * kSlotBytes<T, V>, sums = (W + 1) * V * kBlock * 4;
        const int smem = queues > sums ? queues : sums;
        if (smem > 48 * 1024 && cudaFuncSetAttribute(conv_bwd<T, W, V>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                     smem) != cudaSuccess)
            return PE_ERR_CUDA;
        conv_bwd<T, W, V><<<dim3((unsigned)sh.rows, (unsigned)cblocks), kBlock, smem, s>>>(p);
        count_launch();
        if (cudaGetLastError() != cudaSuccess) return PE_ERR_CUDA;
    }
    const int64_t n = (W - 1) * a->channels;
    if (g->dinit && a->nseq && (a->cu || a->tokens == 0)) {
        conv_empty<T><<<(unsigned)ceil_div(n * a->nseq, kBlock), kBlock, 0, s>>>(p.f.seqs, n, p.dstate, p.dinit);
        count_launch();
        if (cudaGetLastError() != cudaSuccess) return PE_ERR_CUDA;
    }
    const SumJob sums[2] = {{p.pw, sh.rows, a->channels * W, (int)a->dtype, g->dweight},
                            {p.pb, sh.rows, a->channels, (int)a->dtype, g->dbias}};
    return sum_rows(sums, 2, s);
}

template <typename T, int W, int V>
int conv_step_run(const pe_conv_step_args* a, cudaStream_t s) {
    ConvStepP<T> p;
    p.C = a->channels; p.CV = a->channels / V; p.batch = a->batch; p.slots = a->slots; p.x_sb = a->x_sb;
    p.s32 = a->slots32; p.s64 = a->slots64;
    p.silu = a->silu != 0;
    p.x = (const T*)a->x; p.w = (const T*)a->weight; p.bias = (const T*)a->bias;
    p.state = (T*)a->state; p.out = (T*)a->out;
    const int64_t blocks = ceil_div(p.batch * p.CV, 128);
    if (blocks > 0x7fffffffll) return PE_ERR_UNSUPPORTED;
    conv_step<T, W, V><<<(unsigned)blocks, 128, 0, s>>>(p);
    count_launch();
    return cudaGetLastError() == cudaSuccess ? PE_OK : PE_ERR_CUDA;
}

#define PE_CONV_W(F, T, V, w, ...)                    \
    switch (w) {                                      \
        case 2: return F<T, 2, V>(__VA_ARGS__);       \
        case 3: return F<T, 3, V>(__VA_ARGS__);       \
        default: return F<T, 4, V>(__VA_ARGS__);      \
    }
template <typename T, int V>
int conv_w(const pe_conv_args* a, cudaStream_t s) { PE_CONV_W(conv_run, T, V, a->width, a, s) }
template <typename T, int V>
int conv_grad_w(const pe_conv_grad_args* a, cudaStream_t s) { PE_CONV_W(conv_grad_run, T, V, a->fwd.width, a, s) }
template <typename T, int V>
int conv_step_w(const pe_conv_step_args* a, cudaStream_t s) { PE_CONV_W(conv_step_run, T, V, a->width, a, s) }

#define PE_CONV_T(F, dtype, vec, ...)                                                               \
    switch (dtype) {                                                                                \
        case PE_F32: return vec ? F<float, 4>(__VA_ARGS__) : F<float, 1>(__VA_ARGS__);              \
        case PE_F16: return vec ? F<__half, 8>(__VA_ARGS__) : F<__half, 1>(__VA_ARGS__);            \
        default: return vec ? F<__nv_bfloat16, 8>(__VA_ARGS__) : F<__nv_bfloat16, 1>(__VA_ARGS__);  \
    }
int conv_any(const pe_conv_args* a, bool vec, cudaStream_t s) { PE_CONV_T(conv_w, a->dtype, vec, a, s) }
int conv_grad_any(const pe_conv_grad_args* a, bool vec, cudaStream_t s) {
    PE_CONV_T(conv_grad_w, a->fwd.dtype, vec, a, s)
}
int conv_step_any(const pe_conv_step_args* a, bool vec, cudaStream_t s) { PE_CONV_T(conv_step_w, a->dtype, vec, a, s) }

bool grad_wide(const pe_conv_grad_args* g) {
    const pe_conv_args* a = &g->fwd;
    return wide(a->dtype, a->channels, {a->x, a->weight, a->bias, a->init, g->dout, g->dstate, g->dx, g->dinit},
                {a->x_sb, a->x_st, g->dout_sb, g->dout_st});
}

}  // namespace

int causal_conv(const pe_conv_args* a, cudaStream_t s) {
    if (int rc = check_conv(a)) return rc;
    if (a->tokens && a->batch && !a->out) return PE_ERR_INVALID;
    return conv_any(a, wide(a->dtype, a->channels, {a->x, a->weight, a->bias, a->init, a->out, a->state}, {a->x_sb, a->x_st}), s);
}

int64_t conv_grad_ws_bytes(const pe_conv_grad_args* g) {
    if (!g || check_conv(&g->fwd) != PE_OK) return 0;
    const pe_conv_args* a = &g->fwd;
    // enough for either width of the loads: the size does not depend on addresses
    const int v = 16 / elem_bytes(a->dtype);
    const int64_t rows = grad_shape(a, 1).rows, wide_rows = a->channels % v ? rows : grad_shape(a, v).rows;
    return (rows > wide_rows ? rows : wide_rows) * a->channels * (a->width + 1) * 4;
}

int causal_conv_grad(const pe_conv_grad_args* g, cudaStream_t s) {
    if (!g) return PE_ERR_INVALID;
    if (int rc = check_conv(&g->fwd)) return rc;
    if (!g->dweight || (g->fwd.tokens && g->fwd.batch && (!g->dout || !g->dx))) return PE_ERR_INVALID;
    const int64_t need = conv_grad_ws_bytes(g);
    if (need && (!g->ws || g->ws_bytes < need)) return PE_ERR_WORKSPACE;
    return conv_grad_any(g, grad_wide(g), s);
}

int causal_conv_step(const pe_conv_step_args* a, cudaStream_t s) {
    if (!a || a->dtype < PE_F32 || a->dtype > PE_BF16 || a->width < 2 || a->width > 4 || a->batch < 0 ||
        a->channels < 1 || a->slots < 0)
        return PE_ERR_INVALID;
    if (a->batch == 0) return PE_OK;
    if (!a->x || !a->weight || !a->state || !a->out) return PE_ERR_INVALID;
    return conv_step_any(a, wide(a->dtype, a->channels, {a->x, a->weight, a->bias, a->state, a->out}, {a->x_sb}), s);
}

int conv_device_error(bool clear) {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_device_error, sizeof(int)) != cudaSuccess) return -1;
    if (v && clear) cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
    return v;
}

}  // namespace pe

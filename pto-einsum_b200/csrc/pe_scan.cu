// pe_scan.cu - selective state space scan: prompts (forward) and single tokens,
// for sm_100a.
//
//   h[n] = exp(dt A[n]) h[n] + dt u B[n],   y = sum_n C[n] h[n] + D u
//
// per channel, dt = softplus(delta + bias). A thread keeps four states of one
// channel in registers; LPC = 1 .. 32 neighbouring lanes share a channel (4 LPC >=
// states). Tokens go through in tiles of 16: what depends on (token, channel) alone
// (softplus, the gate) is computed once by all threads of the block and passed in
// shared memory, and so are B and C in fp32; the sums over states of 16 tokens are
// reduced together (reduce_scatter: LPC - 1 shuffles for LPC tokens).
#include <cmath>

#include "pe_scan.cuh"

namespace pe {

namespace {

// ---- forward --------------------------------------------------------------------
// What a thread has loaded of a tile: I items of four tokens of one channel, and its
// part of the tile's B and C. Loads of the next tile are issued before the current
// one's recurrence and used after it.
template <typename T, int LPC, bool STATE_ONLY>
struct TileRegs {
    static constexpr int CH = kThreads / LPC, I = LPC < 4 ? 4 / LPC : 1, J = LPC * 4 * TS / kThreads > 0 ? LPC * 4 * TS / kThreads : 1;
    T d[I][4], u[I][4], z[STATE_ONLY ? 1 : I][4];
    T b[J], c[STATE_ONLY ? 1 : J];

    __device__ __forceinline__ void load(const ScanP<T>& p, const Place& w, const T* up, const T* dp, const T* zp,
                                         const T* Bp, const T* Cp, int64_t at, int cnt) {
        constexpr int NP = 4 * LPC;
        const int tid = threadIdx.x;
#pragma unroll
        for (int k = 0; k < I; ++k) {
            const int it = tid + k * kThreads, ic = it % CH, t4 = it / CH * 4;
            const int64_t cc = w.c0 + ic;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = ic < w.nch && t4 + i < cnt;
                const int64_t t = at + t4 + i;
                d[k][i] = in ? __ldg(dp + t * p.d_st + cc) : from_float<T>(0.0f);
                u[k][i] = in ? __ldg(up + t * p.u_st + cc) : from_float<T>(0.0f);
                if (!STATE_ONLY) z[k][i] = in && zp ? __ldg(zp + t * p.z_st + cc) : from_float<T>(0.0f);
            }
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int i = tid + j * kThreads, t = i / NP, n = i % NP;
            const bool in = t < cnt && n < p.N;
            b[j] = in ? __ldg(Bp + (at + t) * p.B_st + n) : from_float<T>(0.0f);
            if (!STATE_ONLY) c[j] = in ? __ldg(Cp + (at + t) * p.C_st + n) : from_float<T>(0.0f);
        }
    }
};

// STATE_ONLY: a piece's last state from a zero start and its sum of dt (first half of
// a split scan); else the whole, starting from what the sequence's earlier pieces left.
template <typename T, int LPC, bool STATE_ONLY>
__global__ void __launch_bounds__(kThreads, LPC == 4 || LPC == 8 ? 4 : 2) scan_fwd(const __grid_constant__ ScanP<T> p) {
    constexpr int CH = kThreads / LPC, NP = 4 * LPC, R = LPC < TS ? LPC : TS;
    using Regs = TileRegs<T, LPC, STATE_ONLY>;
    constexpr int I = Regs::I, J = Regs::J, BUF = (STATE_ONLY ? 2 : 3) * CH * LD + (STATE_ONLY ? 1 : 2) * TS * NP;
    extern __shared__ __align__(16) float smem[];   // two buffers: dt, dt u, y [CH][LD] and B, C [TS][NP]
    const int tid = threadIdx.x, lane = tid & 31;
    if (blockIdx.x == 0 && tid < 32) check_offsets(p.seqs, lane, kSiteOffsets);
    const Place w = place_of<CH>(p);
    if (!w.any || (STATE_ONLY && w.t1 == w.sp.len)) return;   // nothing starts from the last piece's state
    const int ch = tid / LPC, q = tid % LPC, c = w.c0 + ch, n0 = 4 * q;
    const bool live = ch < w.nch;
    const int64_t tok = w.sp.start;

    float A[4], h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool in = live && n0 + i < p.N;
        A[i] = in ? __ldg(p.A + (int64_t)c * p.N + n0 + i) * kLog2e : 0.0f;
        h[i] = 0.0f;
    }
    const int64_t DN = (int64_t)p.D * p.N, cn = (int64_t)c * p.N + n0;
    const T* u = p.u + w.sp.row * p.u_sb;
    const T* delta = p.delta + w.sp.row * p.d_sb;
    const T* z = p.z ? p.z + w.sp.row * p.z_sb : nullptr;
    const T* B = p.B + w.sp.row * p.B_sb + w.g * p.B_sg;
    const T* C = p.C + w.sp.row * p.C_sb + w.g * p.C_sg;
    T* out = STATE_ONLY ? nullptr : p.out + (w.sp.row * p.seqs.tokens) * p.D;
    Regs r;
    r.load(p, w, u, delta, z, B, C, tok + w.t0, (int)min((int64_t)TS, w.t1 - w.t0));
    float bias[I], Dw[I];
#pragma unroll
    for (int k = 0; k < I; ++k) {
        const int ic = (tid + k * kThreads) % CH;
        bias[k] = p.bias && ic < w.nch ? __ldg(p.bias + w.c0 + ic) : 0.0f;
        Dw[k] = !STATE_ONLY && p.Dw && ic < w.nch ? __ldg(p.Dw + w.c0 + ic) : 0.0f;
    }
    if (!STATE_ONLY) {
        const float* from = p.hloc ? p.hloc + w.number * DN : p.h0 ? p.h0 + w.s * DN : nullptr;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (from && live && n0 + i < p.N) h[i] = from[cn + i];
    }
    const f32x2 A01 = pack2(A[0], A[1]), A23 = pack2(A[2], A[3]);
    f32x2 h01 = pack2(h[0], h[1]), h23 = pack2(h[2], h[3]);
    float dtsum = 0.0f;
    float add[STATE_ONLY ? 1 : I][4], gate[STATE_ONLY ? 1 : I][4];   // of the tile before: D u and silu(z)
    int buf = 0, last = 0;
    float* ckpt = !STATE_ONLY && p.ckpt && live ? p.ckpt + (piece_base(p.seqs, w.s, TS) + w.t0 / TS) * DN + cn : nullptr;

    // out of the tile that ended at token `end`: (y + D u) silu(z)
    auto finish = [&](int64_t at, int cnt, const float* sy) {
#pragma unroll
        for (int k = 0; k < I; ++k) {
            const int it = tid + k * kThreads, ic = it % CH, t4 = it / CH * 4;
            if (it >= CH * (TS / 4) || ic >= w.nch) continue;
            const float4 y4 = *reinterpret_cast<const float4*>(sy + ic * LD + t4);
            const float yv[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (t4 + i < cnt)
                    out[(at + t4 + i) * p.D + w.c0 + ic] = from_float<T>((yv[i] + add[k][i]) * gate[k][i]);
        }
    };

    for (int64_t t = w.t0; t < w.t1; t += TS) {
        const int cnt = (int)min((int64_t)TS, w.t1 - t);
        const int64_t at = tok + t;
        float* sdt = smem + buf * BUF;
        float* sx = sdt + CH * LD;
        float* sB = sx + CH * LD;
        float* sC = sB + TS * NP;
        float* sy = sC + TS * NP;
        float gadd[STATE_ONLY ? 1 : I][4], ggate[STATE_ONLY ? 1 : I][4];
#pragma unroll
        for (int k = 0; k < I; ++k) {
            const int it = tid + k * kThreads, ic = it % CH, t4 = it / CH * 4;
            float dt[4], x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float uv = to_float(r.u[k][i]);
                dt[i] = to_float(r.d[k][i]) + bias[k];
                if (p.softplus) dt[i] = softplusf(dt[i]);
                x[i] = dt[i] * uv;
                if (!STATE_ONLY) {
                    const float zv = to_float(r.z[k][i]);
                    gadd[k][i] = Dw[k] * uv;
                    ggate[k][i] = z ? zv * sigmoidf(zv) : 1.0f;
                }
            }
            if (it < CH * (TS / 4)) {
                *reinterpret_cast<float4*>(sdt + ic * LD + t4) = make_float4(dt[0], dt[1], dt[2], dt[3]);
                *reinterpret_cast<float4*>(sx + ic * LD + t4) = make_float4(x[0], x[1], x[2], x[3]);
            }
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int i = tid + j * kThreads;
            if (i < TS * NP) {
                sB[i] = to_float(r.b[j]);
                if (!STATE_ONLY) sC[i] = to_float(r.c[j]);
            }
        }
        __syncthreads();
        if (!STATE_ONLY && t > w.t0) finish(at - TS, last, smem + (buf ^ 1) * BUF + 2 * CH * LD + 2 * TS * NP);
        if (t + TS < w.t1)
            r.load(p, w, u, delta, z, B, C, at + TS, (int)min((int64_t)TS, w.t1 - t - TS));
        if (!STATE_ONLY) {
#pragma unroll
            for (int k = 0; k < I; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) add[k][i] = gadd[k][i], gate[k][i] = ggate[k][i];
            if (ckpt) {
                unpack2(h01, h[0], h[1]);
                unpack2(h23, h[2], h[3]);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n0 + i < p.N) ckpt[i] = h[i];
                ckpt += DN;
            }
        }
        float y[TS];
        auto token = [&](int k, float dt, float x) {
            const f32x2 dt2 = pack2(dt, dt), x2 = pack2(x, x);
            const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(sB + k * NP + n0);
            h01 = fma2(exp2_2(mul2(dt2, A01)), h01, mul2(x2, b.x));
            h23 = fma2(exp2_2(mul2(dt2, A23)), h23, mul2(x2, b.y));
            if (STATE_ONLY) {
                dtsum += dt;
            } else {
                const ulonglong2 cv = *reinterpret_cast<const ulonglong2*>(sC + k * NP + n0);
                float lo, hi;
                unpack2(fma2(cv.y, h23, mul2(cv.x, h01)), lo, hi);
                y[k] = lo + hi;
            }
        };
        if (cnt == TS) {
#pragma unroll
            for (int t4 = 0; t4 < TS; t4 += 4) {
                const float4 d4 = *reinterpret_cast<const float4*>(sdt + ch * LD + t4);
                const float4 x4 = *reinterpret_cast<const float4*>(sx + ch * LD + t4);
                token(t4, d4.x, x4.x);
                token(t4 + 1, d4.y, x4.y);
                token(t4 + 2, d4.z, x4.z);
                token(t4 + 3, d4.w, x4.w);
            }
        } else {
#pragma unroll
            for (int k = 0; k < TS; ++k) {
                y[k] = 0.0f;
                if (k < cnt) token(k, sdt[ch * LD + k], sx[ch * LD + k]);
            }
        }
        if (!STATE_ONLY) {
#pragma unroll
            for (int k = 0; k < TS; k += R) {
                float v[R];
#pragma unroll
                for (int i = 0; i < R; ++i) v[i] = y[k + i];
                float sum = reduce_scatter<R, 1>(v, lane);
                if (LPC > R) sum += __shfl_xor_sync(0xffffffffu, sum, R);
                if (q < R) sy[ch * LD + k + q] = sum;
            }
        }
        last = cnt;
        buf ^= 1;
    }
    if (!STATE_ONLY && w.t1 > w.t0) {
        __syncthreads();
        finish(tok + w.t0 + (w.t1 - w.t0 - 1) / TS * TS, last, smem + (buf ^ 1) * BUF + 2 * CH * LD + 2 * TS * NP);
    }
    if (!live) return;
    unpack2(h01, h[0], h[1]);
    unpack2(h23, h[2], h[3]);
    if (STATE_ONLY) {
        if (q == 0) p.dtsum[w.number * p.D + c] = dtsum;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n0 + i < p.N) p.hloc[w.number * DN + cn + i] = h[i];
    } else if (p.state && w.t1 == w.sp.len) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n0 + i < p.N) p.state[w.s * DN + cn + i] = h[i];
    }
}

// Between the halves of a split scan: each piece's own last state gives way to the state
// before the piece. One thread a (sequence, channel, state); the products exp(A sum dt)
// do not depend on one another, so the loads of eight pieces are in flight together.
template <typename T>
__global__ void __launch_bounds__(kThreads) scan_carry(const __grid_constant__ ScanP<T> p) {
    const int64_t DN = (int64_t)p.D * p.N, i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= DN) return;
    const int s = blockIdx.y;
    const int64_t len = seq_span(p.seqs, s).len, base = piece_base(p.seqs, s, p.piece);
    const int64_t n = len > p.piece ? ceil_div(len, p.piece) : 1;
    const int c = (int)(i / p.N);
    const float A = __ldg(p.A + i) * kLog2e;
    float h = p.h0 ? __ldg(p.h0 + s * DN + i) : 0.0f;
    float* hp = p.hloc + base * DN + i;
    const float* sp = p.dtsum + base * p.D + c;
    for (int64_t k0 = 0; k0 < n; k0 += 8) {
        float own[8], keep[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k0 + k < n - 1) {
                own[k] = hp[(k0 + k) * DN];
                keep[k] = exp2_fast(A * __ldg(sp + (k0 + k) * p.D));
            }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k0 + k < n) {
                hp[(k0 + k) * DN] = h;
                if (k0 + k < n - 1) h = fmaf(keep[k], h, own[k]);
            }
    }
}

// ---- one token --------------------------------------------------------------------
template <typename T>
struct StepP {
    int64_t batch, slots;
    int D, N, G, Dg, softplus;
    const int32_t* s32;
    const int64_t* s64;
    const T *u, *delta, *z, *B, *C;
    const float *A, *Dw, *bias;
    int64_t u_sb, d_sb, z_sb, B_sb, B_sg, C_sb, C_sg;
    float* state;
    T* out;
};

template <typename T, int LPC, bool VEC>
__global__ void __launch_bounds__(kThreads) scan_step(const __grid_constant__ StepP<T> p) {
    constexpr int CH = kThreads / LPC;
    const int tid = threadIdx.x, q = tid % LPC, n0 = 4 * q;
    const int c = blockIdx.x * CH + tid / LPC;
    const bool live = c < p.D;
    const int64_t b = blockIdx.y;
    int64_t slot = b;
    if (p.s32) slot = __ldg(p.s32 + b);
    if (p.s64) slot = __ldg(p.s64 + b);
    if (slot < 0 || slot >= p.slots) {
        if (slot >= 0 && blockIdx.x == 0 && tid == 0) record_error(PE_ERR_INVALID | (kSiteSlot << 8));
        if (live && q == 0) p.out[b * p.D + c] = from_float<T>(0.0f);
        return;
    }
    float y = 0.0f, uv = 0.0f;
    if (live) {
        uv = to_float(__ldg(p.u + b * p.u_sb + c));
        float dt = to_float(__ldg(p.delta + b * p.d_sb + c)) + (p.bias ? __ldg(p.bias + c) : 0.0f);
        if (p.softplus) dt = softplusf(dt);
        const float x = dt * uv;
        const int g = c / p.Dg;
        const T* B = p.B + b * p.B_sb + g * p.B_sg + n0;
        const T* C = p.C + b * p.C_sb + g * p.C_sg + n0;
        const int64_t cn = (int64_t)c * p.N + n0;
        float* hp = p.state + slot * p.D * p.N + cn;
        if (VEC) {
            if (n0 < p.N) {
                float4 h = *reinterpret_cast<const float4*>(hp);
                const float4 a = __ldg(reinterpret_cast<const float4*>(p.A + cn));
                h.x = fmaf(exp2_fast(dt * (a.x * kLog2e)), h.x, x * to_float(__ldg(B)));
                h.y = fmaf(exp2_fast(dt * (a.y * kLog2e)), h.y, x * to_float(__ldg(B + 1)));
                h.z = fmaf(exp2_fast(dt * (a.z * kLog2e)), h.z, x * to_float(__ldg(B + 2)));
                h.w = fmaf(exp2_fast(dt * (a.w * kLog2e)), h.w, x * to_float(__ldg(B + 3)));
                y = to_float(__ldg(C)) * h.x + to_float(__ldg(C + 1)) * h.y + to_float(__ldg(C + 2)) * h.z +
                    to_float(__ldg(C + 3)) * h.w;
                *reinterpret_cast<float4*>(hp) = h;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (n0 + i >= p.N) break;
                const float h = fmaf(exp2_fast(dt * (__ldg(p.A + cn + i) * kLog2e)), hp[i], x * to_float(__ldg(B + i)));
                y = fmaf(to_float(__ldg(C + i)), h, y);
                hp[i] = h;
            }
        }
    }
#pragma unroll
    for (int m = LPC / 2; m >= 1; m /= 2) y += __shfl_xor_sync(0xffffffffu, y, m);
    if (live && q == 0) {
        if (p.Dw) y = fmaf(__ldg(p.Dw + c), uv, y);
        if (p.z) {
            const float zv = to_float(__ldg(p.z + b * p.z_sb + c));
            y *= zv * sigmoidf(zv);
        }
        p.out[b * p.D + c] = from_float<T>(y);
    }
}

// ---- host -------------------------------------------------------------------------
// Tokens a piece of a scan split along time; 0 = not split.
//
// Not split, a block (4 warps) takes its channels through a whole sequence: at best
// kFull clocks a token of SM time, kAlone when it has the SM to itself. Split, all SMs
// work, for the price of computing every exponential twice (kState more clocks a
// token) and of two more launches. The longest of n packed sequences, whose lengths
// the host does not know, is taken as (1 + ln n) average ones, as random cuts make it.
constexpr double kAlone = 60, kFull = 42, kState = 36, kLaunches = 15000;
int64_t piece_tokens(const pe_scan_args* a) {
    const int64_t ch = kThreads / lanes_for(a->states), dg = a->channels / a->groups;
    const int64_t tiles = a->groups * ceil_div(dg, ch);
    if (a->nseq < 1 || a->nseq > 65535 || a->tokens < 256) return 0;
    const double sms = num_sms(), total = (double)a->tokens * (a->cu ? 1 : a->nseq) * tiles;
    double longest = (double)a->tokens;
    if (a->cu) longest = min(longest, longest / a->nseq * (1.0 + log((double)a->nseq)));
    const double whole = max(longest * kAlone, total / sms * kFull);
    const double split = total / sms * (kFull + kState) * 1.1 + kLaunches;
    if (split >= whole) return 0;
    const int64_t piece = (int64_t)(total / (3.0 * sms));   // three blocks an SM
    return max((int64_t)64, ceil_div(piece, TS) * TS);
}

template <typename T, int LPC>
int scan_run(const pe_scan_args* a, cudaStream_t s) {
    ScanP<T> p = scan_params<T>(a, kThreads / LPC);
    const int64_t piece = piece_tokens(a);
    if (piece) {
        p.piece = piece;
        const int64_t n = piece_count(p.seqs, piece);
        p.hloc = (float*)a->ws;
        p.dtsum = p.hloc + n * p.D * p.N;
    }
    unsigned grid;
    if (int rc = grid_of(piece_count(p.seqs, p.piece) * p.G * p.ntile, &grid)) return rc;
    constexpr int CH = kThreads / LPC, cols = TS * 4 * LPC;
    if (piece) {
        if (int rc = launch(scan_fwd<T, LPC, true>, p, grid, 2 * (2 * CH * LD + cols) * 4, s)) return rc;
        const dim3 carry((unsigned)ceil_div((int64_t)p.D * p.N, kThreads), (unsigned)p.seqs.nseq);
        scan_carry<T><<<carry, kThreads, 0, s>>>(p);
        count_launch();
        if (cudaGetLastError() != cudaSuccess) return PE_ERR_CUDA;
    }
    return launch(scan_fwd<T, LPC, false>, p, grid, 2 * (3 * CH * LD + 2 * cols) * 4, s);
}

template <typename T>
int scan_lanes(const pe_scan_args* a, cudaStream_t s) {
    PE_LANES(scan_run, lanes_for(a->states), a, s)
}

template <typename T, int LPC>
int step_run(const pe_scan_step_args* a, cudaStream_t s) {
    StepP<T> p;
    p.batch = a->batch; p.slots = a->slots;
    p.D = (int)a->channels; p.N = (int)a->states; p.G = (int)a->groups; p.Dg = p.D / p.G;
    p.softplus = a->softplus != 0;
    p.s32 = a->slots32; p.s64 = a->slots64;
    p.u = (const T*)a->u; p.delta = (const T*)a->delta; p.z = (const T*)a->z;
    p.B = (const T*)a->B; p.C = (const T*)a->C;
    p.A = a->A; p.Dw = a->D; p.bias = a->delta_bias;
    p.u_sb = a->u_sb; p.d_sb = a->delta_sb; p.z_sb = a->z_sb;
    p.B_sb = a->B_sb; p.B_sg = a->B_sg; p.C_sb = a->C_sb; p.C_sg = a->C_sg;
    p.state = a->state; p.out = (T*)a->out;
    const dim3 grid((unsigned)ceil_div(p.D, kThreads / LPC), (unsigned)a->batch);
    const bool vec = p.N % 4 == 0 && ((uintptr_t)p.state | (uintptr_t)p.A) % 16 == 0;
    if (vec)
        scan_step<T, LPC, true><<<grid, kThreads, 0, s>>>(p);
    else
        scan_step<T, LPC, false><<<grid, kThreads, 0, s>>>(p);
    count_launch();
    return cudaGetLastError() == cudaSuccess ? PE_OK : PE_ERR_CUDA;
}
template <typename T>
int step_lanes(const pe_scan_step_args* a, cudaStream_t s) {
    PE_LANES(step_run, lanes_for(a->states), a, s)
}

int scan_any(const pe_scan_args* a, cudaStream_t s) { PE_TYPES(scan_lanes, a->dtype, a, s) }
int step_any(const pe_scan_step_args* a, cudaStream_t s) { PE_TYPES(step_lanes, a->dtype, a, s) }

}  // namespace

int64_t scan_ckpt_floats(int64_t tokens, int64_t nseq, int64_t packed, int64_t channels, int64_t states) {
    const int32_t none = 0;
    return piece_count(Seqs{packed ? &none : nullptr, tokens, (int32_t)nseq}, TS) * channels * states;
}

int64_t scan_ws_bytes(const pe_scan_args* a) {
    if (check_scan(a) != PE_OK) return 0;
    const int64_t piece = piece_tokens(a);
    return piece ? piece_count(seqs_of(a), piece) * (a->channels * a->states + a->channels) * 4 : 0;
}

int selective_scan(const pe_scan_args* a, cudaStream_t s) {
    if (int rc = check_scan(a)) return rc;
    if (a->nseq == 0) return PE_OK;
    const int64_t need = scan_ws_bytes(a);
    if (need && (!a->ws || a->ws_bytes < need)) return PE_ERR_WORKSPACE;
    return scan_any(a, s);
}

int selective_scan_step(const pe_scan_step_args* a, cudaStream_t s) {
    if (!a || a->dtype < PE_F32 || a->dtype > PE_BF16 || a->batch < 0 || a->channels < 1 || a->groups < 1 ||
        a->states < 1 || a->slots < 0 || a->channels % a->groups)
        return PE_ERR_INVALID;
    if (a->states > 128 || a->channels > (1 << 24) || a->batch > 65535) return PE_ERR_UNSUPPORTED;
    if (a->batch == 0) return PE_OK;
    if (!a->state || !a->u || !a->delta || !a->B || !a->C || !a->A || !a->out) return PE_ERR_INVALID;
    return step_any(a, s);
}

int scan_device_error(bool clear) {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_device_error, sizeof(int)) != cudaSuccess) return -1;
    if (v && clear) cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
    return v;
}

}  // namespace pe

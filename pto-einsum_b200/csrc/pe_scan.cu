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
#include "pe_scan.cuh"

namespace pe {

namespace {

// ---- forward --------------------------------------------------------------------
// STATE_ONLY: a piece's last state from a zero start and its sum of dt (first half of
// a split scan); else the whole, starting from what the sequence's earlier pieces left.
template <typename T, int LPC, bool STATE_ONLY>
__global__ void __launch_bounds__(kThreads) scan_fwd(const __grid_constant__ ScanP<T> p) {
    constexpr int CH = kThreads / LPC, NP = 4 * LPC, R = LPC < TS ? LPC : TS;
    __shared__ __align__(16) float sdt[CH * LD], sx[CH * LD], sy[STATE_ONLY ? 1 : CH * LD];
    __shared__ __align__(16) float sB[TS * NP], sC[STATE_ONLY ? 1 : TS * NP];
    const int tid = threadIdx.x, lane = tid & 31;
    if (blockIdx.x == 0 && tid < 32) check_offsets(p.seqs, lane, kSiteOffsets);
    const Place w = place_of<CH>(p);
    if (!w.any) return;
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
    if (!STATE_ONLY) {
        const int64_t first = w.number - w.j;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (p.h0 && live && n0 + i < p.N) h[i] = __ldg(p.h0 + w.s * DN + cn + i);
        for (int64_t k = first; k < w.number; ++k) {
            const float sum = live ? __ldg(p.dtsum + k * p.D + c) : 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (live && n0 + i < p.N) h[i] = fmaf(exp2_fast(A[i] * sum), h[i], __ldg(p.hloc + k * DN + cn + i));
        }
    }
    float dtsum = 0.0f;
    const T* u = p.u + w.sp.row * p.u_sb;
    const T* delta = p.delta + w.sp.row * p.d_sb;
    const T* z = p.z ? p.z + w.sp.row * p.z_sb : nullptr;
    const T* B = p.B + w.sp.row * p.B_sb + w.g * p.B_sg;
    const T* C = p.C + w.sp.row * p.C_sb + w.g * p.C_sg;
    T* out = p.out + (w.sp.row * p.seqs.tokens) * p.D;

    for (int64_t t = w.t0; t < w.t1; t += TS) {
        const int cnt = (int)min((int64_t)TS, w.t1 - t);
        const int64_t at = tok + t;
        for (int it = tid; it < CH * (TS / 4); it += kThreads) {
            const int ic = it % CH, t4 = it / CH * 4;
            const int64_t cc = w.c0 + ic;
            float dt[4], x[4];
            const float bias = p.bias && ic < w.nch ? __ldg(p.bias + cc) : 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = ic < w.nch && t4 + i < cnt;
                dt[i] = in ? to_float(__ldg(delta + (at + t4 + i) * p.d_st + cc)) + bias : 0.0f;
                if (p.softplus) dt[i] = softplusf(dt[i]);
                x[i] = in ? dt[i] * to_float(__ldg(u + (at + t4 + i) * p.u_st + cc)) : 0.0f;
            }
            *reinterpret_cast<float4*>(sdt + ic * LD + t4) = make_float4(dt[0], dt[1], dt[2], dt[3]);
            *reinterpret_cast<float4*>(sx + ic * LD + t4) = make_float4(x[0], x[1], x[2], x[3]);
        }
        stage_cols<LPC>(sB, B + at * p.B_st, p.B_st, cnt, p.N);
        if (!STATE_ONLY) stage_cols<LPC>(sC, C + at * p.C_st, p.C_st, cnt, p.N);
        __syncthreads();
        if (!STATE_ONLY && p.ckpt && live) {
            float* k = p.ckpt + (piece_base(p.seqs, w.s, TS) + t / TS) * DN + cn;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n0 + i < p.N) k[i] = h[i];
        }
        float y[TS];
#pragma unroll
        for (int t4 = 0; t4 < TS; t4 += 4) {
            const float4 dt4 = *reinterpret_cast<const float4*>(sdt + ch * LD + t4);
            const float4 x4 = *reinterpret_cast<const float4*>(sx + ch * LD + t4);
            const float dt[4] = {dt4.x, dt4.y, dt4.z, dt4.w}, x[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                y[t4 + k] = 0.0f;
                if (t4 + k < cnt) {
                    const float4 b = *reinterpret_cast<const float4*>(sB + (t4 + k) * NP + n0);
                    h[0] = fmaf(exp2_fast(dt[k] * A[0]), h[0], x[k] * b.x);
                    h[1] = fmaf(exp2_fast(dt[k] * A[1]), h[1], x[k] * b.y);
                    h[2] = fmaf(exp2_fast(dt[k] * A[2]), h[2], x[k] * b.z);
                    h[3] = fmaf(exp2_fast(dt[k] * A[3]), h[3], x[k] * b.w);
                    if (STATE_ONLY) {
                        dtsum += dt[k];
                    } else {
                        const float4 cv = *reinterpret_cast<const float4*>(sC + (t4 + k) * NP + n0);
                        y[t4 + k] = fmaf(cv.x, h[0], cv.y * h[1]) + fmaf(cv.z, h[2], cv.w * h[3]);
                    }
                }
            }
        }
        if (!STATE_ONLY) {
#pragma unroll
            for (int r = 0; r < TS; r += R) {
                float v[R];
#pragma unroll
                for (int i = 0; i < R; ++i) v[i] = y[r + i];
                float sum = reduce_scatter<R, 1>(v, lane);
                if (LPC > R) sum += __shfl_xor_sync(0xffffffffu, sum, R);
                if (q < R) sy[ch * LD + r + q] = sum;
            }
        }
        __syncthreads();
        if (!STATE_ONLY) {
            for (int it = tid; it < CH * (TS / 4); it += kThreads) {
                const int ic = it % CH, t4 = it / CH * 4;
                const int64_t cc = w.c0 + ic;
                if (ic >= w.nch) continue;
                const float4 y4 = *reinterpret_cast<const float4*>(sy + ic * LD + t4);
                float yv[4] = {y4.x, y4.y, y4.z, y4.w};
                const float Dw = p.Dw ? __ldg(p.Dw + cc) : 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (t4 + i >= cnt) break;
                    if (p.Dw) yv[i] = fmaf(Dw, to_float(__ldg(u + (at + t4 + i) * p.u_st + cc)), yv[i]);
                    if (z) {
                        const float zv = to_float(__ldg(z + (at + t4 + i) * p.z_st + cc));
                        yv[i] *= zv * sigmoidf(zv);
                    }
                    out[(at + t4 + i) * p.D + cc] = from_float<T>(yv[i]);
                }
            }
            // sy is written again only after the next tile's first barrier
        }
    }
    if (!live) return;
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
int64_t piece_tokens(const pe_scan_args*) { return 0; }

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
    if (piece) {
        scan_fwd<T, LPC, true><<<grid, kThreads, 0, s>>>(p);
        count_launch();
    }
    scan_fwd<T, LPC, false><<<grid, kThreads, 0, s>>>(p);
    count_launch();
    return cudaGetLastError() == cudaSuccess ? PE_OK : PE_ERR_CUDA;
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

// pe_scan_grad.cu - gradients of the selective scan, for sm_100a.
#include "pe_scan.cuh"

namespace pe {

namespace {

// ---- backward -------------------------------------------------------------------
template <typename T>
struct GradP {
    ScanP<T> f;
    const T* dout;
    int64_t o_sb, o_st;
    const float* dstate;
    T *du, *ddelta, *dz;
    float *dh0;
    float *pBC;       // [2][tiles][batch * tokens][G][N]: each channel tile's share of dB and dC
    float *pA;        // [nseq][D][N]
    float *pD, *pb;   // [nseq][D]
};

// One block takes the channel tile through a whole sequence, tile by tile from its
// end: the 16 states of a tile are computed again from its checkpoint and stay in
// registers, then the adjoint runs back over them.
//   g = C dy + a' g' ;  q = sum_n g B ;  r = sum_n g h' a A
//   du = q dt + D dy ;  ddt = q u + r ;  dB += g dt u ;  dC += dy h ;  dA += g h' a dt
template <typename T, int LPC>
__global__ void __launch_bounds__(kThreads) scan_bwd(const __grid_constant__ GradP<T> p) {
    constexpr int CH = kThreads / LPC, NP = 4 * LPC, R = LPC < TS ? LPC : TS;
    constexpr int CW = 32 / LPC;              // channels a warp
    constexpr int RC = CW < 8 ? CW : 8;       // lanes that share the eight dB and dC sums
    constexpr int VL = 8 / RC;                // sums a lane ends with
    extern __shared__ __align__(16) float smem[];
    float *sdt = smem, *sx = sdt + CH * LD, *sdy = sx + CH * LD, *sy = sdy + CH * LD, *sq = sy + CH * LD,
          *sr = sq + CH * LD;             // [CH][LD] each
    float *sB = sr + CH * LD, *sC = sB + TS * NP;
    float* sred = sC + TS * NP;           // [4 warps][TS][2][NP]
    const ScanP<T>& f = p.f;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
    if (blockIdx.x == 0 && tid < 32) check_offsets(f.seqs, lane, kSiteOffsets);
    const Place w = place_of<CH>(f);
    const int ch = tid / LPC, q = tid % LPC, c = w.c0 + ch, n0 = 4 * q;
    const bool live = ch < w.nch;
    const int64_t DN = (int64_t)f.D * f.N, cn = (int64_t)c * f.N + n0;
    const int tile = (w.c0 - w.g * f.Dg) / CH;

    float A[4], dA[4], carry[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool in = live && n0 + i < f.N;
        A[i] = in ? __ldg(f.A + cn + i) * kLog2e : 0.0f;
        carry[i] = in && p.dstate ? __ldg(p.dstate + w.s * DN + cn + i) : 0.0f;
        dA[i] = 0.0f;
    }
    float dD = 0.0f, db = 0.0f;   // of channel tid % CH, this thread's tokens
    const T* u = f.u + w.sp.row * f.u_sb;
    const T* delta = f.delta + w.sp.row * f.d_sb;
    const T* z = f.z ? f.z + w.sp.row * f.z_sb : nullptr;
    const T* dout = p.dout + w.sp.row * p.o_sb;
    const T* B = f.B + w.sp.row * f.B_sb + w.g * f.B_sg;
    const T* C = f.C + w.sp.row * f.C_sb + w.g * f.C_sg;
    const int64_t row0 = w.sp.row * f.seqs.tokens;
    const int64_t rows = f.seqs.tokens * (f.seqs.cu ? 1 : f.seqs.nseq);

    for (int64_t t = w.sp.len > 0 ? (w.sp.len - 1) / TS * TS : -1; t >= 0; t -= TS) {
        const int cnt = (int)min((int64_t)TS, w.sp.len - t);
        const int64_t at = w.sp.start + t;
        for (int it = tid; it < CH * (TS / 4); it += kThreads) {
            const int ic = it % CH, t4 = it / CH * 4;
            const int64_t cc = w.c0 + ic;
            const float bias = f.bias && ic < w.nch ? __ldg(f.bias + cc) : 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = ic < w.nch && t4 + i < cnt;
                const int64_t tt = at + t4 + i;
                float dt = in ? to_float(__ldg(delta + tt * f.d_st + cc)) + bias : 0.0f;
                if (f.softplus) dt = softplusf(dt);
                float dy = in ? to_float(__ldg(dout + tt * p.o_st + cc)) : 0.0f;
                if (z && in) {
                    const float zv = to_float(__ldg(z + tt * f.z_st + cc));
                    dy *= zv * sigmoidf(zv);
                }
                const int k = ic * LD + t4 + i;
                sdt[k] = dt;
                sx[k] = in ? dt * to_float(__ldg(u + tt * f.u_st + cc)) : 0.0f;
                sdy[k] = dy;
            }
        }
        stage_cols<LPC>(sB, B + at * f.B_st, f.B_st, cnt, f.N);
        stage_cols<LPC>(sC, C + at * f.C_st, f.C_st, cnt, f.N);
        __syncthreads();

        float hs[TS + 1][4];   // hs[0] before the tile, hs[k + 1] after its token k
        {
            const float* k = f.ckpt + (piece_base(f.seqs, w.s, TS) + t / TS) * DN + cn;
#pragma unroll
            for (int i = 0; i < 4; ++i) hs[0][i] = live && n0 + i < f.N ? k[i] : 0.0f;
        }
        float yv[TS];
#pragma unroll
        for (int k = 0; k < TS; ++k) {
            yv[k] = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) hs[k + 1][i] = hs[k][i];
            if (k < cnt) {
                const float dt = sdt[ch * LD + k], x = sx[ch * LD + k];
                const float4 b = *reinterpret_cast<const float4*>(sB + k * NP + n0);
                const float4 cv = *reinterpret_cast<const float4*>(sC + k * NP + n0);
                hs[k + 1][0] = fmaf(exp2_fast(dt * A[0]), hs[k][0], x * b.x);
                hs[k + 1][1] = fmaf(exp2_fast(dt * A[1]), hs[k][1], x * b.y);
                hs[k + 1][2] = fmaf(exp2_fast(dt * A[2]), hs[k][2], x * b.z);
                hs[k + 1][3] = fmaf(exp2_fast(dt * A[3]), hs[k][3], x * b.w);
                yv[k] = fmaf(cv.x, hs[k + 1][0], cv.y * hs[k + 1][1]) + fmaf(cv.z, hs[k + 1][2], cv.w * hs[k + 1][3]);
            }
        }
        if (z) {
#pragma unroll
            for (int r = 0; r < TS; r += R) {
                float v[R];
#pragma unroll
                for (int i = 0; i < R; ++i) v[i] = yv[r + i];
                float sum = reduce_scatter<R, 1>(v, lane);
                if (LPC > R) sum += __shfl_xor_sync(0xffffffffu, sum, R);
                if (q < R) sy[ch * LD + r + q] = sum;
            }
        }
        float qv[TS], rv[TS];
#pragma unroll
        for (int k = TS - 1; k >= 0; --k) {
            qv[k] = rv[k] = 0.0f;
            if (k < cnt) {
                const float dt = sdt[ch * LD + k], x = sx[ch * LD + k], dy = sdy[ch * LD + k];
                const float4 b4 = *reinterpret_cast<const float4*>(sB + k * NP + n0);
                const float4 c4 = *reinterpret_cast<const float4*>(sC + k * NP + n0);
                const float b[4] = {b4.x, b4.y, b4.z, b4.w}, cv[4] = {c4.x, c4.y, c4.z, c4.w};
                float v[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float g = fmaf(cv[i], dy, carry[i]);
                    qv[k] = fmaf(g, b[i], qv[k]);
                    v[i] = g * x;
                    v[4 + i] = dy * hs[k + 1][i];
                    carry[i] = g * exp2_fast(dt * A[i]);
                    const float e = carry[i] * hs[k][i];
                    rv[k] = fmaf(e, A[i], rv[k]);
                    dA[i] = fmaf(e, dt, dA[i]);
                }
                // sum over the warp's channels: lanes that differ in the bits LPC .. 16
                float* dst = sred + ((warp * TS + k) * 2) * NP + n0;
                if constexpr (RC == 8) {
                    float s = reduce_scatter<8, LPC>(v, lane);
#pragma unroll
                    for (int m = 8 * LPC; m < 32; m *= 2) s += __shfl_xor_sync(0xffffffffu, s, m);
                    const int i = (lane / LPC) % 8;
                    if (lane < 8 * LPC) dst[(i / 4) * NP + i % 4] = s;
                } else {
                    // fewer lanes than sums: every lane halves its set until RC lanes hold VL each
#pragma unroll
                    for (int m = 4, half = RC / 2; half >= 1; m /= 2, half /= 2) {
                        const bool hi = lane & (half * LPC);
#pragma unroll
                        for (int i = 0; i < m; ++i) {
                            const float send = hi ? v[i] : v[i + m];
                            const float keep = hi ? v[i + m] : v[i];
                            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, half * LPC);
                        }
                    }
                    const int first = (lane / LPC) % RC * VL;
#pragma unroll
                    for (int i = 0; i < VL; ++i) dst[((first + i) / 4) * NP + (first + i) % 4] = v[i];
                }
            }
        }
#pragma unroll
        for (int r = 0; r < TS; r += R) {
            float v[R];
#pragma unroll
            for (int i = 0; i < R; ++i) v[i] = qv[r + i];
            float sum = reduce_scatter<R, 1>(v, lane);
            if (LPC > R) sum += __shfl_xor_sync(0xffffffffu, sum, R);
            if (q < R) sq[ch * LD + r + q] = sum;
#pragma unroll
            for (int i = 0; i < R; ++i) v[i] = rv[r + i];
            sum = reduce_scatter<R, 1>(v, lane);
            if (LPC > R) sum += __shfl_xor_sync(0xffffffffu, sum, R);
            if (q < R) sr[ch * LD + r + q] = sum * kLn2;
        }
        __syncthreads();
        for (int it = tid; it < CH * (TS / 4); it += kThreads) {
            const int ic = it % CH, t4 = it / CH * 4;
            const int64_t cc = w.c0 + ic;
            if (ic >= w.nch) continue;
            const float Dw = f.Dw ? __ldg(f.Dw + cc) : 0.0f;
            const float bias = f.bias ? __ldg(f.bias + cc) : 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (t4 + i >= cnt) break;
                const int64_t tt = at + t4 + i, o = (row0 + tt) * f.D + cc;
                const int k = ic * LD + t4 + i;
                const float uv = to_float(__ldg(u + tt * f.u_st + cc));
                const float dy = sdy[k], gq = sq[k];
                p.du[o] = from_float<T>(fmaf(gq, sdt[k], Dw * dy));
                float dd = fmaf(gq, uv, sr[k]);
                if (f.softplus) dd *= sigmoidf(to_float(__ldg(delta + tt * f.d_st + cc)) + bias);
                p.ddelta[o] = from_float<T>(dd);
                dD = fmaf(dy, uv, dD);
                db += dd;
                if (p.dz) {
                    const float zv = to_float(__ldg(z + tt * f.z_st + cc));
                    const float y = fmaf(Dw, uv, sy[k]);
                    p.dz[o] = from_float<T>(to_float(__ldg(dout + tt * p.o_st + cc)) * y * silu_slope(zv, sigmoidf(zv)));
                }
            }
        }
        for (int i = tid; i < cnt * 2 * NP; i += kThreads) {
            const int n = i % NP, which = i / NP % 2, k = i / (2 * NP);
            if (n >= f.N) continue;
            float s = 0.0f;
#pragma unroll
            for (int v = 0; v < kThreads / 32; ++v) s += sred[((v * TS + k) * 2 + which) * NP + n];
            p.pBC[(((int64_t)which * f.ntile + tile) * rows + row0 + at + k) * f.G * f.N + w.g * f.N + n] = s;
        }
        __syncthreads();
    }
    // sums over the tokens: dA by its own lane, dD and dbias over the threads of a channel
    if (live) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n0 + i < f.N) {
                p.pA[w.s * DN + cn + i] = dA[i];
                if (p.dh0) p.dh0[w.s * DN + cn + i] = carry[i];
            }
    }
    if (CH >= kThreads) {
        if (tid < w.nch) {
            p.pD[(int64_t)w.s * f.D + w.c0 + tid] = dD;
            p.pb[(int64_t)w.s * f.D + w.c0 + tid] = db;
        }
    } else {
        sred[tid] = dD;   // read last before the loop's final barrier
        sred[kThreads + tid] = db;
        __syncthreads();
        if (tid < w.nch) {
            float a = 0.0f, b = 0.0f;
            for (int k = tid; k < kThreads; k += CH) { a += sred[k]; b += sred[kThreads + k]; }
            p.pD[(int64_t)w.s * f.D + w.c0 + tid] = a;
            p.pb[(int64_t)w.s * f.D + w.c0 + tid] = b;
        }
    }
}

// ---- host -------------------------------------------------------------------------
struct GradWs {
    int64_t bc, a, d, b, total;   // float offsets
};
GradWs grad_ws(const pe_scan_args* a) {
    const int64_t ch = kThreads / lanes_for(a->states), dg = a->channels / a->groups;
    const int64_t rows = a->tokens * (a->cu ? 1 : a->nseq);
    GradWs w;
    w.bc = 0;
    w.a = 2 * ceil_div(dg, ch) * rows * a->groups * a->states;
    w.d = w.a + a->nseq * a->channels * a->states;
    w.b = w.d + a->nseq * a->channels;
    w.total = w.b + a->nseq * a->channels;
    return w;
}

template <typename T, int LPC>
int grad_run(const pe_scan_grad_args* a, cudaStream_t s) {
    constexpr int CH = kThreads / LPC;
    const pe_scan_args* f = &a->fwd;
    GradP<T> p;
    p.f = scan_params<T>(f, CH);
    const GradWs w = grad_ws(f);
    float* ws = (float*)a->ws;
    p.dout = (const T*)a->dout; p.o_sb = a->dout_sb; p.o_st = a->dout_st;
    p.dstate = a->dstate;
    p.du = (T*)a->du; p.ddelta = (T*)a->ddelta; p.dz = (T*)a->dz;
    p.dh0 = a->dh0;
    p.pBC = ws + w.bc; p.pA = ws + w.a; p.pD = ws + w.d; p.pb = ws + w.b;
    unsigned grid;
    if (int rc = grid_of((int64_t)p.f.seqs.nseq * p.f.G * p.f.ntile, &grid)) return rc;
    // every sequence is one piece here, numbered by itself
    const int smem = (6 * CH * LD + (2 + 2 * kThreads / 32) * TS * 4 * LPC) * 4;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(scan_bwd<T, LPC>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return PE_ERR_CUDA;
    }
    if (grid) {
        scan_bwd<T, LPC><<<grid, kThreads, smem, s>>>(p);
        count_launch();
        if (cudaGetLastError() != cudaSuccess) return PE_ERR_CUDA;
    }
    const int64_t rows = f->tokens * (f->cu ? 1 : f->nseq), cols = rows * f->groups * f->states;
    const int64_t DN = f->channels * f->states;
    int rc = sum_rows(p.pBC, p.f.ntile, cols, (int)f->dtype, a->dB, s);
    if (!rc) rc = sum_rows(p.pBC + p.f.ntile * cols, p.f.ntile, cols, (int)f->dtype, a->dC, s);
    if (!rc) rc = sum_rows(p.pA, f->nseq, DN, PE_F32, a->dA, s);
    if (!rc && a->dD) rc = sum_rows(p.pD, f->nseq, f->channels, PE_F32, a->dD, s);
    if (!rc && a->ddelta_bias) rc = sum_rows(p.pb, f->nseq, f->channels, PE_F32, a->ddelta_bias, s);
    return rc;
}

template <typename T>
int grad_lanes(const pe_scan_grad_args* a, cudaStream_t s) {
    PE_LANES(grad_run, lanes_for(a->fwd.states), a, s)
}

int grad_any(const pe_scan_grad_args* a, cudaStream_t s) { PE_TYPES(grad_lanes, a->fwd.dtype, a, s) }

}  // namespace

int64_t scan_grad_ws_bytes(const pe_scan_grad_args* a) {
    return a && check_scan(&a->fwd) == PE_OK ? grad_ws(&a->fwd).total * 4 : 0;
}

int selective_scan_grad(const pe_scan_grad_args* a, cudaStream_t s) {
    if (!a) return PE_ERR_INVALID;
    if (int rc = check_scan(&a->fwd)) return rc;
    if (!a->dA || (a->dz && !a->fwd.z)) return PE_ERR_INVALID;
    if (a->fwd.tokens && a->fwd.nseq && (!a->dout || !a->du || !a->ddelta || !a->dB || !a->dC || !a->fwd.ckpt))
        return PE_ERR_INVALID;
    const int64_t need = scan_grad_ws_bytes(a);
    if (need && (!a->ws || a->ws_bytes < need)) return PE_ERR_WORKSPACE;
    return grad_any(a, s);
}

int scan_grad_device_error(bool clear) {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_device_error, sizeof(int)) != cudaSuccess) return -1;
    if (v && clear) cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int));
    return v;
}

}  // namespace pe

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

// Adds v to a sum that keeps its rounding errors (Kahan): a sum over thousands of
// tokens would lose what two passes of a pairwise sum keep.
__device__ __forceinline__ void add_exactly(float& sum, float& err, float v) {
    const float y = __fsub_rn(v, err), t = __fadd_rn(sum, y);
    err = __fsub_rn(__fsub_rn(t, sum), y);
    sum = t;
}

// A tile's inputs on their way from memory: loaded while the tile before is worked on.
template <typename T, int LPC>
struct GradRegs {
    static constexpr int CH = kThreads / LPC, I = LPC < 4 ? 4 / LPC : 1, J = LPC * 4 * TS / kThreads > 0 ? LPC * 4 * TS / kThreads : 1;
    T d[I][4], u[I][4], z[I][4], o[I][4], b[J], c[J];

    __device__ __forceinline__ void load(const GradP<T>& p, const Place& w, const T* up, const T* dp, const T* zp,
                                         const T* op, const T* Bp, const T* Cp, int64_t at, int cnt) {
        constexpr int NP = 4 * LPC;
        const int tid = threadIdx.x;
        const T zero = from_float<T>(0.0f);
#pragma unroll
        for (int k = 0; k < I; ++k) {
            const int it = tid + k * kThreads, ic = it % CH, t4 = it / CH * 4;
            const int64_t cc = w.c0 + ic;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = ic < w.nch && t4 + i < cnt;
                const int64_t t = at + t4 + i;
                d[k][i] = in ? __ldg(dp + t * p.f.d_st + cc) : zero;
                u[k][i] = in ? __ldg(up + t * p.f.u_st + cc) : zero;
                o[k][i] = in ? __ldg(op + t * p.o_st + cc) : zero;
                z[k][i] = in && zp ? __ldg(zp + t * p.f.z_st + cc) : zero;
            }
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int i = tid + j * kThreads, t = i / NP, n = i % NP;
            const bool in = t < cnt && n < p.f.N;
            b[j] = in ? __ldg(Bp + (at + t) * p.f.B_st + n) : zero;
            c[j] = in ? __ldg(Cp + (at + t) * p.f.C_st + n) : zero;
        }
    }
};

// Sums of R values over the LPC lanes of a channel, TS values in: lane q of the channel
// stores value k + q of each run of R.
template <int LPC>
__device__ __forceinline__ void sum_states(const float (&y)[TS], float* row, int q, int lane, float scale) {
    constexpr int R = LPC < TS ? LPC : TS;
#pragma unroll
    for (int k = 0; k < TS; k += R) {
        float v[R];
#pragma unroll
        for (int i = 0; i < R; ++i) v[i] = y[k + i];
        float sum = reduce_scatter<R, 1>(v, lane);
        if (LPC > R) sum += __shfl_xor_sync(0xffffffffu, sum, R);
        if (q < R) row[k + q] = sum * scale;
    }
}

// One block takes the channel tile through a whole sequence, tile by tile from its
// end: the 16 states of a tile are computed again from its checkpoint and stay in
// registers, then the adjoint runs back over them.
//   g = C dy + a' g' ;  q = sum_n g B ;  r = sum_n g h' a A
//   du = q dt + D dy ;  ddt = q u + r ;  dB += g dt u ;  dC += dy h ;  dA += g h' a dt
template <typename T, int LPC>
__global__ void __launch_bounds__(kThreads, LPC == 4 || LPC == 8 ? 3 : 2) scan_bwd(const __grid_constant__ GradP<T> p) {
    constexpr int CH = kThreads / LPC, NP = 4 * LPC;
    constexpr int CW = 32 / LPC;              // channels a warp
    constexpr int RC = CW < 8 ? CW : 8;       // lanes that share the eight dB and dC sums
    constexpr int VL = 8 / RC;                // sums a lane ends with
    using Regs = GradRegs<T, LPC>;
    constexpr int I = Regs::I, J = Regs::J;
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

    float A[4], dA[4], eA[4], carry[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool in = live && n0 + i < f.N;
        A[i] = in ? __ldg(f.A + cn + i) * kLog2e : 0.0f;
        carry[i] = in && p.dstate ? __ldg(p.dstate + w.s * DN + cn + i) : 0.0f;
        dA[i] = eA[i] = 0.0f;
    }
    const f32x2 A01 = pack2(A[0], A[1]), A23 = pack2(A[2], A[3]);
    f32x2 c01 = pack2(carry[0], carry[1]), c23 = pack2(carry[2], carry[3]);
    float dD = 0.0f, db = 0.0f, eD = 0.0f, eb = 0.0f;   // of channel tid % CH, this thread's tokens
    const T* u = f.u + w.sp.row * f.u_sb;
    const T* delta = f.delta + w.sp.row * f.d_sb;
    const T* z = f.z ? f.z + w.sp.row * f.z_sb : nullptr;
    const T* dout = p.dout + w.sp.row * p.o_sb;
    const T* B = f.B + w.sp.row * f.B_sb + w.g * f.B_sg;
    const T* C = f.C + w.sp.row * f.C_sb + w.g * f.C_sg;
    const int64_t row0 = w.sp.row * f.seqs.tokens;
    const int64_t rows = f.seqs.tokens * (f.seqs.cu ? 1 : f.seqs.nseq);
    float bias[I], Dw[I];
#pragma unroll
    for (int k = 0; k < I; ++k) {
        const int ic = (tid + k * kThreads) % CH;
        bias[k] = f.bias && ic < w.nch ? __ldg(f.bias + w.c0 + ic) : 0.0f;
        Dw[k] = f.Dw && ic < w.nch ? __ldg(f.Dw + w.c0 + ic) : 0.0f;
    }
    const int64_t top = w.sp.len > 0 ? (w.sp.len - 1) / TS * TS : -1;
    const float* ckpt = f.ckpt + (piece_base(f.seqs, w.s, TS) + (top >= 0 ? top / TS : 0)) * DN + cn;
    Regs r;
    float hc[4];
    auto load_state = [&]() {
#pragma unroll
        for (int i = 0; i < 4; ++i) hc[i] = live && n0 + i < f.N ? ckpt[i] : 0.0f;
        ckpt -= DN;
    };
    if (top >= 0) {
        r.load(p, w, u, delta, z, dout, B, C, w.sp.start + top, (int)(w.sp.len - top));
        load_state();
    }

    for (int64_t t = top; t >= 0; t -= TS) {
        const int cnt = (int)min((int64_t)TS, w.sp.len - t);
        const int64_t at = w.sp.start + t;
        // what the tile's gradients need of each (token, channel) after the recurrence:
        // u, slope of softplus, d out / d z without y
        float ku[I][4], ks[I][4], kz[I][4];
#pragma unroll
        for (int k = 0; k < I; ++k) {
            const int it = tid + k * kThreads, ic = it % CH, t4 = it / CH * 4;
            float dt[4], x[4], dy[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = ic < w.nch && t4 + i < cnt;
                const float raw = to_float(r.d[k][i]) + bias[k], zv = to_float(r.z[k][i]);
                ku[k][i] = to_float(r.u[k][i]);
                dy[i] = to_float(r.o[k][i]);
                dt[i] = f.softplus ? softplusf(raw) : raw;
                ks[k][i] = f.softplus ? sigmoidf(raw) : 1.0f;
                kz[k][i] = 0.0f;
                if (z) {
                    const float s = sigmoidf(zv);
                    kz[k][i] = dy[i] * silu_slope(zv, s);
                    dy[i] *= zv * s;
                }
                x[i] = dt[i] * ku[k][i];
                if (!in) dt[i] = x[i] = dy[i] = 0.0f;
            }
            if (it < CH * (TS / 4)) {
                *reinterpret_cast<float4*>(sdt + ic * LD + t4) = make_float4(dt[0], dt[1], dt[2], dt[3]);
                *reinterpret_cast<float4*>(sx + ic * LD + t4) = make_float4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<float4*>(sdy + ic * LD + t4) = make_float4(dy[0], dy[1], dy[2], dy[3]);
            }
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int i = tid + j * kThreads;
            if (i < TS * NP) {
                sB[i] = to_float(r.b[j]);
                sC[i] = to_float(r.c[j]);
            }
        }
        __syncthreads();

        f32x2 hs[TS + 1][2];   // hs[0] before the tile, hs[k + 1] after its token k
        hs[0][0] = pack2(hc[0], hc[1]);
        hs[0][1] = pack2(hc[2], hc[3]);
        if (t > 0) {
            r.load(p, w, u, delta, z, dout, B, C, at - TS, TS);
            load_state();
        }
        {
            float yv[TS];
#pragma unroll
            for (int k = 0; k < TS; ++k) {
                yv[k] = 0.0f;
                hs[k + 1][0] = hs[k][0];
                hs[k + 1][1] = hs[k][1];
                if (k < cnt) {
                    const float dt = sdt[ch * LD + k], x = sx[ch * LD + k];
                    const f32x2 dt2 = pack2(dt, dt), x2 = pack2(x, x);
                    const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(sB + k * NP + n0);
                    hs[k + 1][0] = fma2(exp2_2(mul2(dt2, A01)), hs[k][0], mul2(x2, b.x));
                    hs[k + 1][1] = fma2(exp2_2(mul2(dt2, A23)), hs[k][1], mul2(x2, b.y));
                    if (z) {
                        const ulonglong2 cv = *reinterpret_cast<const ulonglong2*>(sC + k * NP + n0);
                        float lo, hi;
                        unpack2(fma2(cv.y, hs[k + 1][1], mul2(cv.x, hs[k + 1][0])), lo, hi);
                        yv[k] = lo + hi;
                    }
                }
            }
            if (z) sum_states<LPC>(yv, sy + ch * LD, q, lane, 1.0f);
        }
        float qv[TS], rv[TS];
        f32x2 t01 = 0, t23 = 0;   // the tile's dA
#pragma unroll
        for (int k = TS - 1; k >= 0; --k) {
            qv[k] = rv[k] = 0.0f;
            if (k < cnt) {
                const float dt = sdt[ch * LD + k], x = sx[ch * LD + k], dy = sdy[ch * LD + k];
                const f32x2 dt2 = pack2(dt, dt), x2 = pack2(x, x), dy2 = pack2(dy, dy);
                const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(sB + k * NP + n0);
                const ulonglong2 cv = *reinterpret_cast<const ulonglong2*>(sC + k * NP + n0);
                const f32x2 g01 = fma2(cv.x, dy2, c01), g23 = fma2(cv.y, dy2, c23);
                float lo, hi, v[8];
                unpack2(fma2(g23, b.y, mul2(g01, b.x)), lo, hi);
                qv[k] = lo + hi;
                unpack2(mul2(g01, x2), v[0], v[1]);
                unpack2(mul2(g23, x2), v[2], v[3]);
                unpack2(mul2(dy2, hs[k + 1][0]), v[4], v[5]);
                unpack2(mul2(dy2, hs[k + 1][1]), v[6], v[7]);
                c01 = mul2(g01, exp2_2(mul2(dt2, A01)));
                c23 = mul2(g23, exp2_2(mul2(dt2, A23)));
                const f32x2 e01 = mul2(c01, hs[k][0]), e23 = mul2(c23, hs[k][1]);
                unpack2(fma2(e23, A23, mul2(e01, A01)), lo, hi);
                rv[k] = lo + hi;
                t01 = fma2(e01, dt2, t01);
                t23 = fma2(e23, dt2, t23);
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
                        const bool hi_half = lane & (half * LPC);
#pragma unroll
                        for (int i = 0; i < m; ++i) {
                            const float send = hi_half ? v[i] : v[i + m];
                            const float keep = hi_half ? v[i + m] : v[i];
                            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, half * LPC);
                        }
                    }
                    const int first = (lane / LPC) % RC * VL;
#pragma unroll
                    for (int i = 0; i < VL; ++i) dst[((first + i) / 4) * NP + (first + i) % 4] = v[i];
                }
            }
        }
        {
            float td[4];
            unpack2(t01, td[0], td[1]);
            unpack2(t23, td[2], td[3]);
#pragma unroll
            for (int i = 0; i < 4; ++i) add_exactly(dA[i], eA[i], td[i]);
        }
        sum_states<LPC>(qv, sq + ch * LD, q, lane, 1.0f);
        sum_states<LPC>(rv, sr + ch * LD, q, lane, kLn2);
        __syncthreads();
        float tD = 0.0f, tb = 0.0f;
#pragma unroll
        for (int k = 0; k < I; ++k) {
            const int it = tid + k * kThreads, ic = it % CH, t4 = it / CH * 4;
            if (it >= CH * (TS / 4) || ic >= w.nch) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (t4 + i >= cnt) continue;
                const int64_t o = (row0 + at + t4 + i) * f.D + w.c0 + ic;
                const int m = ic * LD + t4 + i;
                const float dy = sdy[m], gq = sq[m];
                p.du[o] = from_float<T>(fmaf(gq, sdt[m], Dw[k] * dy));
                const float dd = fmaf(gq, ku[k][i], sr[m]) * ks[k][i];
                p.ddelta[o] = from_float<T>(dd);
                tD = fmaf(dy, ku[k][i], tD);
                tb += dd;
                if (p.dz) p.dz[o] = from_float<T>(kz[k][i] * fmaf(Dw[k], ku[k][i], sy[m]));
            }
        }
        add_exactly(dD, eD, tD);
        add_exactly(db, eb, tb);
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
        unpack2(c01, carry[0], carry[1]);
        unpack2(c23, carry[2], carry[3]);
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

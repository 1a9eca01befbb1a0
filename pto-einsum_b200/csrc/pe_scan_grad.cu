// pe_scan_grad.cu - gradients of the selective scan, for sm_100a.
#include "pe_scan.cuh"

namespace pe {

namespace {

constexpr int K = 8;         // tokens a lane
constexpr int SEG = K + 4;   // a lane's K tokens in a shared row: float4 reads of eight lanes fall on
                             // all banks once
// A warp takes LT K consecutive tokens, a lane K of them, for 32 / LT channels (scan_bwd) or
// channel pairs (scan_adjoint); the block's warps have other channels and the same tokens.
template <int LT>
struct Tile {
    static constexpr int TT = LT * K;                 // tokens
    static constexpr int CB = 2 * (32 / LT) * kWarps; // channels
    static constexpr int RS = LT * SEG + 4;           // row of a [..][token] array
};
__device__ __forceinline__ int at_token(int t) { return t / K * SEG + t % K; }

// B or C of a tile's tokens, rows of NC states as in memory, into fp32 [state][token];
// zero past the last token (a token there must leave the state alone) and state.
template <int LT, int NC, int NT, typename T>
__device__ __forceinline__ void widen_cols(float* dst, const T* src, int cnt, int nn) {
    constexpr int TT = Tile<LT>::TT, RS = Tile<LT>::RS;
#pragma unroll
    for (int i = threadIdx.x; i < TT * NC / 4; i += NT) {
        const int t = i / (NC / 4), n = i % (NC / 4) * 4;
        const Vec<T, 4> v = *reinterpret_cast<const Vec<T, 4>*>(src + t * NC + n);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            dst[(n + e) * RS + at_token(t)] = t < cnt && n + e < nn ? to_float(v.v[e]) : 0.0f;
    }
}

// Eight consecutive floats as four pairs, 16-byte aligned.
struct Pairs {
    f32x2 p[K / 2];
};
__device__ __forceinline__ Pairs load_pairs(const float* s) {
    Pairs r;
#pragma unroll
    for (int i = 0; i < K / 4; ++i) {
        const ulonglong2 v = reinterpret_cast<const ulonglong2*>(s)[i];
        r.p[2 * i] = v.x;
        r.p[2 * i + 1] = v.y;
    }
    return r;
}
__device__ __forceinline__ void store_pairs(float* s, const Pairs& r) {
#pragma unroll
    for (int i = 0; i < K / 4; ++i)
        reinterpret_cast<ulonglong2*>(s)[i] = ulonglong2{r.p[2 * i], r.p[2 * i + 1]};
}
__device__ __forceinline__ void to_scalars(const Pairs& r, float (&f)[K]) {
#pragma unroll
    for (int i = 0; i < K / 2; ++i) unpack2(r.p[i], f[2 * i], f[2 * i + 1]);
}
__device__ __forceinline__ float product(const Pairs& a) {
    float lo, hi;
    unpack2(mul2(mul2(a.p[0], a.p[1]), mul2(a.p[2], a.p[3])), lo, hi);
    return lo * hi;
}
__device__ __forceinline__ f32x2 shfl2_down(f32x2 v, int d, int width) {
    float lo, hi;
    unpack2(v, lo, hi);
    return pack2(__shfl_down_sync(0xffffffffu, lo, d, width), __shfl_down_sync(0xffffffffu, hi, d, width));
}

// What the lanes of a channel (or of a pair, both at once) do to the adjoint state, composed
// from the last token to the first. Lane tl maps the state after it, g, to P g + H. Returns
// the state after the lane, and in `last` the state before lane 0, given the state `h0`
// after the last lane.
template <int LT>
__device__ __forceinline__ f32x2 scan_lanes_down(f32x2 P, f32x2 H, f32x2 h0, int tl, f32x2& last) {
    if (tl == LT - 1) H = fma2(P, h0, H);
#pragma unroll
    for (int d = 1; d < LT; d *= 2) {
        const f32x2 Hu = shfl2_down(H, d, LT), Pu = shfl2_down(P, d, LT);
        if (tl < LT - d) {
            H = fma2(P, Hu, H);
            P = mul2(P, Pu);
        }
    }
    last = H;
    const f32x2 after = shfl2_down(H, 1, LT);
    return tl == LT - 1 ? h0 : after;
}

// One channel, and from the first token to the last.
template <int LT>
__device__ __forceinline__ float scan_lanes_up(float P, float H, float h0, int tl) {
    if (tl == 0) H = fmaf(P, h0, H);
#pragma unroll
    for (int d = 1; d < LT; d *= 2) {
        const float Hu = __shfl_up_sync(0xffffffffu, H, d, LT), Pu = __shfl_up_sync(0xffffffffu, P, d, LT);
        if (tl >= d) {
            H = fmaf(P, Hu, H);
            P *= Pu;
        }
    }
    const float before = __shfl_up_sync(0xffffffffu, H, 1, LT);
    return tl == 0 ? h0 : before;
}
template <int LT>
__device__ __forceinline__ float scan_lanes_down(float P, float H, float h0, int tl, float& last) {
    if (tl == LT - 1) H = fmaf(P, h0, H);
#pragma unroll
    for (int d = 1; d < LT; d *= 2) {
        const float Hu = __shfl_down_sync(0xffffffffu, H, d, LT), Pu = __shfl_down_sync(0xffffffffu, P, d, LT);
        if (tl < LT - d) {
            H = fmaf(P, Hu, H);
            P *= Pu;
        }
    }
    last = H;
    const float after = __shfl_down_sync(0xffffffffu, H, 1, LT);
    return tl == LT - 1 ? h0 : after;
}

constexpr int LT = 8;         // lanes along the tokens: tiles of 64 tokens, one a checkpoint
using L = Tile<LT>;
constexpr int TT = L::TT, CB = L::CB, RS = L::RS;
static_assert(TT == KCK, "a checkpoint a tile");

// ---- backward -------------------------------------------------------------------
template <typename T>
struct GradP {
    ScanP<T> f;
    const T* dout;
    int64_t o_sb, o_st;
    int o_cb;
    const float* dstate;
    T *du, *ddelta, *dz;
    float *dh0;
    float *pBC;       // [2][tiles][G][N][batch * tokens]: each channel tile's share of dB and dC
    float *pA;        // [pieces][D][N]
    float *pD, *pb;   // [pieces][D]
    float *gloc, *dtsum;   // split: each piece's own adjoint state at its start, later the one after it; sum of dt
};

constexpr int kGradThreads = 256, kGradWarps = kGradThreads / 32;
static_assert(CB == 32 / LT * kGradWarps, "a channel for every eight lanes");

template <typename T>
struct GradSmem {
    static constexpr int NC = 8;                         // states at a time: two blocks fit an SM
    alignas(16) T u[TT * CB];                            // as in memory
    T d[TT * CB], z[TT * CB], o[TT * CB], b[TT * NC], c[TT * NC];
    // fp32, [channel or state][token]; the first three end as du, q u + r and y + D u
    alignas(16) float dt[CB * RS];
    float x[CB * RS], dy[CB * RS];
    float B[NC * RS], C[NC * RS];
    float red[kGradWarps][NC][2][TT];                    // a warp's share of dB and dC
    float rows[];   // [N][CB] adjoint states, A log2(e), dA; [CB][N] checkpoint
};

// One block takes 32 channels through a sequence (or a piece of it), tile by tile from
// its end. Per state n a lane composes the maps of its K tokens of its channel forwards
// (from the checkpoint) and backwards (from the tile after), scans them with the other
// seven lanes of the channel, and runs both recurrences again in registers:
//   h = a h' + b,  a = exp(dt A),  b = dt u B;   g = C dy + a' g'
//   q = sum_n g B,  r = sum_n g a h' A:   du = q dt + D dy,  ddt = q u + r
//   dB = sum_c g dt u,  dC = sum_c dy h,  dA = sum_t g a h' dt
// Bound by the instructions issued (about 160 a warp for what the forward pass does in 42)
// and by their latencies: sixteen warps an SM at 128 registers issue in half of the clocks.
// 4 x 2048 tokens of 2048 channels and 16 states take 600 us, 0.45 T states a second. Run
// backwards in time instead, a channel's states stored every tile and recomputed, it took
// 170 instructions, at a quarter of the parallelism. Two channels a lane and eight warps
// were as fast at twice the registers.
template <typename T>
__global__ void __launch_bounds__(kGradThreads, 2) scan_bwd(const __grid_constant__ GradP<T> p) {
    using M = GradSmem<T>;
    constexpr int NC = M::NC, NT = kGradThreads;
    extern __shared__ __align__(16) unsigned char smem[];
    M& m = *reinterpret_cast<M*>(smem);
    const ScanP<T>& f = p.f;
    float *sG = m.rows, *sA = sG + f.N * CB, *sD = sA + f.N * CB, *sK = sD + f.N * CB;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
    if (blockIdx.x == 0 && tid < 32) check_offsets(f.seqs, lane, kSiteOffsets);
    const Place w = place_of<CB>(f);
    const int tl = lane % LT, c = warp * (32 / LT) + lane / LT;
    const int64_t DN = (int64_t)f.D * f.N;
    const int tile = (w.c0 - w.g * f.Dg) / CB;

    if (!w.any) {   // a number that stands for no piece: nothing in the sums
        for (int i = tid; i < w.nch * f.N; i += NT) p.pA[w.number * DN + (int64_t)w.c0 * f.N + i] = 0.0f;
        if (tid < w.nch) p.pD[w.number * f.D + w.c0 + tid] = p.pb[w.number * f.D + w.c0 + tid] = 0.0f;
        return;
    }
    const int64_t start = w.sp.start, len = w.t1;   // tokens are counted from the sequence's start
    const T* u = f.u + w.sp.row * f.u_sb + start * f.u_st + w.c0;
    const T* delta = f.delta + w.sp.row * f.d_sb + start * f.d_st + w.c0;
    const T* z = f.z ? f.z + w.sp.row * f.z_sb + start * f.z_st + w.c0 : nullptr;
    const T* dout = p.dout + w.sp.row * p.o_sb + start * p.o_st + w.c0;
    const T* B = f.B + w.sp.row * f.B_sb + start * f.B_st + w.g * f.B_sg;
    const T* C = f.C + w.sp.row * f.C_sb + start * f.C_st + w.g * f.C_sg;
    const int64_t row0 = w.sp.row * f.seqs.tokens + start;
    const int64_t rows = f.seqs.tokens * (f.seqs.cu ? 1 : f.seqs.nseq);
    const float* ckpt = f.ckpt + piece_base(f.seqs, w.s, KCK) * DN + (int64_t)w.c0 * f.N;
    auto copy_states = [&](int64_t t, int n0) {
        const int cnt = (int)min((int64_t)TT, len - t), nn = min(NC, f.N - n0);
        stage<TT, NC, NT>(m.b, B + t * f.B_st + n0, f.B_st, cnt, nn, f.B_cb);
        stage<TT, NC, NT>(m.c, C + t * f.C_st + n0, f.C_st, cnt, nn, f.C_cb);
    };
    auto copy = [&](int64_t t) {
        const int cnt = (int)min((int64_t)TT, len - t);
        const float* k = ckpt + t / KCK * DN;
        for (int i = tid; i < w.nch * f.N; i += NT) cp_async<4>(sK + i, k + i, 4);
        if (!f.chunks || !p.o_cb) {
            Elements<TT, CB, NT, T> eu, ed, eo, ez;
            Elements<TT, NC, NT, T> eb, ec;
            const int nn = min(NC, f.N);
            eu.load(u + t * f.u_st, f.u_st, cnt, w.nch);
            ed.load(delta + t * f.d_st, f.d_st, cnt, w.nch);
            eo.load(dout + t * p.o_st, p.o_st, cnt, w.nch);
            if (z) ez.load(z + t * f.z_st, f.z_st, cnt, w.nch);
            eb.load(B + t * f.B_st, f.B_st, cnt, nn);
            ec.load(C + t * f.C_st, f.C_st, cnt, nn);
            eu.store(m.u);
            ed.store(m.d);
            eo.store(m.o);
            if (z) ez.store(m.z);
            eb.store(m.b);
            ec.store(m.c);
            return;
        }
        stage<TT, CB, NT>(m.u, u + t * f.u_st, f.u_st, cnt, w.nch, f.u_cb);
        stage<TT, CB, NT>(m.d, delta + t * f.d_st, f.d_st, cnt, w.nch, f.d_cb);
        stage<TT, CB, NT>(m.o, dout + t * p.o_st, p.o_st, cnt, w.nch, p.o_cb);
        if (z) stage<TT, CB, NT>(m.z, z + t * f.z_st, f.z_st, cnt, w.nch, f.z_cb);
        copy_states(t, 0);
    };
    const int64_t top = len > w.t0 ? (len - 1) / TT * TT : -1;
    if (top >= 0) copy(top);
    cp_commit();
    const float* from = p.gloc ? p.gloc + w.number * DN : p.dstate ? p.dstate + w.s * DN : nullptr;
    for (int i = tid; i < CB * f.N; i += NT) {
        const int ci = i / f.N, n = i - ci * f.N;
        const int64_t k = (int64_t)(w.c0 + ci) * f.N + n;
        const bool in = ci < w.nch;
        sG[n * CB + ci] = in && from ? from[k] : 0.0f;
        sA[n * CB + ci] = in ? rate(__ldg(f.A + k)) : 0.0f;
        sD[n * CB + ci] = 0.0f;
        if (!in) sK[i] = 0.0f;
    }
    const float Dw = f.Dw && c < w.nch ? __ldg(f.Dw + w.c0 + c) : 0.0f;
    float dD = 0.0f, db[2] = {0.0f, 0.0f};
    // of the element-wise work: channels cp, cp + 1 of four tokens t4 (a thread's only item)
    const int cp = tid % (CB / 2) * 2, t4 = tid / (CB / 2) * 4;
    static_assert(TT / 4 * (CB / 2) == NT, "one item a thread");
    float bias[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) bias[e] = f.bias && cp + e < w.nch ? __ldg(f.bias + w.c0 + cp + e) : 0.0f;
    float* dtr = m.dt + c * RS + tl * SEG;
    float* xr = m.x + c * RS + tl * SEG;
    float* dyr = m.dy + c * RS + tl * SEG;
    using T2 = Vec<T, 2>;
    auto raw = [&](const T* a, int k) { return *reinterpret_cast<const T2*>(a + (t4 + k) * CB + cp); };

    for (int64_t t = top; t >= w.t0; t -= TT) {
        const int cnt = (int)min((int64_t)TT, len - t);
        Pairs dt, x, dy, y, q, r;
        for (int n0 = 0; n0 < f.N; n0 += NC) {
            const int nn = min(NC, f.N - n0);
            cp_wait();
            __syncthreads();
            if (n0 == 0) {
                // dt, u and dy = dout silu(z), transposed; zero past the last token and channel
                float fd[2][4], fu[2][4], fy[2][4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const T2 vd = raw(m.d, k), vu = raw(m.u, k), vo = raw(m.o, k);
                    T2 vz = vo;
                    if (z) vz = raw(m.z, k);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const bool ok = cp + e < w.nch && t4 + k < cnt;
                        float v = to_float(vd.v[e]) + bias[e];
                        if (f.softplus) v = softplusf(v);
                        fd[e][k] = ok ? v : 0.0f;
                        fu[e][k] = ok ? to_float(vu.v[e]) : 0.0f;
                        v = to_float(vo.v[e]);
                        if (z) {
                            const float zv = to_float(vz.v[e]);
                            v *= zv * sigmoidf(zv);
                        }
                        fy[e][k] = ok ? v : 0.0f;
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int to = (cp + e) * RS + at_token(t4);
                    *reinterpret_cast<float4*>(m.dt + to) = make_float4(fd[e][0], fd[e][1], fd[e][2], fd[e][3]);
                    *reinterpret_cast<float4*>(m.x + to) = make_float4(fu[e][0], fu[e][1], fu[e][2], fu[e][3]);
                    *reinterpret_cast<float4*>(m.dy + to) = make_float4(fy[e][0], fy[e][1], fy[e][2], fy[e][3]);
                }
            }
            widen_cols<LT, NC, NT>(m.B, m.b, cnt, nn);
            widen_cols<LT, NC, NT>(m.C, m.c, cnt, nn);
            __syncthreads();
            if (n0 + NC < f.N) {
                copy_states(t, n0 + NC);
                cp_commit();
            }
            if (n0 == 0) {
                dt = load_pairs(dtr);
                x = load_pairs(xr);
                dy = load_pairs(dyr);
                f32x2 s = 0;
#pragma unroll
                for (int i = 0; i < K / 2; ++i) {
                    s = fma2(x.p[i], dy.p[i], s);
                    x.p[i] = mul2(dt.p[i], x.p[i]);
                    y.p[i] = q.p[i] = r.p[i] = 0;
                }
                dD += halves(s);
            }
#pragma unroll 1
            for (int n = 0; n < nn; ++n) {
                const Pairs Bn = load_pairs(m.B + n * RS + tl * SEG), Cn = load_pairs(m.C + n * RS + tl * SEG);
                const int at = (n0 + n) * CB + c;
                const float g0 = sG[at], h0 = sK[c * f.N + n0 + n];
                const f32x2 A2 = both(sA[at]);
                float a[K], b[K], v[K], P;
                {
                    Pairs ap, bp, vp;
#pragma unroll
                    for (int i = 0; i < K / 2; ++i) {
                        ap.p[i] = decay2(dt.p[i], A2);
                        bp.p[i] = mul2(x.p[i], Bn.p[i]);
                        vp.p[i] = mul2(dy.p[i], Cn.p[i]);
                    }
                    P = product(ap);
                    to_scalars(ap, a);
                    to_scalars(bp, b);
                    to_scalars(vp, v);
                }
                float H = b[0], G = v[K - 1], last;
#pragma unroll
                for (int k = 1; k < K; ++k) {
                    H = fmaf(a[k], H, b[k]);
                    G = fmaf(a[K - k], G, v[K - 1 - k]);
                }
                G *= a[0];
                float h = scan_lanes_up<LT>(P, H, h0, tl);
                float g = scan_lanes_down<LT>(P, G, g0, tl, last);
                if (tl == 0) sG[at] = last;   // the last lane read it before the shuffles
                float s[K], gs[K], hs[K];     // s = a h'
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    s[k] = a[k] * h;
                    gs[K - 1 - k] = g + v[K - 1 - k];
                    h = hs[k] = s[k] + b[k];
                    g = gs[K - 1 - k] * a[K - 1 - k];
                }
                f32x2 sum = 0;
                float vb[K], vc[K];
#pragma unroll
                for (int i = 0; i < K / 2; ++i) {
                    const f32x2 g2 = pack2(gs[2 * i], gs[2 * i + 1]), h2 = pack2(hs[2 * i], hs[2 * i + 1]);
                    y.p[i] = fma2(Cn.p[i], h2, y.p[i]);
                    q.p[i] = fma2(Bn.p[i], g2, q.p[i]);
                    const f32x2 e2 = mul2(g2, pack2(s[2 * i], s[2 * i + 1]));
                    r.p[i] = fma2(e2, A2, r.p[i]);
                    sum = fma2(e2, dt.p[i], sum);
                    unpack2(mul2(g2, x.p[i]), vb[2 * i], vb[2 * i + 1]);
                    unpack2(mul2(h2, dy.p[i]), vc[2 * i], vc[2 * i + 1]);
                }
                float da = halves(sum);
#pragma unroll
                for (int d = LT / 2; d >= 1; d /= 2) da += __shfl_xor_sync(0xffffffffu, da, d);
                if (tl == 0) sD[at] += da;
                // over the warp's four channels: lanes 16 .. 31 end with dC, the odd channels with
                // the second half of the tokens
                const bool hi = lane & 16, odd = lane & 8;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const float send = hi ? vb[k] : vc[k], keep = hi ? vc[k] : vb[k];
                    vb[k] = keep + __shfl_xor_sync(0xffffffffu, send, 16);
                }
#pragma unroll
                for (int k = 0; k < K / 2; ++k) {
                    const float send = odd ? vb[k] : vb[k + K / 2], keep = odd ? vb[k + K / 2] : vb[k];
                    vb[k] = keep + __shfl_xor_sync(0xffffffffu, send, 8);
                }
                *reinterpret_cast<float4*>(&m.red[warp][n][hi][tl * K + (odd ? K / 2 : 0)]) =
                    make_float4(vb[0], vb[1], vb[2], vb[3]);
            }
            __syncthreads();
            for (int i = tid; i < nn * 2 * TT; i += NT) {
                const int k = i % TT, which = i / TT % 2, n = i / (2 * TT);
                if (k >= cnt) continue;
                float s = 0.0f;
#pragma unroll
                for (int v = 0; v < kGradWarps; ++v) s += m.red[v][n][which][k];
                p.pBC[((((int64_t)which * f.ntile + tile) * f.G + w.g) * f.N + n0 + n) * rows + row0 + t + k] = s;
            }
        }
        // a lane's own parts of the rows take what the element-wise work needs
        {
            const Pairs uv = load_pairs(xr);
            const f32x2 D2 = both(Dw), ln2 = both(kLn2);
#pragma unroll
            for (int i = 0; i < K / 2; ++i) {
                dt.p[i] = fma2(q.p[i], dt.p[i], mul2(D2, dy.p[i]));
                r.p[i] = fma2(q.p[i], uv.p[i], mul2(ln2, r.p[i]));
                y.p[i] = fma2(D2, uv.p[i], y.p[i]);
            }
            store_pairs(dtr, dt);
            store_pairs(xr, r);
            store_pairs(dyr, y);
        }
        __syncthreads();
        {
            float du[2][4], dd[2][4], yv[2][4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int at = (cp + e) * RS + at_token(t4);
                const float4 v0 = *reinterpret_cast<const float4*>(m.dt + at);
                const float4 v1 = *reinterpret_cast<const float4*>(m.x + at);
                const float4 v2 = *reinterpret_cast<const float4*>(m.dy + at);
                du[e][0] = v0.x, du[e][1] = v0.y, du[e][2] = v0.z, du[e][3] = v0.w;
                dd[e][0] = v1.x, dd[e][1] = v1.y, dd[e][2] = v1.z, dd[e][3] = v1.w;
                yv[e][0] = v2.x, yv[e][1] = v2.y, yv[e][2] = v2.z, yv[e][3] = v2.w;
            }
            int64_t o = (row0 + t + t4) * f.D + w.c0 + cp;
#pragma unroll
            for (int k = 0; k < 4; ++k, o += f.D) {
                if (t4 + k >= cnt || cp >= w.nch) break;
                T2 vu, vd, vz;
                const T2 rd = raw(m.d, k), ro = raw(m.o, k);
                T2 rz = ro;
                if (p.dz) rz = raw(m.z, k);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float g = dd[e][k];
                    if (f.softplus) g *= sigmoidf(to_float(rd.v[e]) + bias[e]);
                    if (cp + e < w.nch) db[e] += g;
                    vu.v[e] = from_float<T>(du[e][k]);
                    vd.v[e] = from_float<T>(g);
                    if (p.dz) {
                        const float zv = to_float(rz.v[e]);
                        vz.v[e] = from_float<T>(to_float(ro.v[e]) * silu_slope(zv, sigmoidf(zv)) * yv[e][k]);
                    }
                }
                if (f.pairs) {
                    *reinterpret_cast<T2*>(p.du + o) = vu;
                    *reinterpret_cast<T2*>(p.ddelta + o) = vd;
                    if (p.dz) *reinterpret_cast<T2*>(p.dz + o) = vz;
                } else {
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (cp + e < w.nch) {
                            p.du[o + e] = vu.v[e];
                            p.ddelta[o + e] = vd.v[e];
                            if (p.dz) p.dz[o + e] = vz.v[e];
                        }
                }
            }
        }
        if (t > w.t0) {
            __syncthreads();
            copy(t - TT);
            cp_commit();
        }
    }
    __syncthreads();
    for (int i = tid; i < w.nch * f.N; i += NT) {
        const int ci = i / f.N, n = i - ci * f.N;
        const int64_t k = (int64_t)(w.c0 + ci) * f.N + n;
        p.pA[w.number * DN + k] = sD[n * CB + ci];
        if (p.dh0 && w.j == 0) p.dh0[w.s * DN + k] = sG[n * CB + ci];
    }
#pragma unroll
    for (int d = LT / 2; d >= 1; d /= 2) dD += __shfl_xor_sync(0xffffffffu, dD, d);
    if (tl == 0 && c < w.nch) p.pD[w.number * f.D + w.c0 + c] = dD;
#pragma unroll
    for (int e = 0; e < 2; ++e) m.dt[e * NT + tid] = db[e];
    __syncthreads();
    if (tid < w.nch) {
        float s = 0.0f;
        for (int k = tid / 2; k < NT; k += CB / 2) s += m.dt[tid % 2 * NT + k];
        p.pb[w.number * f.D + w.c0 + tid] = s;
    }
}

// The first half of a backward pass split along the tokens: the adjoint state at a
// piece's start that the piece's own tokens give, and its sum of dt. As scan_bwd, with
// nothing but g's recurrence; half of scan_bwd's time for the same tokens.
template <typename T>
struct AdjSmem {
    static constexpr int NC = 16;
    alignas(16) T d[TT * CB];
    T z[TT * CB], o[TT * CB], c[TT * NC];
    alignas(16) float dt[CB * RS];
    float dy[CB * RS], C[NC * RS];
    float rows[];   // [N][CB] adjoint states, A log2(e)
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 3) scan_adjoint(const __grid_constant__ GradP<T> p) {
    using M = AdjSmem<T>;
    constexpr int NC = M::NC;
    extern __shared__ __align__(16) unsigned char smem[];
    M& m = *reinterpret_cast<M*>(smem);
    const ScanP<T>& f = p.f;
    float *sG = m.rows, *sA = sG + f.N * CB;
    const int tid = threadIdx.x, lane = tid & 31;
    const Place w = place_of<CB>(f);
    if (!w.any || w.j == 0) return;   // nothing comes before a sequence's first piece
    const int tl = lane % LT, c = 2 * (tid / 32 * (32 / LT) + lane / LT);
    const int64_t DN = (int64_t)f.D * f.N;
    const int64_t start = w.sp.start, len = w.t1;
    const T* delta = f.delta + w.sp.row * f.d_sb + start * f.d_st + w.c0;
    const T* z = f.z ? f.z + w.sp.row * f.z_sb + start * f.z_st + w.c0 : nullptr;
    const T* dout = p.dout + w.sp.row * p.o_sb + start * p.o_st + w.c0;
    const T* C = f.C + w.sp.row * f.C_sb + start * f.C_st + w.g * f.C_sg;
    auto copy_states = [&](int64_t t, int n0) {
        stage<TT, NC>(m.c, C + t * f.C_st + n0, f.C_st, (int)min((int64_t)TT, len - t), min(NC, f.N - n0), f.C_cb);
    };
    auto copy = [&](int64_t t) {
        const int cnt = (int)min((int64_t)TT, len - t);
        if (!f.d_cb || !p.o_cb || (z && !f.z_cb)) {
            Elements<TT, CB, kThreads, T> ed, eo, ez;
            ed.load(delta + t * f.d_st, f.d_st, cnt, w.nch);
            eo.load(dout + t * p.o_st, p.o_st, cnt, w.nch);
            if (z) ez.load(z + t * f.z_st, f.z_st, cnt, w.nch);
            ed.store(m.d);
            eo.store(m.o);
            if (z) ez.store(m.z);
            return;
        }
        stage<TT, CB>(m.d, delta + t * f.d_st, f.d_st, cnt, w.nch, f.d_cb);
        stage<TT, CB>(m.o, dout + t * p.o_st, p.o_st, cnt, w.nch, p.o_cb);
        if (z) stage<TT, CB>(m.z, z + t * f.z_st, f.z_st, cnt, w.nch, f.z_cb);
    };
    const int64_t top = (len - 1) / TT * TT;
    copy(top);
    copy_states(top, 0);
    cp_commit();
    for (int i = tid; i < CB * f.N; i += kThreads) {
        const int ci = i / f.N, n = i - ci * f.N;
        sG[n * CB + ci] = 0.0f;
        sA[n * CB + ci] = ci < w.nch ? rate(__ldg(f.A + (int64_t)(w.c0 + ci) * f.N + n)) : 0.0f;
    }
    const int cp = tid % (CB / 2) * 2;
    float bias[2], dtsum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 2; ++e) bias[e] = f.bias && cp + e < w.nch ? __ldg(f.bias + w.c0 + cp + e) : 0.0f;

    for (int64_t t = top; t >= w.t0; t -= TT) {
        const int cnt = (int)min((int64_t)TT, len - t);
        Pairs dt[2], dy[2];
        for (int n0 = 0; n0 < f.N; n0 += NC) {
            const int nn = min(NC, f.N - n0);
            cp_wait();
            __syncthreads();
            if (n0 == 0) {
#pragma unroll 2
                for (int i = tid; i < TT / 4 * (CB / 2); i += kThreads) {
                    const int t4 = i / (CB / 2) * 4;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float fd[4], fy[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int at = (t4 + k) * CB + cp + e;
                            const bool ok = cp + e < w.nch && t4 + k < cnt;
                            float v = to_float(m.d[at]) + bias[e];
                            if (f.softplus) v = softplusf(v);
                            fd[k] = ok ? v : 0.0f;
                            v = to_float(m.o[at]);
                            if (z) {
                                const float zv = to_float(m.z[at]);
                                v *= zv * sigmoidf(zv);
                            }
                            fy[k] = ok ? v : 0.0f;
                        }
                        const int to = (cp + e) * RS + at_token(t4);
                        *reinterpret_cast<float4*>(m.dt + to) = make_float4(fd[0], fd[1], fd[2], fd[3]);
                        *reinterpret_cast<float4*>(m.dy + to) = make_float4(fy[0], fy[1], fy[2], fy[3]);
                    }
                }
            }
            widen_cols<LT, NC, kThreads>(m.C, m.c, cnt, nn);
            __syncthreads();
            if (n0 + NC < f.N) {
                copy_states(t, n0 + NC);
            } else if (t > w.t0) {
                copy(t - TT);
                copy_states(t - TT, 0);
            }
            cp_commit();
            if (n0 == 0) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    dt[e] = load_pairs(m.dt + (c + e) * RS + tl * SEG);
                    dy[e] = load_pairs(m.dy + (c + e) * RS + tl * SEG);
                    float s[K];
                    to_scalars(dt[e], s);
#pragma unroll
                    for (int k = 0; k < K; ++k) dtsum[e] += s[k];
                }
            }
#pragma unroll 1
            for (int n = 0; n < nn; ++n) {
                const Pairs Cn = load_pairs(m.C + n * RS + tl * SEG);
                const int at = (n0 + n) * CB + c;
                const float2 A = *reinterpret_cast<const float2*>(sA + at);
                f32x2* gp = reinterpret_cast<f32x2*>(sG + at);
                const f32x2 g0 = *gp;
                float P[2], G[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float Ae = e ? A.y : A.x;
                    const f32x2 A2 = pack2(Ae, Ae);
                    Pairs ap, vp;
                    float a[K], v[K];
#pragma unroll
                    for (int i = 0; i < K / 2; ++i) {
                        ap.p[i] = decay2(dt[e].p[i], A2);
                        vp.p[i] = mul2(dy[e].p[i], Cn.p[i]);
                    }
                    P[e] = product(ap);
                    to_scalars(ap, a);
                    to_scalars(vp, v);
                    G[e] = v[K - 1];
#pragma unroll
                    for (int k = 1; k < K; ++k) G[e] = fmaf(a[K - k], G[e], v[K - 1 - k]);
                    G[e] *= a[0];
                }
                f32x2 last;
                scan_lanes_down<LT>(pack2(P[0], P[1]), pack2(G[0], G[1]), g0, tl, last);
                if (tl == 0) *gp = last;   // the last lane read it before the shuffles
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < w.nch * f.N; i += kThreads) {
        const int ci = i / f.N, n = i - ci * f.N;
        p.gloc[w.number * DN + (int64_t)(w.c0 + ci) * f.N + n] = sG[n * CB + ci];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = LT / 2; d >= 1; d /= 2) dtsum[e] += __shfl_xor_sync(0xffffffffu, dtsum[e], d);
        if (tl == 0 && c + e < w.nch) p.dtsum[w.number * f.D + w.c0 + c + e] = dtsum[e];
    }
}

// Each piece's own adjoint state gives way to the one after the piece, from the
// sequence's end. One thread a (sequence, channel, state).
template <typename T>
__global__ void __launch_bounds__(kThreads) adjoint_carry(const __grid_constant__ GradP<T> p) {
    const ScanP<T>& f = p.f;
    const int64_t DN = (int64_t)f.D * f.N, i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= DN) return;
    const int s = blockIdx.y;
    const int64_t len = seq_span(f.seqs, s).len, base = piece_base(f.seqs, s, f.piece);
    const int64_t n = len > f.piece ? ceil_div(len, f.piece) : 1;
    const float A = rate(__ldg(f.A + i));
    float g = p.dstate ? __ldg(p.dstate + s * DN + i) : 0.0f;
    float* gp = p.gloc + base * DN + i;
    const float* sp = p.dtsum + base * f.D + i / f.N;
    for (int64_t k0 = n - 1; k0 >= 0; k0 -= 8) {
        float own[8], keep[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k0 - k > 0) {
                own[k] = gp[(k0 - k) * DN];
                keep[k] = exp2_fast(A * __ldg(sp + (k0 - k) * f.D));
            }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k0 - k >= 0) {
                gp[(k0 - k) * DN] = g;
                if (k0 - k > 0) g = fmaf(keep[k], g, own[k]);
            }
    }
}

// dB and dC [row][G N] from the channel tiles' shares [tile][G N][row]: 32 rows by 32
// columns a block, transposed in shared memory; blockIdx.z 0 is dB, 1 dC. Bound by memory.
template <typename T>
__global__ void __launch_bounds__(256) sum_tiles(const float* __restrict__ part, int ntile, int64_t rows, int cols,
                                                 T* dB, T* dC) {
    __shared__ float s[32][33];
    const int x = threadIdx.x % 32, y = threadIdx.x / 32;
    const int64_t r0 = (int64_t)blockIdx.x * 32;
    const int c0 = blockIdx.y * 32;
    part += (int64_t)blockIdx.z * ntile * cols * rows;
    T* out = blockIdx.z ? dC : dB;
#pragma unroll
    for (int k = y; k < 32; k += 8) {
        float a = 0.0f;
        if (c0 + k < cols && r0 + x < rows) {
            const float* b = part + (int64_t)(c0 + k) * rows + r0 + x;
#pragma unroll 8
            for (int i = 0; i < ntile; ++i) a += __ldg(b + (int64_t)i * cols * rows);
        }
        s[k][x] = a;
    }
    __syncthreads();
#pragma unroll
    for (int k = y; k < 32; k += 8)
        if (r0 + k < rows && c0 + x < cols) out[(r0 + k) * cols + c0 + x] = from_float<T>(s[x][k]);
}

// ---- host -------------------------------------------------------------------------
// Tokens a piece of the backward pass; 0 = whole sequences. A block that has an SM to
// itself leaves most of it idle, and the pass that finds the adjoint states between
// pieces costs half as much as the pass itself: split where there are fewer blocks than
// SMs, into as many pieces as two blocks an SM take. Forward and backward of a bf16
// sequence with 16 states, split against whole: 1024 x 256 62 and 237 us, 4096 x 2048
// 585 and 1028, 4096 x 4096 (128 blocks) 1107 and 1153; two blocks an SM and more give a
// rule of this form one piece.
int64_t grad_piece(const pe_scan_args* a) {
    const int64_t tiles = a->groups * ceil_div(a->channels / a->groups, CB), rows = a->cu ? 1 : a->nseq;
    const int64_t blocks = a->nseq * tiles;
    if (blocks < 1 || a->nseq > 65535 || blocks >= num_sms() || a->tokens / (a->nseq / rows) < 4 * KCK)
        return 0;
    int64_t pieces = 2 * num_sms() / (rows * tiles) - (a->cu ? a->nseq : 0);
    if (pieces < 2) return 0;
    return ceil_div(ceil_div(a->tokens, pieces), KCK) * KCK;
}

struct GradWs {
    int64_t piece, pieces, bc, a, d, b, g, s, total;   // tokens a piece, pieces; float offsets
};
GradWs grad_ws(const pe_scan_args* a) {
    const int64_t rows = a->tokens * (a->cu ? 1 : a->nseq), DN = a->channels * a->states;
    GradWs w;
    w.piece = grad_piece(a);
    w.pieces = piece_count(seqs_of(a), w.piece ? w.piece : (a->tokens / KCK + 1) * KCK);
    w.bc = 0;
    w.a = 2 * ceil_div(a->channels / a->groups, CB) * rows * a->groups * a->states;
    w.d = w.a + w.pieces * DN;
    w.b = w.d + w.pieces * a->channels;
    w.g = w.b + w.pieces * a->channels;
    w.s = w.g + (w.piece ? w.pieces * DN : 0);
    w.total = w.s + (w.piece ? w.pieces * a->channels : 0);
    return w;
}

template <typename T>
int grad_type(const pe_scan_grad_args* a, cudaStream_t s) {
    const pe_scan_args* f = &a->fwd;
    GradP<T> p;
    p.f = scan_params<T>(f, CB, GradSmem<T>::NC);
    const GradWs w = grad_ws(f);
    float* ws = (float*)a->ws;
    p.dout = (const T*)a->dout; p.o_sb = a->dout_sb; p.o_st = a->dout_st;
    p.o_cb = chunk_of(p.dout, sizeof(T), CB * sizeof(T), {p.o_sb, p.o_st, CB}, p.f.G > 1 ? p.f.Dg : CB);
    p.dstate = a->dstate;
    p.du = (T*)a->du; p.ddelta = (T*)a->ddelta; p.dz = (T*)a->dz;
    p.dh0 = a->dh0;
    p.f.pairs = p.f.Dg % 2 == 0 &&
                ((uintptr_t)p.du | (uintptr_t)p.ddelta | (uintptr_t)p.dz) % (2 * sizeof(T)) == 0;
    p.pBC = ws + w.bc; p.pA = ws + w.a; p.pD = ws + w.d; p.pb = ws + w.b;
    p.gloc = p.dtsum = nullptr;
    unsigned grid;
    if (int rc = grid_of(w.pieces * p.f.G * p.f.ntile, &grid)) return rc;
    if (f->nseq == 0) grid = 0;
    if (grid && w.piece) {
        p.f.split(w.piece);
        p.gloc = ws + w.g;
        p.dtsum = ws + w.s;
        if (int rc = launch(scan_adjoint<T>, p, grid, sizeof(AdjSmem<T>) + 2 * p.f.N * CB * 4, s)) return rc;
        const dim3 blocks((unsigned)ceil_div(f->channels * f->states, kThreads), (unsigned)f->nseq);
        adjoint_carry<T><<<blocks, kThreads, 0, s>>>(p);
        count_launch();
        if (cudaGetLastError() != cudaSuccess) return PE_ERR_CUDA;
    }
    if (grid)
        if (int rc = launch(scan_bwd<T>, p, grid, sizeof(GradSmem<T>) + 4 * p.f.N * CB * 4, s, kGradThreads)) return rc;
    const int64_t rows = f->tokens * (f->cu ? 1 : f->nseq), cols = f->groups * f->states;
    if (rows) {
        if (ceil_div(rows, 32) > 0x7fffffffll || ceil_div(cols, 32) > 65535) return PE_ERR_UNSUPPORTED;
        const dim3 blocks((unsigned)ceil_div(rows, 32), (unsigned)ceil_div(cols, 32), 2);
        sum_tiles<T><<<blocks, 256, 0, s>>>(p.pBC, p.f.ntile, rows, (int)cols, (T*)a->dB, (T*)a->dC);
        count_launch();
        if (cudaGetLastError() != cudaSuccess) return PE_ERR_CUDA;
    }
    const SumJob sums[3] = {{p.pA, grid ? w.pieces : 0, f->channels * f->states, PE_F32, a->dA},
                            {p.pD, grid ? w.pieces : 0, f->channels, PE_F32, a->dD},
                            {p.pb, grid ? w.pieces : 0, f->channels, PE_F32, a->ddelta_bias}};
    return sum_rows(sums, 3, s);
}

int grad_any(const pe_scan_grad_args* a, cudaStream_t s) { PE_TYPES(grad_type, a->fwd.dtype, a, s) }

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

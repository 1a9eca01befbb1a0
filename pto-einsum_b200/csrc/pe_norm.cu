// pe_norm.cu - group norm over channels-last tensors with silu or a silu gate,
// forward and backward, for sm_100a.
//
//   xn = (x - mean) rstd,  v = xn w + b,  out = v | silu(v) | v silu(gate)
//   g = d out / d v . dout,  dw = sum g xn,  db = sum g,
//   dx = rstd (g w - mean(g w) - xn mean(g w xn))          (means over the group)
//
// Bound by memory. A small group stays in the registers of the lanes that share it: one
// read of x, two-pass statistics. A larger one of a single place is a block's, in L1; of
// several places it stays in the shared memory of a cluster of up to eight blocks, while
// the SMs hold all clusters at once. Else the tensor is read twice: per-channel sums of
// row chunks, their combination, then the result; the second read comes from L2 while the
// tensor fits there. Variances are never formed as a difference of large squares: two
// passes in registers, and sums shifted by a first value that are joined by Chan's formula
// elsewhere. Every sum has a fixed order. Times in the comments are of a B200, by replays
// of a captured call.
#include "pe_mixer.cuh"

namespace pe {

namespace {

constexpr int kBlock = 256;
enum Mode { kPlain = 0, kSilu = 1, kGate = 2 };

template <typename T>
struct NormP {
    int64_t N, S, C;
    int G, cg, mode;
    float eps;
    const T *x, *w, *b, *gate;
    int64_t x_sb, x_sp, g_sb, g_sp;
    T* out;
    float *mean, *rstd;
    // backward
    const T* dout;
    int64_t o_sb, o_sp;
    T *dx, *dgate;
};

// ---- groups in registers ------------------------------------------------------------
// Sum over the L lanes of a group: part of a warp (L <= 32) or the whole block.
template <int NV>
__device__ __forceinline__ void group_sum(float (&v)[NV], int L, float* red) {
    if (L <= 32) {
#pragma unroll
        for (int m = 16; m >= 1; m /= 2)
            if (m < L)
#pragma unroll
                for (int i = 0; i < NV; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], m);
        return;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
#pragma unroll
    for (int m = 16; m >= 1; m /= 2)
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], m);
    __syncthreads();
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < NV; ++i) red[i * 8 + warp] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        v[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < kBlock / 32; ++k) v[i] += red[i * 8 + k];
    }
}

// Blocks an SM holds of the kernels below, by loads a lane and elements a load.
__host__ __device__ constexpr int reg_blocks(int k, int v, bool grad) {
    if (v == 1) return k <= 2 ? 4 : 2;
    return grad ? (k == 1 ? 2 : 1) : k == 1 ? 3 : k == 2 ? 2 : 1;
}

// The items of a lane: item i of a group is channel vector i % per of place i / per.
template <int V, int K>
struct Items {
    bool in[K];
    int place[K], c[K];
    __device__ __forceinline__ Items(int l, int L, int per, int items, int c0) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = l + k * L;
            in[k] = i < items;
            place[k] = in[k] ? i / per : 0;
            c[k] = in[k] ? c0 + (i - place[k] * per) * V : 0;
        }
    }
};

// L lanes share a group and take its rows r, r + R, ...; the next three rows are on their
// way while the current one is reduced. All lanes make the same number of rounds, for
// the shuffles take all of them. 8192 rows of 4096 bf16 channels in 32 gated groups: 45 us,
// 4.5 TB/s; the next row alone, in registers, 71. One wave of blocks (R rows at work) against
// one row a group of lanes: 44 and 97 us.
template <typename T, int V, int K>
__global__ void __launch_bounds__(kBlock, reg_blocks(K, V, false)) norm_reg(const __grid_constant__ NormP<T> p, int L, int R) {
    __shared__ float red[8];
    const int unit = (int)(((int64_t)blockIdx.x * kBlock + threadIdx.x) / L), l = threadIdx.x % L;
    const bool live = unit / p.G < R;
    const int r = live ? unit / p.G : 0, g = live ? unit % p.G : 0;
    const int per = p.cg / V;
    const Items<V, K> it(l, L, per, live ? per * (int)p.S : 0, g * p.cg);
    const float inv = 1.0f / (float)(p.cg * (int)p.S);
    constexpr int Q = kPairs<V>;
    constexpr int DEPTH = 4;   // three rows on their way
    extern __shared__ __align__(16) unsigned char queues[];
    constexpr int each_queue = DEPTH * K * kBlock * kSlotBytes<T, V>;
    Ring<T, V, DEPTH * K> rx(queues, kBlock), rz(queues + each_queue, kBlock);
    auto at_x = [&](int64_t n, int k) { return p.x + n * p.x_sb + it.place[k] * p.x_sp + it.c[k]; };
    auto at_gate = [&](int64_t n, int k) { return p.gate + n * p.g_sb + it.place[k] * p.g_sp + it.c[k]; };
    f32x2 w[K][Q], b[K][Q];
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int q = 0; q < Q; ++q) w[k][q] = both(1.0f), b[k][q] = 0;
        if (it.in[k] && p.w) widen<T, V>(load_vec<T, V>(p.w + it.c[k]), w[k]);
        if (it.in[k] && p.b) widen<T, V>(load_vec<T, V>(p.b + it.c[k]), b[k]);
    }
    auto fetch = [&](int64_t n, int step) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const bool on = it.in[k] && n < p.N;
            rx.fetch(step * K + k, at_x(n, k), on);
            if (p.mode == kGate) rz.fetch(step * K + k, at_gate(n, k), on);
        }
        cp_commit();
    };
#pragma unroll
    for (int i = 0; i < DEPTH - 1; ++i) fetch(r + (int64_t)i * R, i);
    int step = 0;
    for (int64_t n0 = 0; n0 < p.N; n0 += R, ++step) {
        const int64_t n = n0 + r;
        const bool on = n < p.N;
        f32x2 f[K][Q], ga[K][Q];
        float sum[1] = {0.0f};
        cp_wait_but<DEPTH - 2>();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            widen<T, V>(rx.get(step * K + k, at_x(n, k)), f[k]);
            if (p.mode == kGate) widen<T, V>(rz.get(step * K + k, at_gate(n, k)), ga[k]);
            f32x2 s = f[k][0];
#pragma unroll
            for (int q = 1; q < Q; ++q) s = add2(s, f[k][q]);
            sum[0] += it.in[k] ? halves(s) : 0.0f;
        }
        fetch(n + (DEPTH - 1) * (int64_t)R, step + DEPTH - 1);   // into the slots of the row before this one
        group_sum(sum, L, red);
        const float mean = sum[0] * inv;
        const f32x2 minus = each<V>(-mean);
        sum[0] = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            f32x2 s = 0;
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                f[k][q] = add2(f[k][q], minus);
                s = fma2(f[k][q], f[k][q], s);
            }
            sum[0] += it.in[k] ? halves(s) : 0.0f;
        }
        group_sum(sum, L, red);
        const float rstd = rsqrtf(sum[0] * inv + p.eps);
        if (!live || !on) continue;
        if (l == 0 && p.mean) {
            p.mean[n * p.G + g] = mean;
            p.rstd[n * p.G + g] = rstd;
        }
        const f32x2 scale = both(rstd);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!it.in[k]) continue;
            f32x2 y[Q];
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                y[q] = fma2(mul2(f[k][q], scale), w[k][q], b[k][q]);
                if (p.mode == kSilu) y[q] = mul2(y[q], sigmoid2(y[q]));
                if (p.mode == kGate) y[q] = mul2(y[q], mul2(ga[k][q], sigmoid2(ga[k][q])));
            }
            store_vec(p.out + (n * p.S + it.place[k]) * p.C + it.c[k], narrow<T, V>(y));
        }
    }
    cp_wait();
}

// g = dL / dv, and the gate's gradient in place of `ga`.
template <int Q>
__device__ __forceinline__ void through_act2(int mode, const f32x2 (&xn)[Q], const f32x2 (&w)[Q], const f32x2 (&b)[Q],
                                             f32x2 (&go)[Q], f32x2 (&ga)[Q]) {
    if (mode == kPlain) return;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const f32x2 val = fma2(xn[q], w[q], b[q]);
        if (mode == kSilu) {
            go[q] = mul2(go[q], silu_slope2(val, sigmoid2(val)));
        } else {
            const f32x2 s = sigmoid2(ga[q]), o = go[q];
            go[q] = mul2(o, mul2(ga[q], s));
            ga[q] = mul2(mul2(o, val), silu_slope2(ga[q], s));
        }
    }
}

// L lanes take rows r, r + R, ... of one group of channels (one place a row) and keep the
// sums of g xn and g of their own channels: pw, pb [R][C]. The rows above: 66 us, 5.1 TB/s
// (92 with the next row in registers).
template <typename T, int V, int K>
__global__ void __launch_bounds__(kBlock, reg_blocks(K, V, true)) norm_reg_bwd(const __grid_constant__ NormP<T> p, int L,
                                                                            int R, float* pw, float* pb) {
    constexpr int Q = kPairs<V>;
    __shared__ float red[16];
    const int unit = (int)(((int64_t)blockIdx.x * kBlock + threadIdx.x) / L), l = threadIdx.x % L;
    const bool live = unit / p.G < R;
    const int r = live ? unit / p.G : 0, g = live ? unit % p.G : 0;
    const int per = p.cg / V;
    const Items<V, K> it(l, L, per, live ? per : 0, g * p.cg);
    const float inv = 1.0f / (float)p.cg;
    constexpr int DEPTH = 4;
    extern __shared__ __align__(16) unsigned char queues[];
    constexpr int each_queue = DEPTH * K * kBlock * kSlotBytes<T, V>;
    Ring<T, V, DEPTH * K> rx(queues, kBlock), ro(queues + each_queue, kBlock), rz(queues + 2 * each_queue, kBlock);
    f32x2 aw[K][Q], ab[K][Q], w[K][Q], b[K][Q];
    float mean = 0.0f, rstd = 0.0f, mean2 = 0.0f, rstd2 = 0.0f;   // of this row and the next
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int q = 0; q < Q; ++q) aw[k][q] = ab[k][q] = b[k][q] = 0, w[k][q] = each<V>(1.0f);
        if (it.in[k] && p.w) widen<T, V>(load_vec<T, V>(p.w + it.c[k]), w[k]);
        if (it.in[k] && p.b) widen<T, V>(load_vec<T, V>(p.b + it.c[k]), b[k]);
    }
    auto fetch = [&](int64_t n, int step) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const bool on = it.in[k] && n < p.N;
            rx.fetch(step * K + k, p.x + n * p.x_sb + it.c[k], on);
            ro.fetch(step * K + k, p.dout + n * p.o_sb + it.c[k], on);
            if (p.mode == kGate) rz.fetch(step * K + k, p.gate + n * p.g_sb + it.c[k], on);
        }
        cp_commit();
    };
    auto stats = [&](int64_t n) {
        if (n < p.N) {
            mean2 = __ldg(p.mean + n * p.G + g);
            rstd2 = __ldg(p.rstd + n * p.G + g);
        }
    };
#pragma unroll
    for (int i = 0; i < DEPTH - 1; ++i) fetch(r + (int64_t)i * R, i);
    stats(r);
    int step = 0;
    for (int64_t n0 = 0; n0 < p.N; n0 += R, ++step) {
        const int64_t n = n0 + r;
        const bool on = n < p.N;
        mean = mean2;
        rstd = rstd2;
        stats(n + R);
        cp_wait_but<DEPTH - 2>();
        const f32x2 minus = each<V>(-mean), scale = both(rstd);
        f32x2 xn[K][Q], go[K][Q];
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!it.in[k] || !on) continue;
            f32x2 ga[Q], s0 = 0, s1 = 0;
            widen<T, V>(rx.get(step * K + k, p.x + n * p.x_sb + it.c[k]), xn[k]);
            widen<T, V>(ro.get(step * K + k, p.dout + n * p.o_sb + it.c[k]), go[k]);
            if (p.mode == kGate) widen<T, V>(rz.get(step * K + k, p.gate + n * p.g_sb + it.c[k]), ga);
#pragma unroll
            for (int q = 0; q < Q; ++q) xn[k][q] = mul2(add2(xn[k][q], minus), scale);
            through_act2<Q>(p.mode, xn[k], w[k], b[k], go[k], ga);
            if (p.mode == kGate) store_vec(p.dgate + n * p.C + it.c[k], narrow<T, V>(ga));
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                aw[k][q] = fma2(go[k][q], xn[k][q], aw[k][q]);
                ab[k][q] = add2(ab[k][q], go[k][q]);
                go[k][q] = mul2(go[k][q], w[k][q]);
                s0 = add2(s0, go[k][q]);
                s1 = fma2(go[k][q], xn[k][q], s1);
            }
            sum[0] += halves(s0);
            sum[1] += halves(s1);
        }
        fetch(n + (DEPTH - 1) * (int64_t)R, step + DEPTH - 1);   // into the slots of the row before this one
        group_sum(sum, L, red);
        const f32x2 m0 = both(-sum[0] * inv), m1 = both(-sum[1] * inv);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!it.in[k] || !on) continue;
            f32x2 d[Q];
#pragma unroll
            for (int q = 0; q < Q; ++q) d[q] = mul2(scale, fma2(xn[k][q], m1, add2(go[k][q], m0)));
            store_vec(p.dx + n * p.C + it.c[k], narrow<T, V>(d));
        }
    }
    cp_wait();
    if (!pw) return;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (!it.in[k]) continue;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float a[2], c[2];
            unpack2(aw[k][v / 2], a[0], a[1]);
            unpack2(ab[k][v / 2], c[0], c[1]);
            pw[(int64_t)r * p.C + it.c[k] + v] = a[v % 2];
            pb[(int64_t)r * p.C + it.c[k] + v] = c[v % 2];
        }
    }
}

// ---- one place a row, too many channels for registers ------------------------------------
// A block takes a group of one row; the passes after the first find it in L1. 4096 gated
// rows of 8192 bf16 channels: 49 us, 4.1 TB/s.
template <typename T, int V>
__global__ void __launch_bounds__(kBlock) norm_wide(const __grid_constant__ NormP<T> p) {
    constexpr int Q = kPairs<V>;
    __shared__ float red[8];
    const int64_t n = blockIdx.x / (unsigned)p.G;
    const int g = blockIdx.x % (unsigned)p.G, c0 = g * p.cg;
    const T* x = p.x + n * p.x_sb + c0;
    const float inv = 1.0f / (float)p.cg;
    f32x2 s = 0;
    float sum[1];
#pragma unroll 4
    for (int c = threadIdx.x * V; c < p.cg; c += kBlock * V) {
        f32x2 f[Q];
        widen<T, V>(load_vec<T, V>(x + c), f);
#pragma unroll
        for (int q = 0; q < Q; ++q) s = add2(s, f[q]);
    }
    sum[0] = halves(s);
    group_sum(sum, kBlock, red);
    const float mean = sum[0] * inv;
    const f32x2 minus = each<V>(-mean);
    s = 0;
#pragma unroll 4
    for (int c = threadIdx.x * V; c < p.cg; c += kBlock * V) {
        f32x2 f[Q];
        widen<T, V>(load_vec<T, V>(x + c), f);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            f[q] = add2(f[q], minus);
            s = fma2(f[q], f[q], s);
        }
    }
    sum[0] = halves(s);
    group_sum(sum, kBlock, red);
    const float rstd = rsqrtf(sum[0] * inv + p.eps);
    if (threadIdx.x == 0 && p.mean) {
        p.mean[blockIdx.x] = mean;
        p.rstd[blockIdx.x] = rstd;
    }
    const f32x2 scale = both(rstd);
#pragma unroll 2
    for (int c = threadIdx.x * V; c < p.cg; c += kBlock * V) {
        f32x2 f[Q], w[Q], b[Q], ga[Q];
        widen<T, V>(load_vec<T, V>(x + c), f);
#pragma unroll
        for (int q = 0; q < Q; ++q) w[q] = both(1.0f), b[q] = 0;
        if (p.w) widen<T, V>(load_vec<T, V>(p.w + c0 + c), w);
        if (p.b) widen<T, V>(load_vec<T, V>(p.b + c0 + c), b);
        if (p.mode == kGate) widen<T, V>(load_vec<T, V>(p.gate + n * p.g_sb + c0 + c), ga);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            f[q] = fma2(mul2(add2(f[q], minus), scale), w[q], b[q]);
            if (p.mode == kSilu) f[q] = mul2(f[q], sigmoid2(f[q]));
            if (p.mode == kGate) f[q] = mul2(f[q], mul2(ga[q], sigmoid2(ga[q])));
        }
        store_vec(p.out + n * p.C + c0 + c, narrow<T, V>(f));
    }
}

// The sums of V channels, from and to memory.
template <int V>
__device__ __forceinline__ void load_sums(const float* from, f32x2 (&s)[kPairs<V>]) {
    if constexpr (V == 1) {
        s[0] = pack2(*from, 0.0f);
    } else {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const float4 v = reinterpret_cast<const float4*>(from)[i];
            s[2 * i] = pack2(v.x, v.y);
            s[2 * i + 1] = pack2(v.z, v.w);
        }
    }
}
template <int V>
__device__ __forceinline__ void store_sums(float* to, const f32x2 (&s)[kPairs<V>]) {
    float h[2 * kPairs<V>];
#pragma unroll
    for (int q = 0; q < kPairs<V>; ++q) unpack2(s[q], h[2 * q], h[2 * q + 1]);
    if constexpr (V == 1) {
        *to = h[0];
    } else {
#pragma unroll
        for (int i = 0; i < V / 4; ++i)
            reinterpret_cast<float4*>(to)[i] = make_float4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
    }
}

// Backward: rows r, r + R, ... of one group a block. The sums of g xn and g of a channel
// belong to the thread that has the channel: in shared memory (LOCAL; a plane for each
// element of a load, for no two lanes share a bank then), or, where that is too small,
// in their places of pw and pb. The rows above: 132 us, 2.5 TB/s.
template <typename T, int V, bool LOCAL>
__global__ void __launch_bounds__(kBlock, 2) norm_wide_bwd(const __grid_constant__ NormP<T> p, int R, float* pw, float* pb) {
    constexpr int Q = kPairs<V>;
    extern __shared__ __align__(16) f32x2 acc[];   // [2][Q][cg / V], g xn and g
    __shared__ float red[16];
    const int r = blockIdx.x / (unsigned)p.G, g = blockIdx.x % (unsigned)p.G, c0 = g * p.cg;
    const float inv = 1.0f / (float)p.cg;
    const int cv = p.cg / V;
    if (LOCAL)
        for (int c = threadIdx.x; c < cv; c += kBlock)
#pragma unroll
            for (int q = 0; q < 2 * Q; ++q) acc[q * cv + c] = 0;
    float *ow = nullptr, *ob = nullptr;
    if (pw) {
        ow = pw + (int64_t)r * p.C + c0;
        ob = pb + (int64_t)r * p.C + c0;
    }
    for (int64_t n = r; n < p.N; n += R) {
        const f32x2 minus = each<V>(-__ldg(p.mean + n * p.G + g)), scale = both(__ldg(p.rstd + n * p.G + g));
        auto load = [&](int c, f32x2 (&xn)[Q], f32x2 (&go)[Q], f32x2 (&ga)[Q], f32x2 (&w)[Q]) {
            f32x2 b[Q];
            widen<T, V>(load_vec<T, V>(p.x + n * p.x_sb + c0 + c), xn);
            widen<T, V>(load_vec<T, V>(p.dout + n * p.o_sb + c0 + c), go);
#pragma unroll
            for (int q = 0; q < Q; ++q) w[q] = each<V>(1.0f), b[q] = 0;
            if (p.w) widen<T, V>(load_vec<T, V>(p.w + c0 + c), w);
            if (p.b) widen<T, V>(load_vec<T, V>(p.b + c0 + c), b);
            if (p.mode == kGate) widen<T, V>(load_vec<T, V>(p.gate + n * p.g_sb + c0 + c), ga);
#pragma unroll
            for (int q = 0; q < Q; ++q) xn[q] = mul2(add2(xn[q], minus), scale);
            through_act2<Q>(p.mode, xn, w, b, go, ga);
        };
        f32x2 s0 = 0, s1 = 0;
#pragma unroll 4
        for (int c = threadIdx.x * V; c < p.cg; c += kBlock * V) {
            f32x2 xn[Q], go[Q], ga[Q], w[Q];
            load(c, xn, go, ga, w);
            if (LOCAL) {
                f32x2* a = acc + c / V;
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    a[q * cv] = fma2(go[q], xn[q], a[q * cv]);
                    a[(Q + q) * cv] = add2(a[(Q + q) * cv], go[q]);
                }
            } else if (ow) {
                f32x2 aw[Q], ab[Q];
#pragma unroll
                for (int q = 0; q < Q; ++q) aw[q] = ab[q] = 0;
                if (n != r) {
                    load_sums<V>(ow + c, aw);
                    load_sums<V>(ob + c, ab);
                }
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    aw[q] = fma2(go[q], xn[q], aw[q]);
                    ab[q] = add2(ab[q], go[q]);
                }
                store_sums<V>(ow + c, aw);
                store_sums<V>(ob + c, ab);
            }
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                go[q] = mul2(go[q], w[q]);
                s0 = add2(s0, go[q]);
                s1 = fma2(go[q], xn[q], s1);
            }
        }
        float sum[2] = {halves(s0), halves(s1)};
        group_sum(sum, kBlock, red);
        const f32x2 m0 = both(-sum[0] * inv), m1 = both(-sum[1] * inv);
#pragma unroll 2
        for (int c = threadIdx.x * V; c < p.cg; c += kBlock * V) {
            f32x2 xn[Q], go[Q], ga[Q], w[Q];
            load(c, xn, go, ga, w);
            if (p.mode == kGate) store_vec(p.dgate + n * p.C + c0 + c, narrow<T, V>(ga));
#pragma unroll
            for (int q = 0; q < Q; ++q) go[q] = mul2(scale, fma2(xn[q], m1, fma2(go[q], w[q], m0)));
            store_vec(p.dx + n * p.C + c0 + c, narrow<T, V>(go));
        }
    }
    if (!LOCAL || !pw) return;
    for (int c = threadIdx.x * V; c < p.cg; c += kBlock * V) {
        f32x2 a[Q], b[Q];
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            a[q] = acc[q * cv + c / V];
            b[q] = acc[(Q + q) * cv + c / V];
        }
        store_sums<V>(ow + c, a);
        store_sums<V>(ob + c, b);
    }
}

// ---- groups in a cluster's shared memory ------------------------------------------------
// A cluster of R blocks takes a slab of whole groups (CS channels) of one row, each block
// its P places, which stay in shared memory: one read of the tensor and one launch. The
// blocks exchange their sums of each group through distributed shared memory and add
// them in rank order. Bound by the latency of its steps (copy, two sums over threads and
// blocks, result), which several blocks an SM hide from one another: 4 x 4096 x 320 f16 in
// 32 groups 19 us, 21 with one block of 512 threads an SM.
constexpr int kSlab = 256;   // threads
struct Slab {
    int CS, slabs, R, P;
};
__host__ __device__ __forceinline__ int slab_floats(int n) { return (n + 3) / 4 * 16; }   // their bytes, whole 16s
// Floats of the segments' sums: at most kSlab segments, or one a channel.
__host__ __device__ __forceinline__ int slab_sums(int cs) { return (cs > kSlab ? cs : kSlab) + 3 & ~3; }

__device__ __forceinline__ float remote(const float* own, int rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_rank(smem_u32(own), rank)) : "memory");
    return v;
}

// A block's part of the layout: channel vector x of row lane y (of by).
template <typename T, int V>
struct SlabPlace {
    int64_t n, c0, s0;
    int cs, pc, cvn, by, x, y;   // channels and places here, vectors a place
    bool on;
    __device__ __forceinline__ SlabPlace(const NormP<T>& p, const Slab& q) {
        const int rank = (int)cluster_rank();
        const unsigned unit = blockIdx.x / (unsigned)q.R;
        n = unit / (unsigned)q.slabs;
        c0 = (int64_t)(unit % (unsigned)q.slabs) * q.CS;
        cs = (int)min((int64_t)q.CS, p.C - c0);
        s0 = (int64_t)rank * q.P;
        pc = (int)max((int64_t)0, min((int64_t)q.P, p.S - s0));
        cvn = cs / V;
        by = kSlab / cvn;
        x = threadIdx.x % cvn;
        y = threadIdx.x / cvn;
        on = y < by;
        segs = max(1, min(by, kSlab / cs));
    }
    // this block's places of a tensor into shared memory [P][cs]
    __device__ __forceinline__ void copy(T* dst, const T* src, int64_t sb, int64_t sp) const {
        if (!on) return;
        const T* from = src + n * sb + s0 * sp + c0 + x * V;
        for (int i = y; i < pc; i += by) {
            if constexpr (V * sizeof(T) >= 8)
                cp_async<V * sizeof(T)>(dst + i * cs + x * V, from + i * sp, V * sizeof(T));
            else
                dst[i * cs + x * V] = load_one(from + i * sp);
        }
    }
    __device__ __forceinline__ void get(const T* tile, int i, f32x2 (&f)[kPairs<V>]) const {
        widen<T, V>(*reinterpret_cast<const Vec<T, V>*>(tile + i * cs + x * V), f);
    }
    // Sums of a value a channel over the block's row lanes, in `segs` segments a channel:
    // sums[ch * segs + i], via red [cs][by].
    int segs;
    __device__ __forceinline__ void channel_sums(const f32x2 (&v)[kPairs<V>], float* red, float* sums) const {
        if (on)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                float h[2];
                unpack2(v[k / 2], h[0], h[1]);
                red[(x * V + k) * by + y] = h[k % 2];
            }
        __syncthreads();
        const int len = (by + segs - 1) / segs;
        for (int i = threadIdx.x; i < cs * segs; i += kSlab) {
            const int c = i / segs, from = (i - c * segs) * len, to = min(by, from + len);
            float a = 0.0f;
            for (int k = from; k < to; ++k) a += red[c * by + k];
            sums[i] = a;
        }
        __syncthreads();
    }
};

// Sums over each group's `items` of a(j, i), into g: the block's own share. A warp a group.
template <typename F>
__device__ __forceinline__ void slab_groups(int groups, int items, float* g, F a) {
    const int lane = threadIdx.x & 31;
    for (int j = threadIdx.x / 32; j < groups; j += kSlab / 32) {
        float s = 0.0f;
        for (int i = lane; i < items; i += 32) s += a(j * items + i);
#pragma unroll
        for (int m = 16; m >= 1; m /= 2) s += __shfl_xor_sync(0xffffffffu, s, m);
        if (lane == 0) g[j] = s;
    }
}
// The blocks' shares of each group added in a fixed order: total[j] = scale * sum. Lane r of
// a warp reads block r's.
__device__ __forceinline__ void cluster_groups(int groups, int R, const float* share, float* total, float scale) {
    const int lane = threadIdx.x & 31;
    for (int j = threadIdx.x / 32; j < groups; j += kSlab / 32) {
        float s = lane < R ? remote(share + j, lane) : 0.0f;
#pragma unroll
        for (int m = 4; m >= 1; m /= 2) s += __shfl_xor_sync(0xffffffffu, s, m);
        if (lane == 0) total[j] = s * scale;
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kSlab, 3) norm_slab(const __grid_constant__ NormP<T> p, const Slab q) {
    constexpr int Q = kPairs<V>;
    extern __shared__ __align__(16) unsigned char smem[];
    float* red = reinterpret_cast<float*>(smem);        // [kSlab V]
    float *sums = red + kSlab * V, *share = sums + slab_sums(q.CS), *own = share + 2 * q.CS;   // 2 a group; a group
    T* tile = reinterpret_cast<T*>(smem + slab_floats(kSlab * V + slab_sums(q.CS) + 3 * q.CS));
    const SlabPlace<T, V> at(p, q);
    const int groups = at.cs / p.cg;
    at.copy(tile, p.x, p.x_sb, p.x_sp);
    cp_commit();
    f32x2 w[Q], b[Q];
#pragma unroll
    for (int k = 0; k < Q; ++k) w[k] = each<V>(1.0f), b[k] = 0;
    if (at.on && p.w) widen<T, V>(load_vec<T, V>(p.w + at.c0 + at.x * V), w);
    if (at.on && p.b) widen<T, V>(load_vec<T, V>(p.b + at.c0 + at.x * V), b);
    const float inv = 1.0f / ((float)p.cg * (float)p.S);
    cp_wait();
    // own places only: a thread reads what it copied
    f32x2 mean[Q], rstd[Q], s[Q];
    int g0[Q], g1[Q];   // the channels' groups in the slab
#pragma unroll
    for (int k = 0; k < Q; ++k) {
        const int c = at.on ? at.x * V + 2 * k : 0;
        s[k] = 0;
        g0[k] = c / p.cg;
        g1[k] = (c + (V > 1)) / p.cg;
    }
    if (at.on)
#pragma unroll 4
        for (int i = at.y; i < at.pc; i += at.by) {
            f32x2 f[Q];
            at.get(tile, i, f);
#pragma unroll
            for (int k = 0; k < Q; ++k) s[k] = add2(s[k], f[k]);
        }
    // (sum over all places of each group) inv, a channel's pair
    auto over_group = [&](float* to, f32x2 (&out)[Q]) {
        at.channel_sums(s, red, sums);
        slab_groups(groups, p.cg * at.segs, to, [&](int i) { return sums[i]; });
        __syncthreads();
        cluster_sync();
        cluster_groups(groups, q.R, to, own, inv);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < Q; ++k) out[k] = pack2(own[g0[k]], V == 1 ? 0.0f : own[g1[k]]);
    };
    over_group(share, mean);
    float keep = 0.0f;
    if (threadIdx.x < groups) keep = own[threadIdx.x];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < Q; ++k) s[k] = 0, mean[k] = mul2(mean[k], both(-1.0f));
    if (at.on)
#pragma unroll 4
        for (int i = at.y; i < at.pc; i += at.by) {
            f32x2 f[Q];
            at.get(tile, i, f);
#pragma unroll
            for (int k = 0; k < Q; ++k) {
                f[k] = add2(f[k], mean[k]);
                s[k] = fma2(f[k], f[k], s[k]);
            }
        }
    over_group(share + q.CS, rstd);
    if (cluster_rank() == 0 && p.mean && threadIdx.x < groups) {
        const int64_t g = at.n * p.G + at.c0 / p.cg + threadIdx.x;
        p.mean[g] = keep;
        p.rstd[g] = rsqrtf(own[threadIdx.x] + p.eps);
    }
#pragma unroll
    for (int k = 0; k < Q; ++k) {
        float lo, hi;
        unpack2(rstd[k], lo, hi);
        rstd[k] = pack2(rsqrtf(lo + p.eps), rsqrtf(hi + p.eps));
    }
    if (at.on) {
        const int64_t c = at.c0 + at.x * V;
        const T* gate = p.mode == kGate ? p.gate + at.n * p.g_sb + at.s0 * p.g_sp + c : nullptr;
        T* out = p.out + (at.n * p.S + at.s0) * p.C + c;
#pragma unroll 4
        for (int i = at.y; i < at.pc; i += at.by) {
            f32x2 f[Q], ga[Q];
            if (gate) widen<T, V>(load_vec<T, V>(gate + i * p.g_sp), ga);
            at.get(tile, i, f);
#pragma unroll
            for (int k = 0; k < Q; ++k) {
                f[k] = fma2(mul2(add2(f[k], mean[k]), rstd[k]), w[k], b[k]);
                if (p.mode == kSilu) f[k] = mul2(f[k], sigmoid2(f[k]));
                if (gate) f[k] = mul2(f[k], mul2(ga[k], sigmoid2(ga[k])));
            }
            store_vec(out + (int64_t)i * p.C, narrow<T, V>(f));
        }
    }
    cluster_sync();   // the others may still read this block's sums
}

// Backward: x and dout stay in shared memory, the gate is read twice. pw, pb [N R][C]: a
// block's share of the sums of g xn and g. The map above: 25 us.
template <typename T, int V>
__global__ void __launch_bounds__(kSlab, 2) norm_slab_bwd(const __grid_constant__ NormP<T> p, const Slab q, float* pw,
                                                           float* pb) {
    constexpr int Q = kPairs<V>;
    extern __shared__ __align__(16) unsigned char smem[];
    float* red = reinterpret_cast<float*>(smem);        // [kSlab V]
    float *sw = red + kSlab * V, *sb = sw + slab_sums(q.CS), *share = sb + slab_sums(q.CS), *own = share + 2 * q.CS;
    T* tx = reinterpret_cast<T*>(smem + slab_floats(kSlab * V + 2 * slab_sums(q.CS) + 4 * q.CS));
    T* to = tx + (int64_t)q.P * q.CS;
    const SlabPlace<T, V> at(p, q);
    const int groups = at.cs / p.cg;
    at.copy(tx, p.x, p.x_sb, p.x_sp);
    at.copy(to, p.dout, p.o_sb, p.o_sp);
    cp_commit();
    const int64_t c = at.c0 + at.x * V;
    f32x2 w[Q], b[Q], mean[Q], rstd[Q], a0[Q], a1[Q];
#pragma unroll
    for (int k = 0; k < Q; ++k) w[k] = each<V>(1.0f), b[k] = a0[k] = a1[k] = mean[k] = rstd[k] = 0;
    if (at.on) {
        if (p.w) widen<T, V>(load_vec<T, V>(p.w + c), w);
        if (p.b) widen<T, V>(load_vec<T, V>(p.b + c), b);
#pragma unroll
        for (int k = 0; k < Q; ++k) {
            const int64_t g0 = at.n * p.G + (int)(c + 2 * k) / p.cg, g1 = at.n * p.G + (int)(c + 2 * k + (V > 1)) / p.cg;
            mean[k] = pack2(-__ldg(p.mean + g0), V == 1 ? 0.0f : -__ldg(p.mean + g1));
            rstd[k] = pack2(__ldg(p.rstd + g0), V == 1 ? 0.0f : __ldg(p.rstd + g1));
        }
    }
    const T* gate = p.mode == kGate ? p.gate + at.n * p.g_sb + at.s0 * p.g_sp + c : nullptr;
    auto load = [&](int i, f32x2 (&xn)[Q], f32x2 (&go)[Q], f32x2 (&ga)[Q]) {
        if (gate) widen<T, V>(load_vec<T, V>(gate + i * p.g_sp), ga);
        at.get(tx, i, xn);
        at.get(to, i, go);
#pragma unroll
        for (int k = 0; k < Q; ++k) xn[k] = mul2(add2(xn[k], mean[k]), rstd[k]);
        through_act2<Q>(p.mode, xn, w, b, go, ga);
    };
    cp_wait();
    if (at.on)
#pragma unroll 2
        for (int i = at.y; i < at.pc; i += at.by) {
            f32x2 xn[Q], go[Q], ga[Q];
            load(i, xn, go, ga);
#pragma unroll
            for (int k = 0; k < Q; ++k) {
                a0[k] = add2(a0[k], go[k]);
                a1[k] = fma2(go[k], xn[k], a1[k]);
            }
        }
    at.channel_sums(a1, red, sw);
    at.channel_sums(a0, red, sb);
    if (pw)
        for (int i = threadIdx.x; i < at.cs; i += kSlab) {
            const int64_t row = at.n * q.R + cluster_rank();
            float a = 0.0f, b = 0.0f;
            for (int k = 0; k < at.segs; ++k) a += sw[i * at.segs + k], b += sb[i * at.segs + k];
            pw[row * p.C + at.c0 + i] = a;
            pb[row * p.C + at.c0 + i] = b;
        }
    auto weight = [&](int i) { return p.w ? to_float(load_one(p.w + at.c0 + i / at.segs)) : 1.0f; };
    slab_groups(groups, p.cg * at.segs, share, [&](int i) { return weight(i) * sb[i]; });
    slab_groups(groups, p.cg * at.segs, share + q.CS, [&](int i) { return weight(i) * sw[i]; });
    __syncthreads();
    cluster_sync();
    const float inv = 1.0f / ((float)p.cg * (float)p.S);
    cluster_groups(groups, q.R, share, own, -inv);
    cluster_groups(groups, q.R, share + q.CS, own + q.CS, -inv);
    __syncthreads();
    if (at.on) {
        f32x2 m0[Q], m1[Q];
#pragma unroll
        for (int k = 0; k < Q; ++k) {
            const int i = at.x * V + 2 * k, g0 = i / p.cg, g1 = V == 1 ? g0 : (i + 1) / p.cg;
            m0[k] = pack2(own[g0], own[g1]);
            m1[k] = pack2(own[q.CS + g0], own[q.CS + g1]);
        }
#pragma unroll 2
        for (int i = at.y; i < at.pc; i += at.by) {
            f32x2 xn[Q], go[Q], ga[Q];
            load(i, xn, go, ga);
            const int64_t o = (at.n * p.S + at.s0 + i) * p.C + c;
            if (gate) store_vec(p.dgate + o, narrow<T, V>(ga));
#pragma unroll
            for (int k = 0; k < Q; ++k) go[k] = mul2(rstd[k], fma2(xn[k], m1[k], fma2(go[k], w[k], m0[k])));
            store_vec(p.dx + o, narrow<T, V>(go));
        }
    }
    cluster_sync();   // the others may still read this block's sums
}

// ---- larger groups ------------------------------------------------------------------
// 16 x 4096 x 320 f16 with silu in 32 groups: 37 us forward, 97 backward, three launches
// each; memory would take 13 and 19 if L2 gave the second read for nothing.
struct Chunks {
    int bx;              // channel vectors a block
    int64_t chunks, rows;   // chunks of `rows` places
};

// (count, mean, sum of squared deviations) joined: Chan, Golub, LeVeque, "Updating
// formulae and a pairwise algorithm for computing sample variances" (1979).
struct Moments {
    float n, mean, m2;
    __device__ __forceinline__ void join(float bn, float bmean, float bm2) {
        if (bn == 0.0f) return;
        const float t = n + bn, d = bmean - mean, f = bn / t;
        mean = fmaf(d, f, mean);
        m2 += bm2 + (d * n) * (d * f);   // 0 from n = 0, and no overflow that the sum does not have
        n = t;
    }
};

// Per-channel moments of a chunk's places: part [n][chunk][2][C] (mean, m2).
template <typename T, int V>
__global__ void __launch_bounds__(kBlock) norm_stats(const __grid_constant__ NormP<T> p, Chunks q, float* part) {
    __shared__ float red[3][V][kBlock];
    const int by = kBlock / q.bx, x = threadIdx.x % q.bx, y = threadIdx.x / q.bx;
    const int64_t n = blockIdx.x / (unsigned)q.chunks, chunk = blockIdx.x % (unsigned)q.chunks;
    const int64_t c = ((int64_t)blockIdx.y * q.bx + x) * V;
    const int64_t s0 = chunk * q.rows, s1 = min(p.S, s0 + q.rows);
    float s[V], ss[V], pv[V];
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = ss[v] = pv[v] = 0.0f;
    float count = 0.0f;
    if (c < p.C && s0 + y < s1) {
        const T* xp = p.x + n * p.x_sb + c;
        unpack(load_vec<T, V>(xp + (s0 + y) * p.x_sp), pv);   // the shift
#pragma unroll 4
        for (int64_t i = s0 + y; i < s1; i += by) {
            float f[V];
            unpack(load_vec<T, V>(xp + i * p.x_sp), f);
            count += 1.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float d = f[v] - pv[v];
                s[v] += d;
                ss[v] = fmaf(d, d, ss[v]);
            }
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const float m = count > 0.0f ? s[v] / count : 0.0f;
        red[0][v][threadIdx.x] = count;
        red[1][v][threadIdx.x] = pv[v] + m;
        red[2][v][threadIdx.x] = fmaf(-m, s[v], ss[v]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < q.bx * V; i += kBlock) {
        const int xi = i % q.bx, v = i / q.bx;
        const int64_t ci = ((int64_t)blockIdx.y * q.bx + xi) * V + v;
        if (ci >= p.C) continue;
        Moments m{0.0f, 0.0f, 0.0f};
        for (int r = 0; r < by; ++r) {
            const int k = r * q.bx + xi;
            m.join(red[0][v][k], red[1][v][k], red[2][v][k]);
        }
        part[((n * q.chunks + chunk) * 2) * p.C + ci] = m.mean;
        part[((n * q.chunks + chunk) * 2 + 1) * p.C + ci] = m.m2;
    }
}

// mean and rstd of one (row, group) from its channels' moments.
__global__ void __launch_bounds__(kBlock) norm_join(const float* part, int64_t S, int64_t C, int G, int cg, Chunks q,
                                                    float eps, float* mean, float* rstd) {
    __shared__ float red[3][kBlock];
    const int64_t n = blockIdx.x / G;
    const int g = (int)(blockIdx.x - n * G);
    Moments m{0.0f, 0.0f, 0.0f};
    const int64_t items = q.chunks * cg;
    for (int i0 = threadIdx.x; i0 < (int)items; i0 += 8 * kBlock) {   // eight loads on their way
        float cnt[8], mean8[8], m28[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = i0 + k * kBlock, chunk = i / cg, c = g * cg + (i - chunk * cg);
            cnt[k] = 0.0f;
            if (i >= (int)items) continue;
            const float* b = part + (n * q.chunks + chunk) * 2 * C + c;
            cnt[k] = (float)(min(S, (chunk + 1) * q.rows) - chunk * q.rows);
            mean8[k] = __ldg(b);
            m28[k] = __ldg(b + C);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (cnt[k] > 0.0f) m.join(cnt[k], mean8[k], m28[k]);
    }
    for (int h = kBlock / 2; h >= 1; h /= 2) {
        red[0][threadIdx.x] = m.n;
        red[1][threadIdx.x] = m.mean;
        red[2][threadIdx.x] = m.m2;
        __syncthreads();
        if (threadIdx.x < h) m.join(red[0][threadIdx.x + h], red[1][threadIdx.x + h], red[2][threadIdx.x + h]);
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        mean[blockIdx.x] = m.mean;
        rstd[blockIdx.x] = rsqrtf(m.m2 / m.n + eps);
    }
}

template <typename T, int V>
struct Channel {
    static constexpr int Q = kPairs<V>;
    f32x2 w[Q], b[Q], minus[Q], rstd[Q];   // minus the mean
    __device__ __forceinline__ Channel(const NormP<T>& p, int64_t n, int64_t c) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const int64_t g0 = n * p.G + (int)(c + 2 * q) / p.cg, g1 = n * p.G + (int)(c + 2 * q + (V > 1)) / p.cg;
            w[q] = each<V>(1.0f);
            b[q] = 0;
            minus[q] = pack2(-__ldg(p.mean + g0), V == 1 ? 0.0f : -__ldg(p.mean + g1));
            rstd[q] = pack2(__ldg(p.rstd + g0), __ldg(p.rstd + g1));
        }
        if (p.w) widen<T, V>(load_vec<T, V>(p.w + c), w);
        if (p.b) widen<T, V>(load_vec<T, V>(p.b + c), b);
    }
    __device__ __forceinline__ f32x2 xn(int q, f32x2 x) const { return mul2(add2(x, minus[q]), rstd[q]); }
};

template <typename T, int V>
__global__ void __launch_bounds__(kBlock, 4) norm_apply(const __grid_constant__ NormP<T> p, Chunks q) {
    constexpr int Q = kPairs<V>;
    const int by = kBlock / q.bx, x = threadIdx.x % q.bx, y = threadIdx.x / q.bx;
    const int64_t n = blockIdx.x / (unsigned)q.chunks, chunk = blockIdx.x % (unsigned)q.chunks;
    const int64_t c = ((int64_t)blockIdx.y * q.bx + x) * V;
    if (c >= p.C) return;
    const int64_t s0 = chunk * q.rows, s1 = min(p.S, s0 + q.rows);
    const Channel<T, V> ch(p, n, c);
#pragma unroll 4
    for (int64_t i = s0 + y; i < s1; i += by) {
        f32x2 f[Q], ga[Q];
        widen<T, V>(load_vec<T, V>(p.x + n * p.x_sb + i * p.x_sp + c), f);
        if (p.mode == kGate) widen<T, V>(load_vec<T, V>(p.gate + n * p.g_sb + i * p.g_sp + c), ga);
#pragma unroll
        for (int k = 0; k < Q; ++k) {
            f[k] = fma2(ch.xn(k, f[k]), ch.w[k], ch.b[k]);
            if (p.mode == kSilu) f[k] = mul2(f[k], sigmoid2(f[k]));
            if (p.mode == kGate) f[k] = mul2(f[k], mul2(ga[k], sigmoid2(ga[k])));
        }
        store_vec(p.out + (n * p.S + i) * p.C + c, narrow<T, V>(f));
    }
}

// Per-channel sums of g xn and g over a chunk's places: part [n][chunk][2][C].
template <typename T, int V>
__global__ void __launch_bounds__(kBlock, 2) norm_sums(const __grid_constant__ NormP<T> p, Chunks q, float* part) {
    constexpr int Q = kPairs<V>;
    __shared__ float red[2][V][kBlock];
    const int by = kBlock / q.bx, x = threadIdx.x % q.bx, y = threadIdx.x / q.bx;
    const int64_t n = blockIdx.x / (unsigned)q.chunks, chunk = blockIdx.x % (unsigned)q.chunks;
    const int64_t c = ((int64_t)blockIdx.y * q.bx + x) * V;
    const int64_t s0 = chunk * q.rows, s1 = min(p.S, s0 + q.rows);
    f32x2 aw[Q], ab[Q];
#pragma unroll
    for (int k = 0; k < Q; ++k) aw[k] = ab[k] = 0;
    if (c < p.C) {
        const Channel<T, V> ch(p, n, c);
#pragma unroll 4
        for (int64_t i = s0 + y; i < s1; i += by) {
            f32x2 xn[Q], go[Q], ga[Q];
            widen<T, V>(load_vec<T, V>(p.x + n * p.x_sb + i * p.x_sp + c), xn);
            widen<T, V>(load_vec<T, V>(p.dout + n * p.o_sb + i * p.o_sp + c), go);
            if (p.mode == kGate) widen<T, V>(load_vec<T, V>(p.gate + n * p.g_sb + i * p.g_sp + c), ga);
#pragma unroll
            for (int k = 0; k < Q; ++k) xn[k] = ch.xn(k, xn[k]);
            through_act2<Q>(p.mode, xn, ch.w, ch.b, go, ga);
#pragma unroll
            for (int k = 0; k < Q; ++k) {
                aw[k] = fma2(go[k], xn[k], aw[k]);
                ab[k] = add2(ab[k], go[k]);
            }
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float a[2], b[2];
        unpack2(aw[v / 2], a[0], a[1]);
        unpack2(ab[v / 2], b[0], b[1]);
        red[0][v][threadIdx.x] = a[v % 2];
        red[1][v][threadIdx.x] = b[v % 2];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < q.bx * V * 2; i += kBlock) {
        const int xi = i % q.bx, v = i / q.bx % V, which = i / (q.bx * V);
        const int64_t ci = ((int64_t)blockIdx.y * q.bx + xi) * V + v;
        if (ci >= p.C) continue;
        float a = 0.0f;
        for (int r = 0; r < by; ++r) a += red[which][v][r * q.bx + xi];
        part[((n * q.chunks + chunk) * 2 + which) * p.C + ci] = a;
    }
}

// Chunks added up per channel (sums [n][C] of g xn and g), then per group: mean of
// g w and of g w xn (gm [n][G][2]).
template <typename T>
__global__ void __launch_bounds__(kBlock) norm_sums_join(const __grid_constant__ NormP<T> p, Chunks q,
                                                         const float* part, float* sw, float* sb, float* gm) {
    __shared__ float red[2][kBlock];
    const int64_t n = blockIdx.x / p.G;
    const int g = (int)(blockIdx.x - n * p.G);
    float s0 = 0.0f, s1 = 0.0f;
    for (int i = threadIdx.x; i < p.cg; i += kBlock) {
        const int64_t c = (int64_t)g * p.cg + i;
        const float* b = part + n * q.chunks * 2 * p.C + c;
        float aw = 0.0f, ab = 0.0f;
#pragma unroll 8
        for (int64_t k = 0; k < q.chunks; ++k) {
            aw += __ldg(b + 2 * k * p.C);
            ab += __ldg(b + (2 * k + 1) * p.C);
        }
        sw[n * p.C + c] = aw;
        sb[n * p.C + c] = ab;
        const float w = p.w ? to_float(load_one(p.w + c)) : 1.0f;
        s0 = fmaf(w, ab, s0);
        s1 = fmaf(w, aw, s1);
    }
    for (int h = kBlock / 2; h >= 1; h /= 2) {
        red[0][threadIdx.x] = s0;
        red[1][threadIdx.x] = s1;
        __syncthreads();
        if (threadIdx.x < h) s0 += red[0][threadIdx.x + h], s1 += red[1][threadIdx.x + h];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const float inv = 1.0f / ((float)p.cg * (float)p.S);
        gm[2 * blockIdx.x] = s0 * inv;
        gm[2 * blockIdx.x + 1] = s1 * inv;
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kBlock, 2) norm_apply_bwd(const __grid_constant__ NormP<T> p, Chunks q,
                                                            const float* gm) {
    constexpr int Q = kPairs<V>;
    const int by = kBlock / q.bx, x = threadIdx.x % q.bx, y = threadIdx.x / q.bx;
    const int64_t n = blockIdx.x / (unsigned)q.chunks, chunk = blockIdx.x % (unsigned)q.chunks;
    const int64_t c = ((int64_t)blockIdx.y * q.bx + x) * V;
    if (c >= p.C) return;
    const int64_t s0 = chunk * q.rows, s1 = min(p.S, s0 + q.rows);
    const Channel<T, V> ch(p, n, c);
    f32x2 m0[Q], m1[Q];
#pragma unroll
    for (int k = 0; k < Q; ++k) {
        const float* a = gm + 2 * (n * p.G + (int)(c + 2 * k) / p.cg);
        const float* b = gm + 2 * (n * p.G + (int)(c + 2 * k + (V > 1)) / p.cg);
        m0[k] = pack2(-__ldg(a), -__ldg(b));
        m1[k] = pack2(-__ldg(a + 1), -__ldg(b + 1));
    }
#pragma unroll 4
    for (int64_t i = s0 + y; i < s1; i += by) {
        f32x2 xn[Q], go[Q], ga[Q];
        const int64_t o = (n * p.S + i) * p.C + c;
        widen<T, V>(load_vec<T, V>(p.x + n * p.x_sb + i * p.x_sp + c), xn);
        widen<T, V>(load_vec<T, V>(p.dout + n * p.o_sb + i * p.o_sp + c), go);
        if (p.mode == kGate) widen<T, V>(load_vec<T, V>(p.gate + n * p.g_sb + i * p.g_sp + c), ga);
#pragma unroll
        for (int k = 0; k < Q; ++k) xn[k] = ch.xn(k, xn[k]);
        through_act2<Q>(p.mode, xn, ch.w, ch.b, go, ga);
        if (p.mode == kGate) store_vec(p.dgate + o, narrow<T, V>(ga));
#pragma unroll
        for (int k = 0; k < Q; ++k) go[k] = mul2(ch.rstd[k], fma2(xn[k], m1[k], fma2(go[k], ch.w[k], m0[k])));
        store_vec(p.dx + o, narrow<T, V>(go));
    }
}

// ---- host ---------------------------------------------------------------------------
int check_norm(const pe_norm_args* a) {
    if (!a || a->dtype < PE_F32 || a->dtype > PE_BF16 || a->batch < 0 || a->places < 0 || a->channels < 1 ||
        a->groups < 1 || a->channels % a->groups || !(a->eps >= 0.0) || (a->silu && a->gate))
        return PE_ERR_INVALID;
    if (a->channels > (1 << 24) || a->places > (1ll << 40)) return PE_ERR_UNSUPPORTED;
    if (a->batch && a->places && !a->x) return PE_ERR_INVALID;
    return PE_OK;
}

// Nothing to normalise, and nothing that plan_of could divide into rows and chunks.
bool empty(const pe_norm_args* a) { return a->batch == 0 || a->places == 0; }

// Elements a load: 16 bytes where all rows start on that boundary, else one (8000 gated
// rows of 8 groups, 4096 and 4008 bf16 channels, groups of 501: 43 and 197 us forward).
int vec_of(const pe_norm_args* a, std::initializer_list<const void*> more, std::initializer_list<int64_t> strides) {
    const int v = a->dtype == PE_F32 ? 4 : 8;
    if (a->channels % v) return 1;
    for (const void* q : {a->x, a->weight, a->bias, a->gate, (const void*)a->out})
        if ((uintptr_t)q % 16) return 1;
    for (const void* q : more)
        if ((uintptr_t)q % 16) return 1;
    for (int64_t s : {a->x_sb, a->x_sp, a->gate ? a->gate_sb : 0, a->gate ? a->gate_sp : 0})
        if (s % v) return 1;
    for (int64_t s : strides)
        if (s % v) return 1;
    return v;
}

int widest(const pe_norm_args* a) {
    const int v = a->dtype == PE_F32 ? 4 : 8;
    return a->channels % v ? 1 : v;
}

struct Plan {
    int v;            // elements a load
    int lanes, k;     // groups in registers: lanes a group, loads a lane; lanes 0: too large for that
    int64_t R;        // in registers: rows at work, a lane takes every R-th
    bool wide, local; // a block a group of one place; its sums in shared memory
    Slab slab;        // in a cluster's shared memory: R > 0
    Chunks q;
};

int64_t slab_smem(int64_t cs, int64_t P, int v, int64_t es, bool grad) {
    return slab_floats(kSlab * v + (grad ? 2 : 1) * slab_sums((int)cs) + (grad ? 4 : 3) * (int)cs) + (grad ? 2 : 1) * ceil_div(P * cs * es, 16) * 16;
}

// The slab of a group that is too large for registers: whole groups and whole loads, 64
// bytes a place or more where there are so many channels; blocks enough to hold it, three
// an SM forward and two backward where that still leaves a thread two loads. R 0: too
// large, or more blocks than the SMs hold at once. Clusters against chunks, f16 with silu
// in 32 groups, forward (with backward): 4 x 4096 x 320 19 and 27 us (45 and 58); beyond one
// wave 64 x 256 x 1280 64 and 44 (177 and 144), 16 x 4096 x 320 63 and 37 (154 and 134).
Slab slab_of(const pe_norm_args* a, int v, bool grad) {
    Slab s{0, 0, 0, 0};
    const int64_t cg = a->channels / a->groups, es = a->dtype == PE_F32 ? 4 : 2;
    int64_t base = cg;
    while (base % v) base += cg;
    int64_t cs = base;
    while (cs * es < 64 && cs + base <= a->channels) cs += base;
    if (cs / v > kSlab || a->places > (1 << 24)) return s;
    const int64_t slabs = ceil_div(a->channels, cs);
    for (int r = 1; r <= 8; r *= 2) {
        const int64_t P = ceil_div(a->places, r);
        if (slab_smem(cs, P, v, es, grad) > 200 * 1024) continue;
        if (r < 8 && slab_smem(cs, P, v, es, grad) > (grad ? 100 : 64) * 1024 && P * (cs / v) > 2 * kSlab) continue;
        const int64_t resident = min((int64_t)(grad ? 2 : 3), 220 * 1024 / slab_smem(cs, P, v, es, grad));
        if (a->batch * slabs * r > num_sms() * resident) return s;
        s.CS = (int)cs; s.slabs = (int)slabs; s.R = r; s.P = (int)P;
        return s;
    }
    return s;
}

Plan plan_of(const pe_norm_args* a, int vec, bool grad) {
    Plan p{};
    const int64_t cg = a->channels / a->groups;
    const int vr = cg % vec == 0 ? vec : 1;      // in registers a load stays within its group
    const int64_t items = a->places <= 1024 ? cg / vr * a->places : 1 << 20;
    // the backward pass keeps sums a channel in registers, where an item is a channel vector.
    // Loads a lane at most: by the registers they need, and where the block a group further
    // down is not faster. Gated bf16 rows in registers against that: two loads, 4096 x 4096,
    // 27 and 31 us (79 and 164 with the backward pass); four loads, 4096 x 8192, 62 and 49.
    // Element by element a block a group is the faster one.
    const int most = vr == 1 ? 8 : grad || a->places == 1 ? 2 : 4;
    if (items <= (vr == 1 ? 32 * most : most * kBlock) && (!grad || a->places == 1)) {
        p.v = vr;
        if (items <= 32 * most) {
            p.lanes = 1;
            while (p.lanes < 32 && p.lanes < items) p.lanes *= 2;
        } else {
            p.lanes = kBlock;
        }
        const int64_t k = ceil_div(items, p.lanes);
        p.k = k <= 1 ? 1 : k <= 2 ? 2 : k <= 4 ? 4 : 8;
        // rows of groups at work: one wave of blocks; each then takes further rows, so that
        // its filter and its sums weigh less
        const int64_t want = (int64_t)num_sms() * reg_blocks(p.k, p.v, grad) * kBlock / p.lanes / a->groups;
        p.R = a->batch < want ? a->batch : want < 1 ? 1 : want;
        return p;
    }
    // one place a row: a block a group while its sums fit shared memory
    const int64_t smem = cg / vr * 2 * ((vr + 1) / 2) * 8;
    if (a->places == 1) {
        p.v = vr;
        p.wide = true;
        p.local = smem <= 200 * 1024;
        const int64_t resident = !p.local ? 2 : smem > 100 * 1024 ? 1 : smem > 50 * 1024 ? 2 : 4;
        const int64_t want = ceil_div((int64_t)num_sms() * resident, a->groups);
        p.R = a->batch < want ? a->batch : want;
        return p;
    }
    p.v = vec;
    p.slab = slab_of(a, vec, grad);
    if (p.slab.R) return p;
    const int64_t cv = a->channels / vec;
    p.q.bx = 32;
    while (p.q.bx > 1 && ceil_div(cv, p.q.bx) * p.q.bx * 8 > cv * 9) p.q.bx /= 2;
    // chunks a row: whole waves of the blocks that the SMs hold, where a block costs its
    // places and about six more (its filter, its statistics, the sums over its lanes). The
    // fewest chunks that give eight blocks an SM instead: 2 x 10000 x 1024 gated 77 us, so 53
    const int64_t blocks = max((int64_t)1, ceil_div(cv, p.q.bx) * a->batch), by = kBlock / p.q.bx;
    const int64_t slots = (int64_t)num_sms() * (grad ? 2 : 4);
    int64_t best = 0;
    for (int64_t w = 1; w <= 8; ++w) {
        const int64_t rows = ceil_div(ceil_div(a->places, max((int64_t)1, w * slots / blocks)), by) * by;
        const int64_t cost = ceil_div(blocks * ceil_div(a->places, rows), slots) * (rows / by + 6);
        if (w == 1 || cost < best) {
            best = cost;
            p.q.rows = rows;
        }
    }
    p.q.chunks = ceil_div(a->places, p.q.rows);
    return p;
}

template <typename T>
NormP<T> norm_params(const pe_norm_args* a) {
    NormP<T> p{};
    p.N = a->batch; p.S = a->places; p.C = a->channels;
    p.G = (int)a->groups; p.cg = (int)(a->channels / a->groups);
    p.mode = a->gate ? kGate : a->silu ? kSilu : kPlain;
    p.eps = (float)a->eps;
    p.x = (const T*)a->x; p.w = (const T*)a->weight; p.b = (const T*)a->bias; p.gate = (const T*)a->gate;
    p.x_sb = a->x_sb; p.x_sp = a->x_sp; p.g_sb = a->gate_sb; p.g_sp = a->gate_sp;
    p.out = (T*)a->out; p.mean = a->mean; p.rstd = a->rstd;
    return p;
}

int launched() {
    count_launch();
    return cudaGetLastError() == cudaSuccess ? PE_OK : PE_ERR_CUDA;
}

int64_t stats_floats(const pe_norm_args* a, const Plan& pl) {
    return pl.lanes || pl.wide || pl.slab.R ? 0 : a->batch * (pl.q.chunks * 2 * a->channels + 2 * a->groups);
}

// Shared memory of the register kernels' queues: four rows of k loads a lane and stream.
template <typename T, int V>
int queue_bytes(int k, int streams) {
    return 4 * k * streams * kBlock * kSlotBytes<T, V>;
}
template <typename K, typename... A>
int launch_reg(K kernel, int64_t blocks, int smem, cudaStream_t s, A... args) {
    if (smem > 40 * 1024 &&   // the kernels have some static shared memory too
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return PE_ERR_CUDA;
    kernel<<<(unsigned)blocks, kBlock, smem, s>>>(args...);
    return launched();
}

template <typename K, typename... A>
int launch_slab(K kernel, int64_t rows, const Slab& q, int64_t smem, cudaStream_t s, A... args) {
    const int64_t blocks = rows * q.slabs * q.R;
    if (blocks > 0x7fffffffll) return PE_ERR_UNSUPPORTED;
    if (smem > 48 * 1024 &&
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return PE_ERR_CUDA;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = q.R;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kSlab);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) return PE_ERR_CUDA;
    count_launch();
    return PE_OK;
}

template <typename T, int V>
int norm_run(const pe_norm_args* a, const Plan& pl, cudaStream_t s) {
    NormP<T> p = norm_params<T>(a);
    const int64_t units = p.N * p.G;
    if (pl.lanes) {
        const int64_t blocks = ceil_div(pl.R * p.G * pl.lanes, kBlock);
        if (blocks > 0x7fffffll) return PE_ERR_UNSUPPORTED;
        const int streams = p.mode == kGate ? 2 : 1;
        if (pl.k == 1) return launch_reg(norm_reg<T, V, 1>, blocks, queue_bytes<T, V>(1, streams), s, p, pl.lanes, (int)pl.R);
        if (pl.k == 2) return launch_reg(norm_reg<T, V, 2>, blocks, queue_bytes<T, V>(2, streams), s, p, pl.lanes, (int)pl.R);
        if constexpr (V == 1)
            if (pl.k == 8)
                return launch_reg(norm_reg<T, V, 8>, blocks, queue_bytes<T, V>(8, streams), s, p, pl.lanes, (int)pl.R);
        return launch_reg(norm_reg<T, V, 4>, blocks, queue_bytes<T, V>(4, streams), s, p, pl.lanes, (int)pl.R);
    }
    if (pl.wide) {
        if (units > 0x7fffffffll) return PE_ERR_UNSUPPORTED;
        norm_wide<T, V><<<(unsigned)units, kBlock, 0, s>>>(p);
        return launched();
    }
    if (pl.slab.R)
        return launch_slab(norm_slab<T, V>, p.N, pl.slab, slab_smem(pl.slab.CS, pl.slab.P, V, sizeof(T), false), s, p,
                           pl.slab);
    float* part = (float*)a->ws;
    if (!p.mean) {
        p.mean = part + p.N * pl.q.chunks * 2 * p.C;
        p.rstd = p.mean + units;
    }
    const int64_t cb = ceil_div(p.C / V, pl.q.bx);
    if (p.N * pl.q.chunks > 0x7fffffffll || cb > 65535 || units > 0x7fffffffll) return PE_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)(p.N * pl.q.chunks), (unsigned)cb);
    norm_stats<T, V><<<grid, kBlock, 0, s>>>(p, pl.q, part);
    if (int rc = launched()) return rc;
    norm_join<<<(unsigned)units, kBlock, 0, s>>>(part, p.S, p.C, p.G, p.cg, pl.q, p.eps, p.mean, p.rstd);
    if (int rc = launched()) return rc;
    norm_apply<T, V><<<grid, kBlock, 0, s>>>(p, pl.q);
    return launched();
}

int64_t grad_floats(const pe_norm_args* a, const Plan& pl) {
    if (pl.lanes || pl.wide) return 2 * pl.R * a->channels;
    if (pl.slab.R) return 2 * a->batch * pl.slab.R * a->channels;
    return a->batch * (pl.q.chunks * 2 * a->channels + 2 * a->channels + 2 * a->groups);
}

template <typename T, int V>
int norm_grad_run(const pe_norm_grad_args* ga, const Plan& pl, cudaStream_t s) {
    const pe_norm_args* a = &ga->fwd;
    NormP<T> p = norm_params<T>(a);
    p.dout = (const T*)ga->dout; p.o_sb = ga->dout_sb; p.o_sp = ga->dout_sp;
    p.dx = (T*)ga->dx; p.dgate = (T*)ga->dgate;
    float* ws = (float*)ga->ws;
    float *sw, *sb;
    int64_t rows;
    if (pl.lanes) {
        const int64_t blocks = ceil_div(pl.R * p.G * pl.lanes, kBlock);
        if (blocks > 0x7fffffll) return PE_ERR_UNSUPPORTED;
        rows = pl.R;
        const bool sums = ga->dweight || ga->dbias;
        sw = ws;
        sb = ws + rows * p.C;
        float* pw = sums ? sw : nullptr;
        const int streams = p.mode == kGate ? 3 : 2;
        auto go = [&](auto kernel, int k) {
            return launch_reg(kernel, blocks, queue_bytes<T, V>(k, streams), s, p, pl.lanes, (int)pl.R, pw, sb);
        };
        int rc = PE_ERR_INVALID;
        if (pl.k == 1) rc = go(norm_reg_bwd<T, V, 1>, 1);
        if (pl.k == 2) rc = go(norm_reg_bwd<T, V, 2>, 2);
        if constexpr (V == 1) {
            if (pl.k == 4) rc = go(norm_reg_bwd<T, V, 4>, 4);
            if (pl.k == 8) rc = go(norm_reg_bwd<T, V, 8>, 8);
        }
        if (rc) return rc;
    } else if (pl.wide) {
        rows = pl.R;
        sw = ws;
        sb = ws + rows * p.C;
        const int smem = p.cg / V * 2 * kPairs<V> * 8;
        if (pl.R * p.G > 0x7fffffffll) return PE_ERR_UNSUPPORTED;
        float* pw = ga->dweight || ga->dbias ? sw : nullptr;
        const int rc = pl.local ? launch_reg(norm_wide_bwd<T, V, true>, pl.R * p.G, smem, s, p, (int)pl.R, pw, sb)
                                : launch_reg(norm_wide_bwd<T, V, false>, pl.R * p.G, 0, s, p, (int)pl.R, pw, sb);
        if (rc) return rc;
    } else if (pl.slab.R) {
        rows = p.N * pl.slab.R;
        sw = ws;
        sb = ws + rows * p.C;
        float* pw = ga->dweight || ga->dbias ? sw : nullptr;
        if (int rc = launch_slab(norm_slab_bwd<T, V>, p.N, pl.slab,
                                 slab_smem(pl.slab.CS, pl.slab.P, V, sizeof(T), true), s, p, pl.slab, pw, sb))
            return rc;
    } else {
        float* part = ws;
        sw = part + p.N * pl.q.chunks * 2 * p.C;
        sb = sw + p.N * p.C;
        float* gm = sb + p.N * p.C;
        rows = p.N;
        const int64_t cb = ceil_div(p.C / V, pl.q.bx);
        if (p.N * pl.q.chunks > 0x7fffffffll || cb > 65535 || p.N * p.G > 0x7fffffffll) return PE_ERR_UNSUPPORTED;
        const dim3 grid((unsigned)(p.N * pl.q.chunks), (unsigned)cb);
        norm_sums<T, V><<<grid, kBlock, 0, s>>>(p, pl.q, part);
        if (int rc = launched()) return rc;
        norm_sums_join<T><<<(unsigned)(p.N * p.G), kBlock, 0, s>>>(p, pl.q, part, sw, sb, gm);
        if (int rc = launched()) return rc;
        norm_apply_bwd<T, V><<<grid, kBlock, 0, s>>>(p, pl.q, gm);
        if (int rc = launched()) return rc;
    }
    const SumJob sums[2] = {{sw, rows, p.C, (int)a->dtype, ga->dweight}, {sb, rows, p.C, (int)a->dtype, ga->dbias}};
    return sum_rows(sums, 2, s);
}

#define PE_NORM_T(F, dtype, vec, ...)                                                                       \
    switch (dtype) {                                                                                        \
        case PE_F32: return (vec) > 1 ? F<float, 4>(__VA_ARGS__) : F<float, 1>(__VA_ARGS__);                \
        case PE_F16: return (vec) > 1 ? F<__half, 8>(__VA_ARGS__) : F<__half, 1>(__VA_ARGS__);              \
        default: return (vec) > 1 ? F<__nv_bfloat16, 8>(__VA_ARGS__) : F<__nv_bfloat16, 1>(__VA_ARGS__);    \
    }
int norm_any(const pe_norm_args* a, const Plan& pl, cudaStream_t s) { PE_NORM_T(norm_run, a->dtype, pl.v, a, pl, s) }
int norm_grad_any(const pe_norm_grad_args* a, const Plan& pl, cudaStream_t s) {
    PE_NORM_T(norm_grad_run, a->fwd.dtype, pl.v, a, pl, s)
}

// ws: norm_wide_bwd keeps sums in it that it reads and writes in vectors.
Plan grad_plan(const pe_norm_grad_args* g) {
    return plan_of(&g->fwd, vec_of(&g->fwd, {g->dout, g->dx, g->dgate, g->ws}, {g->dout_sb, g->dout_sp}), true);
}

}  // namespace

int64_t norm_ws_bytes(const pe_norm_args* a) {
    if (check_norm(a) != PE_OK || empty(a)) return 0;
    // enough for either width of the loads: the size does not depend on addresses
    const int64_t x = stats_floats(a, plan_of(a, 1, false)), y = stats_floats(a, plan_of(a, widest(a), false));
    return (x > y ? x : y) * 4;
}

int group_norm(const pe_norm_args* a, cudaStream_t s) {
    if (int rc = check_norm(a)) return rc;
    if (empty(a)) return PE_OK;
    if (!a->out || !a->mean != !a->rstd) return PE_ERR_INVALID;
    const Plan pl = plan_of(a, vec_of(a, {}, {}), false);
    const int64_t need = stats_floats(a, pl) * 4;
    if (need && (!a->ws || a->ws_bytes < need)) return PE_ERR_WORKSPACE;
    return norm_any(a, pl, s);
}

int64_t norm_grad_ws_bytes(const pe_norm_grad_args* g) {
    if (!g || check_norm(&g->fwd) != PE_OK || empty(&g->fwd)) return 0;
    const pe_norm_args* a = &g->fwd;
    const int64_t x = grad_floats(a, plan_of(a, 1, true)), y = grad_floats(a, plan_of(a, widest(a), true));
    return (x > y ? x : y) * 4;
}

int group_norm_grad(const pe_norm_grad_args* g, cudaStream_t s) {
    if (!g) return PE_ERR_INVALID;
    const pe_norm_args* a = &g->fwd;
    if (int rc = check_norm(a)) return rc;
    if (empty(a)) {
        const SumJob none[2] = {{nullptr, 0, a->channels, (int)a->dtype, g->dweight},
                                {nullptr, 0, a->channels, (int)a->dtype, g->dbias}};
        return sum_rows(none, 2, s);
    }
    if (!a->mean || !a->rstd || !g->dout || !g->dx || (a->gate && !g->dgate)) return PE_ERR_INVALID;
    const Plan pl = grad_plan(g);
    const int64_t need = grad_floats(a, pl) * 4;   // pe_group_norm_grad_ws_bytes is that or more
    if (!g->ws || g->ws_bytes < need) return PE_ERR_WORKSPACE;
    return norm_grad_any(g, pl, s);
}

}  // namespace pe

// pe_norm.cu - group norm over channels-last tensors with silu or a silu gate,
// forward and backward, for sm_100a.
//
//   xn = (x - mean) rstd,  v = xn w + b,  out = v | silu(v) | v silu(gate)
//   g = d out / d v . dout,  dw = sum g xn,  db = sum g,
//   dx = rstd (g w - mean(g w) - xn mean(g w xn))          (means over the group)
//
// Bound by memory. A group of up to 1024 loads (512 backward; 16 bytes each where
// the layout allows) stays in the registers of the lanes that share it: one read of x, two-pass
// statistics. A larger one goes over the tensor twice: per-channel sums of row chunks,
// their combination, then the result; the second read comes from L2 while the tensor
// fits there. Variances are never formed as a difference of large squares: two passes
// in registers, and sums shifted by a first value that are joined by Chan's formula
// elsewhere. Every sum has a fixed order.
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

// Blocks an SM holds of the kernels below, by loads a lane.
__host__ __device__ constexpr int reg_blocks(int k, bool grad) {
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

// L lanes share a group and take its rows r, r + R, ...; the next row's loads are on the
// way while the current one is reduced. All lanes make the same number of rounds, for
// the shuffles take all of them.
template <typename T, int V, int K>
__global__ void __launch_bounds__(kBlock, reg_blocks(K, false)) norm_reg(const __grid_constant__ NormP<T> p, int L, int R) {
    __shared__ float red[8];
    const int unit = (int)(((int64_t)blockIdx.x * kBlock + threadIdx.x) / L), l = threadIdx.x % L;
    const bool live = unit / p.G < R;
    const int r = live ? unit / p.G : 0, g = live ? unit % p.G : 0;
    const int per = p.cg / V;
    const Items<V, K> it(l, L, per, live ? per * (int)p.S : 0, g * p.cg);
    const float inv = 1.0f / (float)(p.cg * (int)p.S);
    int64_t xo[K], go[K];
    Vec<T, V> w[K], b[K], x[K], z[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        xo[k] = it.place[k] * p.x_sp + it.c[k];
        go[k] = it.place[k] * p.g_sp + it.c[k];
        if (it.in[k] && p.w) w[k] = load_vec<T, V>(p.w + it.c[k]);
        if (it.in[k] && p.b) b[k] = load_vec<T, V>(p.b + it.c[k]);
    }
    auto load = [&](int64_t n) {
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (it.in[k] && n < p.N) {
                x[k] = load_vec<T, V>(p.x + n * p.x_sb + xo[k]);
                if (p.mode == kGate) z[k] = load_vec<T, V>(p.gate + n * p.g_sb + go[k]);
            }
    };
    load(r);
    for (int64_t n0 = 0; n0 < p.N; n0 += R) {
        const int64_t n = n0 + r;
        const bool on = n < p.N;
        float f[K][V], ga[K][V], sum[1] = {0.0f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            unpack(x[k], f[k]);
            if (p.mode == kGate) unpack(z[k], ga[k]);
            float s = 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) s += f[k][v];
            sum[0] += it.in[k] ? s : 0.0f;
        }
        load(n + R);
        group_sum(sum, L, red);
        const float mean = sum[0] * inv;
        sum[0] = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float s = 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                f[k][v] -= mean;
                s = fmaf(f[k][v], f[k][v], s);
            }
            sum[0] += it.in[k] ? s : 0.0f;
        }
        group_sum(sum, L, red);
        const float rstd = rsqrtf(sum[0] * inv + p.eps);
        if (!live || !on) continue;
        if (l == 0 && p.mean) {
            p.mean[n * p.G + g] = mean;
            p.rstd[n * p.G + g] = rstd;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!it.in[k]) continue;
            float y[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                y[v] = f[k][v] * rstd;
                if (p.w) y[v] *= to_float(w[k].v[v]);
                if (p.b) y[v] += to_float(b[k].v[v]);
                if (p.mode == kSilu) y[v] *= sigmoidf(y[v]);
                if (p.mode == kGate) y[v] *= ga[k][v] * sigmoidf(ga[k][v]);
            }
            store_vec(p.out + (n * p.S + it.place[k]) * p.C + it.c[k], pack<T, V>(y));
        }
    }
}

// g = dL / dv, and the gate's gradient in place of `ga`.
template <int V>
__device__ __forceinline__ void through_act(int mode, const float (&xn)[V], const float (&w)[V], const float (&b)[V],
                                            float (&go)[V], float (&ga)[V]) {
    if (mode == kPlain) return;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const float val = fmaf(xn[v], w[v], b[v]);
        if (mode == kSilu) {
            go[v] *= silu_slope(val, sigmoidf(val));
        } else {
            const float s = sigmoidf(ga[v]), o = go[v];
            go[v] = o * ga[v] * s;
            ga[v] = o * val * silu_slope(ga[v], s);
        }
    }
}

// L lanes take rows r, r + R, ... of one group of channels (one place a row) and keep the
// sums of g xn and g of their own channels: pw, pb [R][C].
template <typename T, int V, int K>
__global__ void __launch_bounds__(kBlock, reg_blocks(K, true)) norm_reg_bwd(const __grid_constant__ NormP<T> p, int L, int R, float* pw,
                                                       float* pb) {
    __shared__ float red[16];
    const int unit = (int)(((int64_t)blockIdx.x * kBlock + threadIdx.x) / L), l = threadIdx.x % L;
    const bool live = unit / p.G < R;
    const int r = live ? unit / p.G : 0, g = live ? unit % p.G : 0;
    const int per = p.cg / V;
    const Items<V, K> it(l, L, per, live ? per : 0, g * p.cg);
    const float inv = 1.0f / (float)p.cg;
    float aw[K][V], ab[K][V];
    Vec<T, V> w[K], b[K], x[K], z[K], o[K];
    float mean = 0.0f, rstd = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            aw[k][v] = ab[k][v] = 0.0f;
            w[k].v[v] = from_float<T>(1.0f);
            b[k].v[v] = from_float<T>(0.0f);
        }
        if (it.in[k] && p.w) w[k] = load_vec<T, V>(p.w + it.c[k]);
        if (it.in[k] && p.b) b[k] = load_vec<T, V>(p.b + it.c[k]);
    }
    auto load = [&](int64_t n) {
        if (n < p.N) {
            mean = __ldg(p.mean + n * p.G + g);
            rstd = __ldg(p.rstd + n * p.G + g);
        }
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (it.in[k] && n < p.N) {
                x[k] = load_vec<T, V>(p.x + n * p.x_sb + it.c[k]);
                o[k] = load_vec<T, V>(p.dout + n * p.o_sb + it.c[k]);
                if (p.mode == kGate) z[k] = load_vec<T, V>(p.gate + n * p.g_sb + it.c[k]);
            }
    };
    load(r);
    for (int64_t n0 = 0; n0 < p.N; n0 += R) {
        const int64_t n = n0 + r;
        const bool on = n < p.N;
        const float scale = rstd;
        float xn[K][V], go[K][V], sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!it.in[k] || !on) continue;
            float ga[V], wf[V], bf[V];
            unpack(x[k], xn[k]);
            unpack(o[k], go[k]);
            unpack(w[k], wf);
            unpack(b[k], bf);
            if (p.mode == kGate) unpack(z[k], ga);
#pragma unroll
            for (int v = 0; v < V; ++v) xn[k][v] = (xn[k][v] - mean) * rstd;
            through_act<V>(p.mode, xn[k], wf, bf, go[k], ga);
            if (p.mode == kGate) store_vec(p.dgate + n * p.C + it.c[k], pack<T, V>(ga));
#pragma unroll
            for (int v = 0; v < V; ++v) {
                aw[k][v] = fmaf(go[k][v], xn[k][v], aw[k][v]);
                ab[k][v] += go[k][v];
                go[k][v] *= wf[v];
                sum[0] += go[k][v];
                sum[1] = fmaf(go[k][v], xn[k][v], sum[1]);
            }
        }
        load(n + R);
        group_sum(sum, L, red);
        const float m0 = sum[0] * inv, m1 = sum[1] * inv;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!it.in[k] || !on) continue;
            float d[V];
#pragma unroll
            for (int v = 0; v < V; ++v) d[v] = scale * (go[k][v] - m0 - xn[k][v] * m1);
            store_vec(p.dx + n * p.C + it.c[k], pack<T, V>(d));
        }
    }
    if (!pw) return;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (!it.in[k]) continue;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            pw[(int64_t)r * p.C + it.c[k] + v] = aw[k][v];
            pb[(int64_t)r * p.C + it.c[k] + v] = ab[k][v];
        }
    }
}

// ---- larger groups ------------------------------------------------------------------
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
        m2 += bm2 + d * d * n * f;
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
    for (int64_t i = threadIdx.x; i < items; i += kBlock) {
        const int64_t chunk = i / cg, c = (int64_t)g * cg + (i - chunk * cg);
        const float cnt = (float)(min(S, (chunk + 1) * q.rows) - chunk * q.rows);
        const float* b = part + (n * q.chunks + chunk) * 2 * C + c;
        m.join(cnt, b[0], b[C]);
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
    float w[V], b[V], mean[V], rstd[V];
    __device__ __forceinline__ Channel(const NormP<T>& p, int64_t n, int64_t c) {
#pragma unroll
        for (int v = 0; v < V; ++v) w[v] = 1.0f, b[v] = 0.0f;
        if (p.w) unpack(load_vec<T, V>(p.w + c), w);
        if (p.b) unpack(load_vec<T, V>(p.b + c), b);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int64_t g = n * p.G + (int)(c + v) / p.cg;
            mean[v] = __ldg(p.mean + g);
            rstd[v] = __ldg(p.rstd + g);
        }
    }
};

template <typename T, int V>
__global__ void __launch_bounds__(kBlock) norm_apply(const __grid_constant__ NormP<T> p, Chunks q) {
    const int by = kBlock / q.bx, x = threadIdx.x % q.bx, y = threadIdx.x / q.bx;
    const int64_t n = blockIdx.x / (unsigned)q.chunks, chunk = blockIdx.x % (unsigned)q.chunks;
    const int64_t c = ((int64_t)blockIdx.y * q.bx + x) * V;
    if (c >= p.C) return;
    const int64_t s0 = chunk * q.rows, s1 = min(p.S, s0 + q.rows);
    const Channel<T, V> ch(p, n, c);
#pragma unroll 4
    for (int64_t i = s0 + y; i < s1; i += by) {
        float f[V], ga[V];
        unpack(load_vec<T, V>(p.x + n * p.x_sb + i * p.x_sp + c), f);
        if (p.mode == kGate) unpack(load_vec<T, V>(p.gate + n * p.g_sb + i * p.g_sp + c), ga);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            f[v] = fmaf((f[v] - ch.mean[v]) * ch.rstd[v], ch.w[v], ch.b[v]);
            if (p.mode == kSilu) f[v] *= sigmoidf(f[v]);
            if (p.mode == kGate) f[v] *= ga[v] * sigmoidf(ga[v]);
        }
        store_vec(p.out + (n * p.S + i) * p.C + c, pack<T, V>(f));
    }
}

// Per-channel sums of g xn and g over a chunk's places: part [n][chunk][2][C].
template <typename T, int V>
__global__ void __launch_bounds__(kBlock) norm_sums(const __grid_constant__ NormP<T> p, Chunks q, float* part) {
    __shared__ float red[2][V][kBlock];
    const int by = kBlock / q.bx, x = threadIdx.x % q.bx, y = threadIdx.x / q.bx;
    const int64_t n = blockIdx.x / (unsigned)q.chunks, chunk = blockIdx.x % (unsigned)q.chunks;
    const int64_t c = ((int64_t)blockIdx.y * q.bx + x) * V;
    const int64_t s0 = chunk * q.rows, s1 = min(p.S, s0 + q.rows);
    float aw[V], ab[V];
#pragma unroll
    for (int v = 0; v < V; ++v) aw[v] = ab[v] = 0.0f;
    if (c < p.C) {
        const Channel<T, V> ch(p, n, c);
#pragma unroll 2
        for (int64_t i = s0 + y; i < s1; i += by) {
            float xn[V], go[V], ga[V];
            unpack(load_vec<T, V>(p.x + n * p.x_sb + i * p.x_sp + c), xn);
            unpack(load_vec<T, V>(p.dout + n * p.o_sb + i * p.o_sp + c), go);
            if (p.mode == kGate) unpack(load_vec<T, V>(p.gate + n * p.g_sb + i * p.g_sp + c), ga);
#pragma unroll
            for (int v = 0; v < V; ++v) xn[v] = (xn[v] - ch.mean[v]) * ch.rstd[v];
            through_act<V>(p.mode, xn, ch.w, ch.b, go, ga);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                aw[v] = fmaf(go[v], xn[v], aw[v]);
                ab[v] += go[v];
            }
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
        red[0][v][threadIdx.x] = aw[v];
        red[1][v][threadIdx.x] = ab[v];
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
        for (int64_t k = 0; k < q.chunks; ++k) {
            aw += __ldg(b + 2 * k * p.C);
            ab += __ldg(b + (2 * k + 1) * p.C);
        }
        sw[n * p.C + c] = aw;
        sb[n * p.C + c] = ab;
        const float w = p.w ? to_float(__ldg(p.w + c)) : 1.0f;
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
__global__ void __launch_bounds__(kBlock) norm_apply_bwd(const __grid_constant__ NormP<T> p, Chunks q,
                                                         const float* gm) {
    const int by = kBlock / q.bx, x = threadIdx.x % q.bx, y = threadIdx.x / q.bx;
    const int64_t n = blockIdx.x / (unsigned)q.chunks, chunk = blockIdx.x % (unsigned)q.chunks;
    const int64_t c = ((int64_t)blockIdx.y * q.bx + x) * V;
    if (c >= p.C) return;
    const int64_t s0 = chunk * q.rows, s1 = min(p.S, s0 + q.rows);
    const Channel<T, V> ch(p, n, c);
    float m0[V], m1[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int64_t g = n * p.G + (int)(c + v) / p.cg;
        m0[v] = __ldg(gm + 2 * g);
        m1[v] = __ldg(gm + 2 * g + 1);
    }
#pragma unroll 2
    for (int64_t i = s0 + y; i < s1; i += by) {
        float xn[V], go[V], ga[V];
        const int64_t o = (n * p.S + i) * p.C + c;
        unpack(load_vec<T, V>(p.x + n * p.x_sb + i * p.x_sp + c), xn);
        unpack(load_vec<T, V>(p.dout + n * p.o_sb + i * p.o_sp + c), go);
        if (p.mode == kGate) unpack(load_vec<T, V>(p.gate + n * p.g_sb + i * p.g_sp + c), ga);
#pragma unroll
        for (int v = 0; v < V; ++v) xn[v] = (xn[v] - ch.mean[v]) * ch.rstd[v];
        through_act<V>(p.mode, xn, ch.w, ch.b, go, ga);
        if (p.mode == kGate) store_vec(p.dgate + o, pack<T, V>(ga));
#pragma unroll
        for (int v = 0; v < V; ++v) go[v] = ch.rstd[v] * (go[v] * ch.w[v] - m0[v] - xn[v] * m1[v]);
        store_vec(p.dx + o, pack<T, V>(go));
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

// Elements a load: 16 bytes where all rows start on that boundary, else one.
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
    Chunks q;
};

Plan plan_of(const pe_norm_args* a, int vec, bool grad) {
    Plan p{};
    const int64_t cg = a->channels / a->groups;
    const int vr = cg % vec == 0 ? vec : 1;      // in registers a load stays within its group
    const int64_t items = a->places <= 1024 ? cg / vr * a->places : 1 << 20;
    // the backward pass keeps sums a channel in registers, where an item is a channel vector
    // (two loads a lane at most: four need more registers than there are)
    const int most = grad ? 2 : 4;
    if (items <= most * kBlock && (!grad || a->places == 1)) {
        p.v = vr;
        if (items <= 32 * most) {
            p.lanes = 1;
            while (p.lanes < 32 && p.lanes < items) p.lanes *= 2;
        } else {
            p.lanes = kBlock;
        }
        const int64_t k = ceil_div(items, p.lanes);
        p.k = k <= 1 ? 1 : k <= 2 ? 2 : 4;
        // rows of groups at work: one wave of blocks; each then takes further rows, so that
        // its filter and its sums weigh less
        const int64_t want = (int64_t)num_sms() * reg_blocks(p.k, grad) * kBlock / p.lanes / a->groups;
        p.R = a->batch < want ? a->batch : want < 1 ? 1 : want;
        return p;
    }
    p.v = vec;
    const int64_t cv = a->channels / vec;
    p.q.bx = 32;
    while (p.q.bx > 1 && ceil_div(cv, p.q.bx) * p.q.bx * 8 > cv * 9) p.q.bx /= 2;
    const int64_t blocks = ceil_div(cv, p.q.bx) * a->batch, by = kBlock / p.q.bx;
    const int64_t want = ceil_div((int64_t)num_sms() * 8, blocks > 0 ? blocks : 1);
    p.q.rows = ceil_div(ceil_div(a->places, want), by) * by;
    if (p.q.rows < 4 * by) p.q.rows = 4 * by;
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
    return pl.lanes ? 0 : a->batch * (pl.q.chunks * 2 * a->channels + 2 * a->groups);
}

template <typename T, int V>
int norm_run(const pe_norm_args* a, const Plan& pl, cudaStream_t s) {
    NormP<T> p = norm_params<T>(a);
    const int64_t units = p.N * p.G;
    if (pl.lanes) {
        const int64_t blocks = ceil_div(pl.R * p.G * pl.lanes, kBlock);
        if (blocks > 0x7fffffll) return PE_ERR_UNSUPPORTED;
        if (pl.k == 1) norm_reg<T, V, 1><<<(unsigned)blocks, kBlock, 0, s>>>(p, pl.lanes, (int)pl.R);
        else if (pl.k == 2) norm_reg<T, V, 2><<<(unsigned)blocks, kBlock, 0, s>>>(p, pl.lanes, (int)pl.R);
        else norm_reg<T, V, 4><<<(unsigned)blocks, kBlock, 0, s>>>(p, pl.lanes, (int)pl.R);
        return launched();
    }
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
    if (pl.lanes) return 2 * pl.R * a->channels;
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
        if (pl.k == 1) norm_reg_bwd<T, V, 1><<<(unsigned)blocks, kBlock, 0, s>>>(p, pl.lanes, (int)pl.R, pw, sb);
        else norm_reg_bwd<T, V, 2><<<(unsigned)blocks, kBlock, 0, s>>>(p, pl.lanes, (int)pl.R, pw, sb);
        if (int rc = launched()) return rc;
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

Plan grad_plan(const pe_norm_grad_args* g) {
    return plan_of(&g->fwd, vec_of(&g->fwd, {g->dout, g->dx, g->dgate}, {g->dout_sb, g->dout_sp}), true);
}

}  // namespace

int64_t norm_ws_bytes(const pe_norm_args* a) {
    if (check_norm(a) != PE_OK) return 0;
    // enough for either width of the loads: the size does not depend on addresses
    const int64_t x = stats_floats(a, plan_of(a, 1, false)), y = stats_floats(a, plan_of(a, widest(a), false));
    return (x > y ? x : y) * 4;
}

int group_norm(const pe_norm_args* a, cudaStream_t s) {
    if (int rc = check_norm(a)) return rc;
    if (a->batch == 0 || a->places == 0) return PE_OK;
    if (!a->out || !a->mean != !a->rstd) return PE_ERR_INVALID;
    const Plan pl = plan_of(a, vec_of(a, {}, {}), false);
    const int64_t need = stats_floats(a, pl) * 4;
    if (need && (!a->ws || a->ws_bytes < need)) return PE_ERR_WORKSPACE;
    return norm_any(a, pl, s);
}

int64_t norm_grad_ws_bytes(const pe_norm_grad_args* g) {
    if (!g || check_norm(&g->fwd) != PE_OK) return 0;
    const pe_norm_args* a = &g->fwd;
    const int64_t x = grad_floats(a, plan_of(a, 1, true)), y = grad_floats(a, plan_of(a, widest(a), true));
    return (x > y ? x : y) * 4;
}

int group_norm_grad(const pe_norm_grad_args* g, cudaStream_t s) {
    if (!g) return PE_ERR_INVALID;
    const pe_norm_args* a = &g->fwd;
    if (int rc = check_norm(a)) return rc;
    if (a->batch == 0 || a->places == 0) {
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

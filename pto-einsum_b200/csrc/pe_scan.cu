// pe_scan.cu - selective state space scan: prompts (forward) and single tokens,
// for sm_100a.
//
//   h[n] = exp(dt A[n]) h[n] + dt u B[n],   y = sum_n C[n] h[n] + D u
//
// per channel, dt = softplus(delta + bias). A thread keeps four states of one channel in
// registers; LPC = 1 .. 32 neighbouring lanes share a channel (4 LPC >= states). Tokens
// go through in tiles of 16: what depends on (token, channel) alone (softplus, the gate)
// is computed once by all threads of the block and passed in shared memory, and so are
// B and C in fp32; the sums over states are reduced for LPC tokens together
// (reduce_scatter: LPC - 1 shuffles for LPC tokens).
//
// Times in these files' comments are of a B200, by replays of a captured call.
#include <cmath>
#include <cstddef>

#include "pe_scan.cuh"

namespace pe {

namespace {

// ---- forward --------------------------------------------------------------------
constexpr int TS = 16;       // tokens a tile

template <int LPC>
struct Lanes {
    static constexpr int CH = kThreads / LPC;    // channels a block
    static constexpr int NP = 4 * LPC;           // states, padded
    static constexpr int R = LPC < TS ? LPC : TS;
    // (token pair, channel pair) items of the element-wise work: I a thread
    static constexpr int ITEMS = CH / 2 * (TS / 2), I = (ITEMS + kThreads - 1) / kThreads;
    // row of a [token][channel] tile of floats: the lanes of a warp hold 32 / LPC channels of
    // LPC tokens, which fall on different banks with these
    static constexpr int Y = LPC == 1 ? 128 : LPC == 2 ? 80 : LPC == 4 ? 40 : LPC == 8 ? 20 : LPC == 16 ? 10 : 6;
};

// B or C of a tile: fp32 [TS][NP], zero past the last token and state.
template <int NP, typename T>
__device__ __forceinline__ void widen_rows(float* dst, const T* src, int cnt, int N) {
    constexpr int J = TS * NP / 2 / kThreads;
#pragma unroll
    for (int j = 0; j < (J > 0 ? J : 1); ++j) {
        const int i = 2 * (threadIdx.x + j * kThreads), t = i / NP, n = i % NP;
        if (J == 0 && i >= TS * NP) break;
        const Vec<T, 2> v = *reinterpret_cast<const Vec<T, 2>*>(src + i);
        *reinterpret_cast<float2*>(dst + i) = make_float2(t < cnt && n < N ? to_float(v.v[0]) : 0.0f,
                                                          t < cnt && n + 1 < N ? to_float(v.v[1]) : 0.0f);
    }
}

// Shared memory of a block; two of each part, for even and odd tiles.
template <typename T, int LPC, bool STATE_ONLY>
struct FwdSmem {
    using L = Lanes<LPC>;
    struct __align__(16) Raw {       // as in memory
        T u[TS * L::CH], d[TS * L::CH], b[TS * L::NP];
        T z[STATE_ONLY ? 8 : TS * L::CH], c[STATE_ONLY ? 8 : TS * L::NP];
    } raw[2];
    struct __align__(16) Wide {      // (dt, dt u) of each token and channel; B, C
        float2 dx[TS][L::CH];
        float B[TS * L::NP], C[STATE_ONLY ? 4 : TS * L::NP];
    } fp[2];
    float y[2][STATE_ONLY ? 4 : TS * L::Y];
};

// The copies of a tile where every row allows 16-byte chunks: the chunks of all tensors
// in one list, a thread's entries of it worked out once.
template <typename T, int LPC, bool STATE_ONLY>
struct Feeder {
    using L = Lanes<LPC>;
    using F = FwdSmem<T, LPC, STATE_ONLY>;
    static constexpr int E = 16 / (int)sizeof(T);
    static constexpr int PC = L::CH / E, PN = L::NP / E;   // chunks a row
    static constexpr bool POSSIBLE = L::CH % E == 0 && L::NP % E == 0;
    static constexpr int TOTAL = TS * ((STATE_ONLY ? 2 : 3) * PC + (STATE_ONLY ? 1 : 2) * PN);
    static constexpr int J = (TOTAL + kThreads - 1) / kThreads;
    const T* src[J];
    int64_t step[J];      // elements a tile
    int to[J], valid[J];  // offset in the raw buffer; bytes
    int t[J];             // row of the tile (TS: none)

    __device__ __forceinline__ void init(const ScanP<T>& p, const Place& w, const T* u, const T* d, const T* z,
                                         const T* b, const T* c) {
        using Raw = typename F::Raw;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            int i = threadIdx.x + j * kThreads;
            t[j] = TS;
            src[j] = u;
            to[j] = valid[j] = 0;
            step[j] = 0;
            auto entry = [&](const T* from, int64_t st, int per, int width, int base, int row) {
                if (i >= 0 && i < TS * per && from) {
                    const int r = i / per, k = i % per * E;
                    if (k < width) {
                        t[j] = r;
                        src[j] = from + r * st + k;
                        step[j] = TS * st;
                        to[j] = base + (r * row + k) * (int)sizeof(T);
                        valid[j] = min(16, (width - k) * (int)sizeof(T));
                    }
                }
                i -= TS * per;
            };
            entry(u, p.u_st, PC, w.nch, (int)offsetof(Raw, u), L::CH);
            entry(d, p.d_st, PC, w.nch, (int)offsetof(Raw, d), L::CH);
            entry(b, p.B_st, PN, p.N, (int)offsetof(Raw, b), L::NP);
            if constexpr (!STATE_ONLY) {
                entry(c, p.C_st, PN, p.N, (int)offsetof(Raw, c), L::NP);
                entry(z, p.z_st, PC, w.nch, (int)offsetof(Raw, z), L::CH);
            }
        }
    }
    // the next tile, of cnt tokens
    __device__ __forceinline__ void copy(void* raw, int cnt) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if (t[j] < cnt) cp_async<16>((char*)raw + to[j], src[j], valid[j]);
            src[j] += step[j];
        }
    }
};

// STATE_ONLY: a piece's last state from a zero start and its sum of dt (first half of
// a split scan); else the whole, starting from what the sequence's earlier pieces left.
//
// Three tiles are under way between two barriers: the copies of tile i + 2 from memory,
// the element-wise work before tile i + 1 and after tile i - 1, and the recurrence of
// tile i; what one barrier interval writes, the next one reads. Tokens past the end have
// dt = 0 and B = 0: they leave the state as it is.
//
// Instructions, 42 a warp and four states of a token, and their latency at four warps a scheduler
// count about alike: it issues in 62% of the clocks. 17 packed fp16 prompts of 8192 tokens in all,
// 4096 channels, 16 states take 253 us, 2.7 T exponentials a second (57% of 16 a clock an SM). More
// tiles than 16 tokens' would take the shared memory of a block (four an SM; five, at 96 registers,
// were 3% slower). A form parallel along the tokens, lanes composing their tokens' maps, needed 64
// instructions and 1.6 times the time.
//
// FAST: 16-byte asynchronous copies, where all rows allow them, against elements through
// registers: 2 x 8000 tokens of 2048 and of 2049 channels 447 and 605 us.
template <typename T, int LPC, bool STATE_ONLY, bool FAST>
__global__ void __launch_bounds__(kThreads, LPC >= 4 ? 4 : LPC == 2 ? 3 : 2)
    scan_fwd(const __grid_constant__ ScanP<T> p) {
    using L = Lanes<LPC>;
    constexpr int CH = L::CH, NP = L::NP, R = L::R, I = L::I, Y = L::Y;
    using F = FwdSmem<T, LPC, STATE_ONLY>;
    extern __shared__ __align__(16) unsigned char smem[];
    F& m = *reinterpret_cast<F*>(smem);
    const int tid = threadIdx.x, lane = tid & 31;
    if (blockIdx.x == 0 && tid < 32) check_offsets(p.seqs, lane, kSiteOffsets);
    const Place w = place_of<CH>(p);
    if (!w.any || (STATE_ONLY && w.t1 == w.sp.len)) return;   // nothing starts from the last piece's state
    const int ch = tid / LPC, q = tid % LPC, c = w.c0 + ch, n0 = 4 * q;
    const bool live = ch < w.nch;

    // rows of the piece's first token
    const int64_t row0 = w.sp.start + w.t0;
    const T* u = p.u + w.sp.row * p.u_sb + row0 * p.u_st + w.c0;
    const T* delta = p.delta + w.sp.row * p.d_sb + row0 * p.d_st + w.c0;
    const T* z = p.z ? p.z + w.sp.row * p.z_sb + row0 * p.z_st + w.c0 : nullptr;
    const T* B = p.B + w.sp.row * p.B_sb + row0 * p.B_st + w.g * p.B_sg;
    const T* C = p.C + w.sp.row * p.C_sb + row0 * p.C_st + w.g * p.C_sg;
    const int64_t count = w.t1 - w.t0;                        // tokens
    using Feed = Feeder<T, LPC, STATE_ONLY>;
    Feed feed;
    Elements<TS, CH, kThreads, T> eu, ed, ez;
    Elements<TS, NP, kThreads, T> eb, ec;
    if constexpr (FAST) feed.init(p, w, u, delta, z, B, C);
    auto copy = [&](int64_t t, int b) {   // tiles in order
        if (t < count) {
            const int cnt = (int)min((int64_t)TS, count - t);
            if constexpr (FAST) {
                feed.copy(&m.raw[b], cnt);
            } else if (p.chunks) {
                stage<TS, CH>(m.raw[b].u, u + t * p.u_st, p.u_st, cnt, w.nch, p.u_cb);
                stage<TS, CH>(m.raw[b].d, delta + t * p.d_st, p.d_st, cnt, w.nch, p.d_cb);
                stage<TS, NP>(m.raw[b].b, B + t * p.B_st, p.B_st, cnt, p.N, p.B_cb);
                if constexpr (!STATE_ONLY) {
                    stage<TS, NP>(m.raw[b].c, C + t * p.C_st, p.C_st, cnt, p.N, p.C_cb);
                    if (z) stage<TS, CH>(m.raw[b].z, z + t * p.z_st, p.z_st, cnt, w.nch, p.z_cb);
                }
            } else {
                eu.load(u + t * p.u_st, p.u_st, cnt, w.nch);
                ed.load(delta + t * p.d_st, p.d_st, cnt, w.nch);
                eb.load(B + t * p.B_st, p.B_st, cnt, p.N);
                if constexpr (!STATE_ONLY) {
                    ec.load(C + t * p.C_st, p.C_st, cnt, p.N);
                    if (z) ez.load(z + t * p.z_st, p.z_st, cnt, w.nch);
                }
            }
        }
        cp_commit();
    };
    // the second half of a copy of elements
    auto land = [&](int b) {
        if constexpr (!FAST) {
            if (p.chunks) return;
            eu.store(m.raw[b].u);
            ed.store(m.raw[b].d);
            eb.store(m.raw[b].b);
            if constexpr (!STATE_ONLY) {
                ec.store(m.raw[b].c);
                if (z) ez.store(m.raw[b].z);
            }
        }
    };
    copy(0, 0);

    float A[4], h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool in = live && n0 + i < p.N;
        A[i] = in ? rate(__ldg(p.A + (int64_t)c * p.N + n0 + i)) : 0.0f;
        h[i] = 0.0f;
    }
    const int64_t DN = (int64_t)p.D * p.N, cn = (int64_t)c * p.N + n0;
    // this thread's items: token pairs 2 tp of channel pairs 2 cp
    float bias[I][2], Dw[I][2];
#pragma unroll
    for (int k = 0; k < I; ++k) {
        const int cp = (tid + k * kThreads) % (CH / 2) * 2;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const bool in = cp + e < w.nch;
            bias[k][e] = p.bias && in ? __ldg(p.bias + w.c0 + cp + e) : 0.0f;
            Dw[k][e] = !STATE_ONLY && p.Dw && in ? __ldg(p.Dw + w.c0 + cp + e) : 0.0f;
        }
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
    float* ckpt = !STATE_ONLY && p.ckpt && live
                      ? p.ckpt + (piece_base(p.seqs, w.s, KCK) + w.t0 / KCK) * DN + cn : nullptr;
    T* out = STATE_ONLY ? nullptr : p.out + (w.sp.row * p.seqs.tokens + row0) * p.D + w.c0;

    // D u and silu(z) of the thread's items: [0] of the tile whose recurrence runs, [1] of the next
    float add[2][I][2][2], gate[2][I][2][2];
    auto before = [&](int64_t t, int b) {
        const int cnt = (int)max((int64_t)0, min((int64_t)TS, count - t));
#pragma unroll
        for (int k = 0; k < I; ++k) {
            const int it = tid + k * kThreads, cp = it % (CH / 2) * 2, tp = it / (CH / 2) * 2;
            if (L::ITEMS % kThreads && it >= L::ITEMS) break;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const Vec<T, 2> dv = *reinterpret_cast<const Vec<T, 2>*>(m.raw[b].d + (tp + i) * CH + cp);
                const Vec<T, 2> uv = *reinterpret_cast<const Vec<T, 2>*>(m.raw[b].u + (tp + i) * CH + cp);
                float f[4];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float x = to_float(uv.v[e]);
                    float dt = to_float(dv.v[e]) + bias[k][e];
                    if (p.softplus) dt = softplusf(dt);
                    f[2 * e] = tp + i < cnt ? dt : 0.0f;
                    f[2 * e + 1] = tp + i < cnt ? dt * x : 0.0f;
                    if constexpr (!STATE_ONLY) add[1][k][i][e] = Dw[k][e] * x;
                }
                *reinterpret_cast<float4*>(&m.fp[b].dx[tp + i][cp]) = make_float4(f[0], f[1], f[2], f[3]);
                if constexpr (!STATE_ONLY) {
                    gate[1][k][i][0] = gate[1][k][i][1] = 1.0f;
                    if (z) {
                        const Vec<T, 2> zv = *reinterpret_cast<const Vec<T, 2>*>(m.raw[b].z + (tp + i) * CH + cp);
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float g = to_float(zv.v[e]);
                            gate[1][k][i][e] = g * sigmoidf(g);
                        }
                    }
                }
            }
        }
        widen_rows<NP>(m.fp[b].B, m.raw[b].b, cnt, p.N);
        if constexpr (!STATE_ONLY) widen_rows<NP>(m.fp[b].C, m.raw[b].c, cnt, p.N);
    };
    auto after = [&](int64_t t, int cnt, int b) {   // out = (y + D u) silu(z)
        if constexpr (!STATE_ONLY) {
#pragma unroll
            for (int k = 0; k < I; ++k) {
                const int it = tid + k * kThreads, cp = it % (CH / 2) * 2, tp = it / (CH / 2) * 2;
                if (L::ITEMS % kThreads && it >= L::ITEMS) break;
                T* o = out + (t + tp) * p.D + cp;
#pragma unroll
                for (int i = 0; i < 2; ++i, o += p.D) {
                    if (tp + i >= cnt) break;
                    const float2 y = *reinterpret_cast<const float2*>(&m.y[b][(tp + i) * Y + cp]);
                    Vec<T, 2> v;
                    v.v[0] = from_float<T>((y.x + add[0][k][i][0]) * gate[0][k][i][0]);
                    v.v[1] = from_float<T>((y.y + add[0][k][i][1]) * gate[0][k][i][1]);
                    if (p.pairs && cp < w.nch) {
                        *reinterpret_cast<Vec<T, 2>*>(o) = v;
                    } else {
                        if (cp < w.nch) o[0] = v.v[0];
                        if (cp + 1 < w.nch) o[1] = v.v[1];
                    }
                }
            }
        }
    };
    auto shift = [&]() {
        if constexpr (!STATE_ONLY) {
#pragma unroll
            for (int k = 0; k < I; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    add[0][k][i / 2][i % 2] = add[1][k][i / 2][i % 2];
                    gate[0][k][i / 2][i % 2] = gate[1][k][i / 2][i % 2];
                }
        }
    };

    land(0);
    cp_wait();
    __syncthreads();
    copy(TS, 1);
    before(0, 0);
    land(1);
    int b = 0;
    for (int64_t t = 0; t < count; t += TS, b ^= 1) {
        cp_wait();
        __syncthreads();
        copy(t + 2 * TS, b);
        if (t > 0) after(t - TS, TS, b ^ 1);
        shift();
        before(t + TS, b ^ 1);
        if (ckpt && t % KCK == 0) {
            unpack2(h01, h[0], h[1]);
            unpack2(h23, h[2], h[3]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n0 + i < p.N) ckpt[i] = h[i];
            ckpt += DN;
        }
        // four tokens at a time: all that does not depend on the state first
        float y[TS];
#pragma unroll
        for (int k0 = 0; k0 < TS; k0 += 4) {
            f32x2 a[4][2], x[4][2];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 dx = m.fp[b].dx[k0 + k][ch];
                const f32x2 dt2 = pack2(dx.x, dx.x), x2 = pack2(dx.y, dx.y);
                const ulonglong2 bv = *reinterpret_cast<const ulonglong2*>(&m.fp[b].B[(k0 + k) * NP + n0]);
                a[k][0] = decay2(dt2, A01);
                a[k][1] = decay2(dt2, A23);
                x[k][0] = mul2(x2, bv.x);
                x[k][1] = mul2(x2, bv.y);
                if constexpr (STATE_ONLY) dtsum += dx.x;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                h01 = fma2(a[k][0], h01, x[k][0]);
                h23 = fma2(a[k][1], h23, x[k][1]);
                if constexpr (!STATE_ONLY) {
                    const ulonglong2 cv = *reinterpret_cast<const ulonglong2*>(&m.fp[b].C[(k0 + k) * NP + n0]);
                    float lo, hi;
                    unpack2(fma2(cv.y, h23, mul2(cv.x, h01)), lo, hi);
                    y[k0 + k] = lo + hi;
                }
            }
            if constexpr (!STATE_ONLY) {
                if ((k0 + 4) % R == 0) {   // R = 8, 16: after so many tokens; R < 4: several sums
#pragma unroll
                    for (int r0 = k0 + 4 - (R > 4 ? R : 4); r0 < k0 + 4; r0 += R) {
                        float v[R];
#pragma unroll
                        for (int i = 0; i < R; ++i) v[i] = y[r0 + i];
                        float sum = reduce_scatter<R, 1>(v, lane);
                        if (LPC > R) sum += __shfl_xor_sync(0xffffffffu, sum, R);
                        if (q < R) m.y[b][(r0 + q) * Y + ch] = sum;
                    }
                }
            }
        }
        land(b);
    }
    if (!STATE_ONLY && count > 0) {
        __syncthreads();
        const int64_t t = (count - 1) / TS * TS;
        after(t, (int)(count - t), b ^ 1);
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
// do not depend on one another, so the loads of eight pieces are in flight together
// (5 us of the 870 that a prompt of 32768 x 2048 x 16 takes).
template <typename T>
__global__ void __launch_bounds__(kThreads) scan_carry(const __grid_constant__ ScanP<T> p) {
    const int64_t DN = (int64_t)p.D * p.N, i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= DN) return;
    const int s = blockIdx.y;
    const int64_t len = seq_span(p.seqs, s).len, base = piece_base(p.seqs, s, p.piece);
    const int64_t n = len > p.piece ? ceil_div(len, p.piece) : 1;
    const int c = (int)(i / p.N);
    const float A = rate(__ldg(p.A + i));
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

// Eight consecutive fp32, one 32-byte access each way (32-byte aligned).
__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7])
                 : "l"(p)
                 : "memory");
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
    asm volatile("st.global.v8.f32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"f"(f[0]), "f"(f[1]), "f"(f[2]),
                 "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]), "l"(p)
                 : "memory");
}
// Eight consecutive elements of B or C as fp32.
template <typename T>
__device__ __forceinline__ void load_cols8(const T* p, float (&f)[8]) {
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int k = 0; k < 8 / E; ++k) {
        float g[E];
        unpack(load_vec<T, E>(p + k * E), g);
#pragma unroll
        for (int i = 0; i < E; ++i) f[k * E + i] = g[i];
    }
}

// A lane has eight states of one channel, LPC lanes a channel, for RB requests: A is read
// once for them, and all their states are on the way before the first is used. Bound by
// memory: the states, 8 bytes a (request, channel, state). Fewer states a lane repeat
// what the channel needs (softplus, gate, loads) on more lanes (four states a lane: 43 us a
// call, eight 29, of which the kernel has 23, 5.9 TB/s of states, for 256 requests of 4096
// channels and 16 states); 256-bit accesses let eight be one sector each. VEC against
// elements: 200 requests of 2048 x 32 and of 2049 x 31 states 21 and 54 us.
template <typename T, int LPC, int RB, bool VEC>
__global__ void __launch_bounds__(kThreads) scan_step(const __grid_constant__ StepP<T> p) {
    constexpr int CH = kThreads / LPC, NS = 8;
    const int tid = threadIdx.x, q = tid % LPC, n0 = NS * q;
    const int c = blockIdx.x * CH + tid / LPC;
    const bool live = c < p.D, some = live && n0 < p.N;
    const int64_t b0 = (int64_t)blockIdx.y * RB, cn = (int64_t)c * p.N + n0;
    const int nn = some ? min(NS, p.N - n0) : 0;   // this lane's states
    float h[RB][NS], B[RB][NS], C[RB][NS], A[NS], u[RB], dt[RB], z[RB];
    float* hp[RB];
    const int g = live ? c / p.Dg : 0;
    const int rows = (int)min((int64_t)RB, p.batch - b0);
#pragma unroll
    for (int r = 0; r < RB; ++r) {
        int64_t slot = -1;
        if (r < rows) {
            const int64_t b = b0 + r;
            slot = p.s32 ? (int64_t)__ldg(p.s32 + b) : p.s64 ? __ldg(p.s64 + b) : b;
            if (slot >= p.slots) {
                if (blockIdx.x == 0 && tid == 0) record_error(PE_ERR_INVALID | (kSiteSlot << 8));
                slot = -1;
            }
        }
        hp[r] = slot >= 0 ? p.state + slot * p.D * p.N + cn : nullptr;
    }
#pragma unroll
    for (int r = 0; r < RB; ++r) {
#pragma unroll
        for (int i = 0; i < NS; ++i) h[r][i] = 0.0f;
        if (VEC) {
            if (hp[r] && some) load8(hp[r], h[r]);
        } else {
#pragma unroll
            for (int i = 0; i < NS; ++i)
                if (hp[r] && i < nn) h[r][i] = hp[r][i];
        }
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) A[i] = 0.0f;
    if (VEC) {
        if (some) load_cols8(p.A + cn, A);
    } else {
#pragma unroll
        for (int i = 0; i < NS; ++i)
            if (i < nn) A[i] = __ldg(p.A + cn + i);
    }
    const float bias = live && p.bias ? __ldg(p.bias + c) : 0.0f, Dw = live && p.Dw ? __ldg(p.Dw + c) : 0.0f;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
        const int64_t b = b0 + r;
        const bool on = hp[r] && live;
        u[r] = on ? to_float(load_one(p.u + b * p.u_sb + c)) : 0.0f;
        dt[r] = on ? to_float(load_one(p.delta + b * p.d_sb + c)) + bias : 0.0f;
        z[r] = on && p.z ? to_float(load_one(p.z + b * p.z_sb + c)) : 0.0f;
        const T* Bp = p.B + b * p.B_sb + g * p.B_sg + n0;
        const T* Cp = p.C + b * p.C_sb + g * p.C_sg + n0;
#pragma unroll
        for (int i = 0; i < NS; ++i) B[r][i] = C[r][i] = 0.0f;
        if (VEC) {
            if (on && some) {
                load_cols8(Bp, B[r]);
                load_cols8(Cp, C[r]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NS; ++i)
                if (on && i < nn) {
                    B[r][i] = to_float(load_one(Bp + i));
                    C[r][i] = to_float(load_one(Cp + i));
                }
        }
    }
#pragma unroll
    for (int r = 0; r < RB; ++r) {
        if (r >= rows) break;
        const float d = p.softplus ? softplusf(dt[r]) : dt[r], x = d * u[r], dl = d * kLog2e;
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            h[r][i] = fmaf(decay(dl, A[i]), h[r][i], x * B[r][i]);
            y = fmaf(C[r][i], h[r][i], y);
        }
        if (VEC) {
            if (hp[r] && some) store8(hp[r], h[r]);
        } else {
#pragma unroll
            for (int i = 0; i < NS; ++i)
                if (hp[r] && i < nn) hp[r][i] = h[r][i];
        }
#pragma unroll
        for (int m = LPC / 2; m >= 1; m /= 2) y += __shfl_xor_sync(0xffffffffu, y, m);
        if (live && q == 0) {
            y = fmaf(Dw, u[r], y);
            if (p.z) y *= z[r] * sigmoidf(z[r]);
            p.out[(b0 + r) * p.D + c] = from_float<T>(hp[r] ? y : 0.0f);
        }
    }
}

// ---- host -------------------------------------------------------------------------
int lanes_for(int64_t states) {
    int l = 1;
    while (4 * l < states) l *= 2;
    return l;
}

// Tokens a piece of a scan split along time; 0 = not split.
//
// Not split, a block (4 warps) takes its channels through a whole sequence: at best
// kFull clocks a token of SM time, kAlone when it has the SM to itself. Split, all SMs
// work, for the price of computing every exponential twice (kState more clocks a
// token) and of two more launches. The longest of n packed sequences, whose lengths
// the host does not know, is taken as (1 + ln n) average ones, as random cuts make it.
//
// bf16, 16 states, split against whole: 512 x 256 19 and 41 us, 2048 x 256 25 and 154,
// 4096 x 2048 133 and 306, 16384 x 4096 887 and 1210; 4 sequences of 2048 x 2048, which
// the rule leaves whole, 234 and 193.
constexpr double kAlone = 150, kFull = 80, kState = 55, kLaunches = 15000;
int64_t piece_tokens(const pe_scan_args* a) {
    const int64_t ch = kThreads / lanes_for(a->states), dg = a->channels / a->groups;
    const int64_t tiles = a->groups * ceil_div(dg, ch);
    if (a->nseq < 1 || a->nseq > 65535 || a->tokens < 256) return 0;
    const double sms = num_sms(), total = (double)a->tokens * (a->cu ? 1 : a->nseq) * tiles;
    double longest = (double)a->tokens;
    if (a->cu) longest = min(longest, longest / a->nseq * (1.0 + log((double)a->nseq)));
    const double whole = max(longest * kAlone, total / sms * kFull);
    const double split = total / sms * (kFull + kState) + kLaunches;
    if (split >= whole) return 0;
    // four blocks an SM, one wave of them: pieces are rounded up
    const int64_t slots = 4 * num_sms(), rows = a->cu ? 1 : a->nseq;
    const int64_t pieces = max((int64_t)1, slots / (rows * tiles) - (a->cu ? a->nseq : 0));
    return max((int64_t)KCK, ceil_div(ceil_div(a->tokens, pieces), KCK) * KCK);
}

template <typename T, int LPC, bool FAST>
int scan_launch(const ScanP<T>& p, unsigned grid, bool split, cudaStream_t s) {
    if (split) {
        if (int rc = launch(scan_fwd<T, LPC, true, FAST>, p, grid, sizeof(FwdSmem<T, LPC, true>), s)) return rc;
        const dim3 blocks((unsigned)ceil_div((int64_t)p.D * p.N, kThreads), (unsigned)p.seqs.nseq);
        scan_carry<T><<<blocks, kThreads, 0, s>>>(p);
        count_launch();
        if (cudaGetLastError() != cudaSuccess) return PE_ERR_CUDA;
    }
    return launch(scan_fwd<T, LPC, false, FAST>, p, grid, sizeof(FwdSmem<T, LPC, false>), s);
}

template <typename T, int LPC>
int scan_run(const pe_scan_args* a, cudaStream_t s) {
    ScanP<T> p = scan_params<T>(a, kThreads / LPC, 4 * LPC);
    const int64_t piece = piece_tokens(a);
    if (piece) {
        p.split(piece);
        const int64_t n = piece_count(p.seqs, piece);
        p.hloc = (float*)a->ws;
        p.dtsum = p.hloc + n * p.D * p.N;
    }
    unsigned grid;
    if (int rc = grid_of(piece_count(p.seqs, p.piece) * p.G * p.ntile, &grid)) return rc;
    if constexpr (Feeder<T, LPC, false>::POSSIBLE)
        if (p.fast) return scan_launch<T, LPC, true>(p, grid, piece, s);
    return scan_launch<T, LPC, false>(p, grid, piece, s);
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

template <typename T>
int scan_type(const pe_scan_args* a, cudaStream_t s) {
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
    const int64_t tiles = ceil_div(p.D, kThreads / LPC);
    // eight states at once: 32 bytes of the state, 16-byte loads of A, B and C
    const int e = 16 / (int)sizeof(T);
    const bool vec = p.N % 8 == 0 && (uintptr_t)p.state % 32 == 0 &&
                     ((uintptr_t)p.A | (uintptr_t)p.B | (uintptr_t)p.C) % 16 == 0 &&
                     (p.B_sb % e | p.B_sg % e | p.C_sb % e | p.C_sg % e) == 0;
    // two requests a thread once that still gives every SM its 16 blocks: fp16, 16 states, two
    // against one, 256 x 4096 22.8 and 25.0 us, 512 x 4096 51.6 and 56.0; 64 x 2048, below the
    // rule, 6.4 both
    const bool two = tiles * a->batch >= 32ll * num_sms();
    const dim3 grid((unsigned)tiles, (unsigned)(two ? ceil_div(a->batch, 2) : a->batch));
    if (vec && two)
        scan_step<T, LPC, 2, true><<<grid, kThreads, 0, s>>>(p);
    else if (two)
        scan_step<T, LPC, 2, false><<<grid, kThreads, 0, s>>>(p);
    else if (vec)
        scan_step<T, LPC, 1, true><<<grid, kThreads, 0, s>>>(p);
    else
        scan_step<T, LPC, 1, false><<<grid, kThreads, 0, s>>>(p);
    count_launch();
    return cudaGetLastError() == cudaSuccess ? PE_OK : PE_ERR_CUDA;
}
template <typename T>
int step_type(const pe_scan_step_args* a, cudaStream_t s) {
    if (a->states <= 8) return step_run<T, 1>(a, s);
    if (a->states <= 16) return step_run<T, 2>(a, s);
    if (a->states <= 32) return step_run<T, 4>(a, s);
    if (a->states <= 64) return step_run<T, 8>(a, s);
    return step_run<T, 16>(a, s);
}

int scan_any(const pe_scan_args* a, cudaStream_t s) { PE_TYPES(scan_type, a->dtype, a, s) }
int step_any(const pe_scan_step_args* a, cudaStream_t s) { PE_TYPES(step_type, a->dtype, a, s) }

}  // namespace

int64_t scan_ckpt_floats(int64_t tokens, int64_t nseq, int64_t packed, int64_t channels, int64_t states) {
    const int32_t none = 0;
    return piece_count(Seqs{packed ? &none : nullptr, tokens, (int32_t)nseq}, KCK) * channels * states;
}

int64_t scan_ws_bytes(const pe_scan_args* a) {
    if (check_scan(a) != PE_OK) return 0;
    const int64_t piece = piece_tokens(a);
    return piece ? piece_count(seqs_of(a), piece) * (a->channels * a->states + a->channels) * 4 : 0;
}

int selective_scan(const pe_scan_args* a, cudaStream_t s) {
    if (int rc = check_scan(a)) return rc;
    if (a->nseq == 0) return PE_OK;
    if (a->tokens && !a->out) return PE_ERR_INVALID;
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

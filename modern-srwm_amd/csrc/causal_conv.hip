// Short causal depthwise convolution over whole sequences and for one token:
//     out_t = f(bias + sum_j w[j] x_{t-W+1+j}),   f = silu or the identity
// Inputs before the first step come from the carried rows, inputs before a reset count as zero.
#include "common.h"
#include "gates.h"
#include "vec_io.h"

namespace fw {
namespace {

// A workgroup: 32 vectors of channels x 8 runs of ST steps; those beside each other along the channels follow one another,
// so that whole rows are read at a time (1 x 65536 steps x 2048 channels, bf16: forward 104 us, backward 212; neighbours
// along the steps first 146 and 280).  Vectors of 8 bytes and 8 steps in the forward (4 x 2048 x 2048: 16.0 us; 16 steps 17.2,
// 16 bytes 18.8: with fewer waves all of them load, compute and store at the same time), of two channels in the backward
// (one 33.9, two 31.3, four 35.0 us with neighbours along the steps first).
constexpr int kConvLanes = 32, kConvRuns = 8, kConvFwdSteps = 8;
// The backward's runs are of 16 steps, of 8 where those would be fewer than kConvWaves waves (16 / 8 steps: 4 x 2048 x 2048 29.3
// / 31.9 us; 2 x 1024 steps x 1024 channels 9.6 / 8.2; 32 x 100 x 256, fp32, 11.6 / 8.9).
constexpr int kConvWaves = 4096;

template <int V>
__device__ __forceinline__ void zero(float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.f;
}
template <typename T, int V>
__device__ __forceinline__ void widen(const Pack<T, V> &r, float (&v)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (float)r.v[i];
}

// A thread's run: ST steps of V channels of one sequence.
struct ConvPlace {
    int64_t d, t0;
    int n, h, e, Ln;
};
// A workgroup's number among the N * runs * cols of a launch, which may take more than one row of the grid (the last one then
// holds workgroups behind them: n >= N).
constexpr int64_t kConvRow = 1 << 23;   // workgroups along x: 256 threads each must stay below 2^32
__device__ __forceinline__ unsigned conv_group() { return blockIdx.y * (unsigned)kConvRow + blockIdx.x; }
template <int V, int ST>
__device__ __forceinline__ ConvPlace conv_place(const ConvParams &p, int runs, unsigned cols) {
    ConvPlace c;
    c.d = ((int64_t)(conv_group() % cols) * kConvLanes + threadIdx.x) * V;
    const unsigned part = conv_group() / cols;
    c.n = part / runs;
    c.t0 = ((int64_t)(part % runs) * kConvRuns + threadIdx.y) * ST;
    c.h = c.d / p.E, c.e = c.d % p.E;
    c.Ln = p.lengths && c.n < p.N ? min(max(p.lengths[c.n], 0), p.L) : p.L;
    return c;
}

// Rows t, t + 1, ... of a run as they lie in memory, all loads in flight at once.  Rows in front of the first step are
// the carried ones (zeros without them), rows behind the sequence's end zeros.
template <typename T, int W, int V, int R>
__device__ __forceinline__ void load_rows(const T *x, int64_t stride, const T *state, int E, int64_t t, int Ln, Pack<T, V> (&r)[R]) {
    if (t >= 0 && t + R <= Ln) {
#pragma unroll
        for (int j = 0; j < R; ++j) r[j] = *reinterpret_cast<const Pack<T, V> *>(x + (t + j) * stride);
    } else {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            r[j] = Pack<T, V>{};
            if (t + j >= 0) {
                if (t + j < Ln) r[j] = *reinterpret_cast<const Pack<T, V> *>(x + (t + j) * stride);
            } else if (state && t + j >= -(W - 1)) {
                r[j] = *reinterpret_cast<const Pack<T, V> *>(state + (W - 1 + t + j) * E);
            }
        }
    }
}
// bit j: a reset in front of step t + j
template <int R>
__device__ __forceinline__ uint32_t load_resets(const float *keep, int64_t t, int Ln) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < R; ++j)
        if (t + j >= 0 && t + j < Ln && is_reset(keep[t + j])) m |= 1u << j;
    return m;
}

// Memory-bound: every input and output once, plus W - 1 rows of the run in front (from the caches).  All of a run's rows
// are asked for before the first is used (4 x 2048 steps x 2048 channels, 4 taps, bf16: 67 MB in 15.3 us, 4.4 TB/s; 1 x 65536
// steps 537 MB in 101 us, 5.3 TB/s).
template <typename T, int W, int V, int ST, bool KEEP>
__global__ __launch_bounds__(kConvLanes *kConvRuns) void conv_fwd_kernel(ConvParams p, int runs, unsigned cols) {
    constexpr int R = ST + W - 1;
    const ConvPlace c = conv_place<V, ST>(p, runs, cols);
    if (c.n >= p.N || c.d >= (int64_t)p.H * p.E || (c.t0 >= p.L && c.t0 > 0)) return;
    const T *x = (const T *)p.x + c.n * p.xs.n + c.h * p.xs.h + c.e;
    const int64_t srow = ((int64_t)c.n * p.H + c.h) * (W - 1) * p.E + c.e;
    T *out = (T *)p.out + c.n * p.os.n + c.h * p.os.h + c.e + c.t0 * p.os.l;
    const int Ln = c.Ln;

    Pack<T, V> raw[R];
    load_rows<T, W, V, R>(x, p.xs.l, p.state ? (const T *)p.state + srow : nullptr, p.E, c.t0 - (W - 1), Ln, raw);
    uint32_t resets = 0;
    if constexpr (KEEP) resets = load_resets<R>(p.keep + (int64_t)c.n * p.L, c.t0 - (W - 1), Ln);
    float w[W][V], bias[V], win[W][V];   // win: the last W inputs, the newest last
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int j = 0; j < W; ++j) w[j][i] = p.weight[(c.d + i) * W + j];
        bias[i] = p.bias ? p.bias[c.d + i] : 0.f;
    }
    // the row's last step is in this run (or the row is empty and this is its first run): it hands the carried rows on
    const bool ends = Ln > 0 ? (c.t0 < Ln && Ln <= c.t0 + ST) : c.t0 == 0;
    const int at_end = (int)(Ln - c.t0);
    T *last = (T *)p.last + srow;
#pragma unroll
    for (int j = 0; j < W; ++j) zero<V>(win[j]);
#pragma unroll
    for (int k = 0; k <= R; ++k) {
        // k rows are in the window, step t0 + k - W the newest of them
        if (k >= W - 1 && ends && k - (W - 1) == at_end) {
#pragma unroll
            for (int j = 0; j + 1 < W; ++j) store_vec<V>(last + (int64_t)j * p.E, win[j + 1]);
        }
        if (k == R) break;
        const bool reset = KEEP && (resets >> k & 1);
#pragma unroll
        for (int j = 0; j + 1 < W; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) win[j][i] = reset ? 0.f : win[j + 1][i];
        widen<T, V>(raw[k], win[W - 1]);
        if (k >= W - 1) {
            const int s = k - (W - 1);
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                o[i] = bias[i];
#pragma unroll
                for (int j = 0; j < W; ++j) o[i] = fmaf(w[j][i], win[j][i], o[i]);
                if (p.silu) o[i] *= sigmoid(o[i]);
                if (s >= at_end) o[i] = 0.f;
            }
            if (c.t0 + s < p.L) store_vec<V>(out + s * p.os.l, o);
        }
    }
}

// gx_t = sum_j w[W-1-j] gp_{t+j} with gp = g f'(pre): a run walks its steps and the W - 1 behind them, carrying the
// gradients of the last W inputs, each complete when the window leaves it.  Between memory and arithmetic (vector
// instructions 76 - 80 % of the time, the sigmoid's and 2 W products per step and channel): same sizes 101 MB in 28 us, 3.6 TB/s,
// 1 x 65536 steps 805 MB in 192 us, 4.2 TB/s.
template <typename T, int W, int V, int ST, bool KEEP>
__global__ __launch_bounds__(kConvLanes *kConvRuns) void conv_bwd_kernel(ConvBwdParams b, int runs, unsigned cols) {
    constexpr int RX = ST + 2 * (W - 1), RG = ST + W - 1;
    const ConvParams &p = b.f;
    const int64_t D = (int64_t)p.H * p.E;
    __shared__ float red[kConvRuns][kConvLanes][V];
    const ConvPlace c = conv_place<V, ST>(p, runs, cols);
    if (c.n >= p.N) return;   // the whole workgroup
    float gw[W + 1][V];
#pragma unroll
    for (int j = 0; j <= W; ++j) zero<V>(gw[j]);
    if (c.d < D && c.t0 < p.L) {
        const int Ln = c.Ln;
        const T *x = (const T *)p.x + c.n * p.xs.n + c.h * p.xs.h + c.e;
        const T *go = (const T *)b.go + c.n * b.gos.n + c.h * b.gos.h + c.e;
        T *gx = (T *)b.gx + c.n * b.gxs.n + c.h * b.gxs.h + c.e;
        const int64_t srow = ((int64_t)c.n * p.H + c.h) * (W - 1) * p.E + c.e;
        const T *glast = b.glast ? (const T *)b.glast + srow : nullptr;
        T *gstate = b.gstate && c.t0 == 0 ? (T *)b.gstate + srow : nullptr;

        Pack<T, V> rx[RX], rg[RG];
        load_rows<T, W, V, RX>(x, p.xs.l, p.state ? (const T *)p.state + srow : nullptr, p.E, c.t0 - (W - 1), Ln, rx);
        load_rows<T, W, V, RG>(go, b.gos.l, nullptr, p.E, c.t0, Ln, rg);
        uint32_t resets = 0;
        if constexpr (KEEP) resets = load_resets<RX>(p.keep + (int64_t)c.n * p.L, c.t0 - (W - 1), Ln);
        float w[W][V], bias[V], win[W][V], acc[W][V];   // acc[j]: gradient of the input j steps back
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
            for (int j = 0; j < W; ++j) w[j][i] = p.weight[(c.d + i) * W + j];
            bias[i] = p.bias ? p.bias[c.d + i] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < W; ++j) zero<V>(win[j]), zero<V>(acc[j]);
        int since = W;   // steps since the last reset, at most W
#pragma unroll
        for (int k = 0; k < RX; ++k) {
            const int s = k - (W - 1);              // step t0 + s
            const int64_t t = c.t0 + s;
            const bool reset = KEEP && (resets >> k & 1);
            if constexpr (KEEP) since = reset ? 0 : min(since + 1, W);
#pragma unroll
            for (int j = 0; j + 1 < W; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) win[j][i] = reset ? 0.f : win[j + 1][i];
            widen<T, V>(rx[k], win[W - 1]);
            if (s < 0) continue;
#pragma unroll
            for (int j = W - 1; j > 0; --j)
#pragma unroll
                for (int i = 0; i < V; ++i) acc[j][i] = acc[j - 1][i];
            zero<V>(acc[0]);
            // rows behind the end are zeros in rg, so that nothing of them is added
            float g[V];
            widen<T, V>(rg[s < 0 ? 0 : s], g);
            if (p.silu) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float o = bias[i];
#pragma unroll
                    for (int j = 0; j < W; ++j) o = fmaf(w[j][i], win[j][i], o);
                    const float q = sigmoid(o);
                    g[i] *= q * fmaf(o, 1.f - q, 1.f);
                    if (t >= Ln) g[i] = 0.f;
                }
            }
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (!KEEP || j <= since)
#pragma unroll
                    for (int i = 0; i < V; ++i) acc[j][i] = fmaf(w[W - 1 - j][i], g[i], acc[j][i]);
            if (s < ST) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
#pragma unroll
                    for (int j = 0; j < W; ++j) gw[j][i] = fmaf(g[i], win[j][i], gw[j][i]);
                    gw[W][i] += g[i];
                }
            }
            if (t == Ln && glast) {   // one step behind the end: the carried rows are the inputs 1 .. W-1 steps back
#pragma unroll
                for (int j = 1; j < W; ++j)
                    if (!KEEP || j <= since) {
                        float gl[V];
                        load_vec<V>(glast + (int64_t)(W - 1 - j) * p.E, gl);
#pragma unroll
                        for (int i = 0; i < V; ++i) acc[j][i] += gl[i];
                    }
            }
            const int done = s - (W - 1);   // the input that leaves the window, t0 + done
            if (done >= 0) {
                if (c.t0 + done < p.L) store_vec<V>(gx + (c.t0 + done) * b.gxs.l, acc[W - 1]);
            } else if (gstate) {
                store_vec<V>(gstate + (int64_t)(W - 1 + done) * p.E, acc[W - 1]);
            }
        }
    }
    float *part = b.part + (int64_t)(conv_group() / cols) * (W + 1) * D;
#pragma unroll
    for (int j = 0; j <= W; ++j) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) red[threadIdx.y][threadIdx.x][i] = gw[j][i];
        __syncthreads();
        for (int i = threadIdx.y * kConvLanes + threadIdx.x; i < kConvLanes * V; i += kConvLanes * kConvRuns) {
            const int64_t at = (int64_t)(conv_group() % cols) * kConvLanes * V + i;
            float v = 0.f;
#pragma unroll
            for (int r = 0; r < kConvRuns; ++r) v += red[r][i / V][i % V];
            if (at < D) part[j * D + at] = v;
        }
    }
}

// Sums the runs' shares of gweight and gbias: 32 columns of one tap per workgroup, 8 threads over the runs of each.
__global__ __launch_bounds__(256) void conv_join_kernel(const float *part, float *gweight, float *gbias, int64_t D, int W,
                                                        int parts) {
    __shared__ float sums[8][32];
    const int c = threadIdx.x % 32, r = threadIdx.x / 32, j = blockIdx.y;
    const int64_t d = (int64_t)blockIdx.x * 32 + c;
    if (j == W && !gbias) return;
    float v = 0.f;
    if (d < D) {
#pragma unroll 8
        for (int k = r; k < parts; k += 8) v += part[((int64_t)k * (W + 1) + j) * D + d];
    }
    sums[r][c] = v;
    __syncthreads();
    if (r == 0 && d < D) {
        v = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) v += sums[k][c];
        if (j < W) gweight[d * W + j] = v;
        else gbias[d] = v;
    }
}

// One token: V channels of one row per thread.  Latency: one row of 2048 channels 3.9 us, 256 rows (9 MB) 6.9 us.
template <typename T, int W, int V>
__global__ __launch_bounds__(256) void conv_step_kernel(ConvParams p) {
    const int64_t D = (int64_t)p.H * p.E;
    const int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t per = D / V;
    if (i0 >= p.N * per) return;
    const int64_t n = i0 / per, d = i0 % per * V;
    const int h = d / p.E, e = d % p.E;
    T *state = (T *)p.last + (n * p.H + h) * (W - 1) * p.E + e;
    float win[W][V], o[V];
    const bool reset = p.keep && is_reset(p.keep[n]);
#pragma unroll
    for (int j = 0; j + 1 < W; ++j) {
        load_vec<V>(state + (int64_t)j * p.E, win[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) win[j][i] = reset ? 0.f : win[j][i];
    }
    load_vec<V>((const T *)p.x + n * p.xs.n + h * p.xs.h + e, win[W - 1]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        o[i] = p.bias ? p.bias[d + i] : 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) o[i] = fmaf(p.weight[(d + i) * W + j], win[j][i], o[i]);
        if (p.silu) o[i] *= sigmoid(o[i]);
    }
    store_vec<V>((T *)p.out + n * p.os.n + h * p.os.h + e, o);
#pragma unroll
    for (int j = 0; j + 1 < W; ++j) store_vec<V>(state + (int64_t)j * p.E, win[j + 1]);
}

// Rows that can be read V elements at a time: E and every stride a multiple of V, bases aligned.
bool vec_ok(const void *q, int64_t bytes) { return ((uintptr_t)q & (bytes - 1)) == 0; }
template <typename T, int V>
bool rows_ok(const void *q, const Strided3 &s) {
    return vec_ok(q, sizeof(T) * V) && s.n % V == 0 && s.h % V == 0 && s.l % V == 0;
}
template <typename T, int V>
bool conv_vec(const ConvParams &p) {
    return p.E % V == 0 && rows_ok<T, V>(p.x, p.xs) && rows_ok<T, V>(p.out, p.os) && vec_ok(p.state, sizeof(T) * V) &&
           vec_ok(p.last, sizeof(T) * V);
}

int conv_runs(int L, int steps) { return (L + kConvRuns * steps - 1) / (kConvRuns * steps); }
int conv_bwd_steps(int N, int H, int L, int E) {
    const int64_t waves = (int64_t)N * conv_runs(L, 16) * (((int64_t)H * E + 63) / 64) * 4;
    return waves < kConvWaves ? 8 : 16;
}
// A launch over runs and columns of `v` channels a lane; false: more workgroups than it takes.
struct ConvGrid {
    unsigned cols;
    int64_t groups;
    ConvGrid(const ConvParams &p, int runs, int v)
        : cols((unsigned)(((int64_t)p.H * p.E / v + kConvLanes - 1) / kConvLanes)), groups((int64_t)p.N * runs * cols) {}
    bool fits() const { return groups < ((int64_t)1 << 32) - kConvRow; }
    dim3 grid() const {
        return groups <= kConvRow ? dim3((unsigned)groups) : dim3((unsigned)kConvRow, (unsigned)((groups + kConvRow - 1) / kConvRow));
    }
};

template <typename T, int W, int V>
int fwd_as(const ConvParams &p, hipStream_t s) {
    constexpr int ST = kConvFwdSteps;
    const int runs = conv_runs(p.L, ST);
    const ConvGrid g(p, runs, V);
    if (!g.fits()) return -1;
    const dim3 block(kConvLanes, kConvRuns);
    if (p.keep) conv_fwd_kernel<T, W, V, ST, true><<<g.grid(), block, 0, s>>>(p, runs, g.cols);
    else conv_fwd_kernel<T, W, V, ST, false><<<g.grid(), block, 0, s>>>(p, runs, g.cols);
    return (int)hipGetLastError();
}
template <typename T, int W>
int fwd(const ConvParams &p, hipStream_t s) {
    constexpr int V = 8 / sizeof(T);
    return conv_vec<T, V>(p) ? fwd_as<T, W, V>(p, s) : fwd_as<T, W, 1>(p, s);
}
template <typename T, int W, int V, int ST>
int bwd_as(const ConvBwdParams &b, hipStream_t s) {
    const ConvParams &p = b.f;
    const int runs = conv_runs(p.L, ST);
    const ConvGrid g(p, runs, V);
    if (!g.fits()) return -1;
    const dim3 block(kConvLanes, kConvRuns);
    if (p.keep) conv_bwd_kernel<T, W, V, ST, true><<<g.grid(), block, 0, s>>>(b, runs, g.cols);
    else conv_bwd_kernel<T, W, V, ST, false><<<g.grid(), block, 0, s>>>(b, runs, g.cols);
    const int r = (int)hipGetLastError();
    if (r) return r;
    const int64_t D = (int64_t)p.H * p.E;
    conv_join_kernel<<<dim3((unsigned)((D + 31) / 32), W + 1), 256, 0, s>>>(b.part, b.gweight, b.gbias, D, W, p.N * runs);
    return (int)hipGetLastError();
}
template <typename T, int W>
int bwd(const ConvBwdParams &b, hipStream_t s) {
    constexpr int V = 2;
    const ConvParams &p = b.f;
    const bool vec = p.E % V == 0 && rows_ok<T, V>(p.x, p.xs) && rows_ok<T, V>(b.go, b.gos) && rows_ok<T, V>(b.gx, b.gxs) &&
                     vec_ok(p.state, sizeof(T) * V) && vec_ok(b.glast, sizeof(T) * V) && vec_ok(b.gstate, sizeof(T) * V);
    if (conv_bwd_steps(p.N, p.H, p.L, p.E) == 8) return vec ? bwd_as<T, W, V, 8>(b, s) : bwd_as<T, W, 1, 8>(b, s);
    return vec ? bwd_as<T, W, V, 16>(b, s) : bwd_as<T, W, 1, 16>(b, s);
}
template <typename T, int W>
int step(const ConvParams &p, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int64_t D = (int64_t)p.H * p.E;
    auto grid = [&](int v) { return (unsigned)((p.N * (D / v) + 255) / 256); };
    if (conv_vec<T, V>(p)) conv_step_kernel<T, W, V><<<grid(V), 256, 0, s>>>(p);
    else conv_step_kernel<T, W, 1><<<grid(1), 256, 0, s>>>(p);
    return (int)hipGetLastError();
}

}  // namespace

int64_t conv_parts(int N, int H, int L, int E) { return (int64_t)N * conv_runs(L, conv_bwd_steps(N, H, L, E)); }

#define FW_BY_TAPS(FN, W, P)                                        \
    switch (W) {                                                    \
        case 2: return bf16 ? FN<__bf16, 2>(P, s) : FN<float, 2>(P, s); \
        case 3: return bf16 ? FN<__bf16, 3>(P, s) : FN<float, 3>(P, s); \
        case 4: return bf16 ? FN<__bf16, 4>(P, s) : FN<float, 4>(P, s); \
    }                                                               \
    return -1;

int launch_conv_fwd(const ConvParams &p, bool bf16, hipStream_t s) { FW_BY_TAPS(fwd, p.W, p) }
int launch_conv_bwd(const ConvBwdParams &b, bool bf16, hipStream_t s) { FW_BY_TAPS(bwd, b.f.W, b) }
int launch_conv_step(const ConvParams &p, bool bf16, hipStream_t s) { FW_BY_TAPS(step, p.W, p) }

}  // namespace fw

// Selective scan, forward over whole sequences, and its single-token form.
#include "selective_scan.h"

namespace fw {
namespace {

// One workgroup carries 64 channels of one sequence through all its steps, 16 at a time.
template <typename T, int SPL, bool KEEP>
__global__ __launch_bounds__(kScanThreads) void scan_fwd_kernel(ScanParams p) {
    constexpr int SP = 4 * SPL;
    __shared__ float bc[2][2][kScanBlock][SP];   // [buffer][B | C][step][state]
    const int n = blockIdx.x % p.N, tile = blockIdx.x / p.N, g = blockIdx.y;
    const ScanLane w = scan_lane(p.H, p.E, p.G, tile, g);
    const int S = p.S, D = p.H * p.E;
    int Ln = p.L;
    if (p.lengths) Ln = min(max(p.lengths[n], 0), p.L);

    const T *u = (const T *)p.u + n * p.us.n + w.h * p.us.h + w.e;
    const T *dl = (const T *)p.delta + n * p.ds.n + w.h * p.ds.h + w.e;
    const T *z = p.z ? (const T *)p.z + n * p.zs.n + w.h * p.zs.h + w.e : nullptr;
    T *out = (T *)p.out + n * p.os.n + w.h * p.os.h + w.e;
    const T *Bp = (const T *)p.B + n * p.Bs.n + g * p.Bs.h;
    const T *Cp = (const T *)p.C + n * p.Cs.n + g * p.Cs.h;
    const float bias = p.bias ? p.bias[w.d] : 0.f, Dc = p.D ? p.D[w.d] : 0.f;

    float A2[SPL], h[SPL];
    load_states<SPL>(p.A + (int64_t)w.d * S, S, w.q, A2);
#pragma unroll
    for (int s = 0; s < SPL; ++s) A2[s] *= kLog2e, h[s] = 0.f;
    if (p.state) load_states<SPL>(p.state + ((int64_t)n * D + w.d) * S, S, w.q, h);

    const int nblk = (Ln + kScanBlock - 1) / kScanBlock;
    const int nsave = (p.L + kScanBlock - 1) / kScanBlock;
    for (int blk = 0; blk < nblk; ++blk) {
        const int t0 = blk * kScanBlock, buf = blk & 1;
        for (int i = threadIdx.x; i < 2 * kScanBlock * SP; i += kScanThreads) {
            const int s = i % SP, t = i / SP % kScanBlock, c = i / (SP * kScanBlock);
            float v = 0.f;
            if (s < S && t0 + t < Ln) v = c ? io_load(Cp + (t0 + t) * p.Cs.l + s) : io_load(Bp + (t0 + t) * p.Bs.l + s);
            bc[buf][c][t][s] = v;
        }
        unsigned resets = 0;
        if constexpr (KEEP) {
            const int t = t0 + (w.lane & 15);
            resets = (unsigned)__ballot(w.lane < 16 && t < Ln && is_reset(p.keep[(int64_t)n * p.L + min(t, p.L - 1)]));
        }
        __syncthreads();
        if (p.saved && w.on)
            store_states<SPL>(p.saved + (((int64_t)n * nsave + blk) * D + w.d) * S, S, w.q, h);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t t = t0 + 4 * i + w.q;
            const bool in = t < Ln;
            float uu = 0.f, dt = 0.f, zz = 0.f;
            if (in) {
                uu = io_load(u + t * p.us.l);
                dt = io_load(dl + t * p.ds.l) + bias;
                if (z) zz = io_load(z + t * p.zs.l);
                float sig;
                if (p.softplus) dt = softplus_sig(dt, sig);
            }
            const float du = dt * uu;
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float dtj = quad_lane(dt, j), duj = quad_lane(du, j);
                const float *Bt = &bc[buf][0][4 * i + j][w.q * SPL], *Ct = &bc[buf][1][4 * i + j][w.q * SPL];
                y[j] = 0.f;
                const bool reset = KEEP && (resets >> (4 * i + j) & 1);
#pragma unroll
                for (int s = 0; s < SPL; ++s) {
                    if constexpr (KEEP) h[s] = reset ? 0.f : h[s];
                    h[s] = fmaf(__builtin_amdgcn_exp2f(dtj * A2[s]), h[s], duj * Bt[s]);
                    y[j] = fmaf(Ct[s], h[s], y[j]);
                }
            }
            float o = quad_sum_scatter(y[0], y[1], y[2], y[3], w.lane) + Dc * uu;
            if (z) o *= zz * sigmoid(zz);
            if (in && w.on) io_store(out + t * p.os.l, o);
        }
    }
    if (w.on) {
        for (int64_t t = Ln + w.q; t < p.L; t += 4) io_store(out + t * p.os.l, 0.f);
        store_states<SPL>(p.last + ((int64_t)n * D + w.d) * S, S, w.q, h);
    }
}

template <typename T, int SPL>
int launch_fwd(const ScanParams &p, hipStream_t s) {
    const int Dg = p.H / p.G * p.E;
    const dim3 grid((Dg + kScanTile - 1) / kScanTile * p.N, p.G);
    if (p.keep) scan_fwd_kernel<T, SPL, true><<<grid, kScanThreads, 0, s>>>(p);
    else scan_fwd_kernel<T, SPL, false><<<grid, kScanThreads, 0, s>>>(p);
    return (int)hipGetLastError();
}

// One token: every lane updates SPL states of a channel in place.
template <typename T, int SPL>
__global__ __launch_bounds__(kScanThreads) void scan_step_kernel(ScanParams p) {
    const int n = blockIdx.x % p.N, tile = blockIdx.x / p.N, g = blockIdx.y;
    const ScanLane w = scan_lane(p.H, p.E, p.G, tile, g);
    if (!w.on) return;
    const int S = p.S, D = p.H * p.E;
    const float uu = io_load((const T *)p.u + n * p.us.n + w.h * p.us.h + w.e);
    float dt = io_load((const T *)p.delta + n * p.ds.n + w.h * p.ds.h + w.e) + (p.bias ? p.bias[w.d] : 0.f), sig;
    const T *Bp = (const T *)p.B + n * p.Bs.n + g * p.Bs.h, *Cp = (const T *)p.C + n * p.Cs.n + g * p.Cs.h;
    if (p.softplus) dt = softplus_sig(dt, sig);
    float *row = p.last + ((int64_t)n * D + w.d) * S;
    float h[SPL], A[SPL];
    load_states<SPL>(row, S, w.q, h);
    load_states<SPL>(p.A + (int64_t)w.d * S, S, w.q, A);
    const bool reset = p.keep && is_reset(p.keep[n]);
    float y = 0.f;
#pragma unroll
    for (int s = 0; s < SPL; ++s) {
        const int k = w.q * SPL + s;
        const float b = k < S ? io_load(Bp + k) : 0.f, c = k < S ? io_load(Cp + k) : 0.f;
        h[s] = fmaf(__builtin_amdgcn_exp2f(dt * (A[s] * kLog2e)), reset ? 0.f : h[s], dt * uu * b);
        y = fmaf(c, h[s], y);
    }
    store_states<SPL>(row, S, w.q, h);
    y = group_sum<4>(y);
    if (w.q == 0) {
        y += (p.D ? p.D[w.d] : 0.f) * uu;
        if (p.z) {
            const float zz = io_load((const T *)p.z + n * p.zs.n + w.h * p.zs.h + w.e);
            y *= zz * sigmoid(zz);
        }
        io_store((T *)p.out + n * p.os.n + w.h * p.os.h + w.e, y);
    }
}

template <typename T, int SPL>
int launch_step(const ScanParams &p, hipStream_t s) {
    const int Dg = p.H / p.G * p.E;
    scan_step_kernel<T, SPL><<<dim3((Dg + kScanTile - 1) / kScanTile * p.N, p.G), kScanThreads, 0, s>>>(p);
    return (int)hipGetLastError();
}

}  // namespace

#define FW_BY_STATES(FN)                                           \
    if (p.S <= 8) return bf16 ? FN<__bf16, 2>(p, s) : FN<float, 2>(p, s);   \
    if (p.S <= 16) return bf16 ? FN<__bf16, 4>(p, s) : FN<float, 4>(p, s);  \
    if (p.S <= 32) return bf16 ? FN<__bf16, 8>(p, s) : FN<float, 8>(p, s);  \
    return bf16 ? FN<__bf16, 16>(p, s) : FN<float, 16>(p, s);

int launch_scan_fwd(const ScanParams &p, bool bf16, hipStream_t s) { FW_BY_STATES(launch_fwd) }
int launch_scan_step(const ScanParams &p, bool bf16, hipStream_t s) { FW_BY_STATES(launch_step) }

}  // namespace fw

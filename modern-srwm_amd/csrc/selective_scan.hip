// Selective scan, forward over whole sequences, and its single-token form.
#include "selective_scan.h"

namespace fw {
namespace {

// Runs 64 channels of one sequence through one segment of its steps, 16 steps at a time.
// LOCAL: from a zero state, for nothing but the segment's last state and its product of decays.  Otherwise the state
// comes from the call's state and the segments in front of this one, and the outputs are formed.
// The inputs of a block are fetched while the block before is computed.
// Bound by the number of vector instructions (busy 86 - 90 % of the time, LDS 4 %): per state and step a multiplication, an
// exponential (twice the cycles of the others) and three more are needed, 5 instructions in 6 issue slots of 4 cycles a wave;
// 8.4 in 9.4 are issued with outputs (softplus, gate, conversions, hand-overs between lanes), 5.7 in 6.7 without.  4 x 2048 steps x 2048 channels x 16
// states, bf16: 56 us (LOCAL) + 83 us, 212 MB read and written by the second; two rows of 12 001 and 8 001 steps: 132 + 195.
// 16 lanes to a channel, which needs no segments, took 667 us for the latter beside 148 + 217 (short runs).
template <typename T, int SPL, bool KEEP, bool LOCAL, typename OFF>
__global__ __launch_bounds__(kScanThreads) void scan_fwd_kernel(ScanParams p) {
    constexpr int SP = 4 * SPL;
    using Bc = ScanBc<T, SPL>;
    __shared__ float bc[2][2][kScanBlock][SP];   // [buffer][B | C][step][state]
    const ScanRun run = scan_run(p, blockIdx.x % p.N, blockIdx.z);
    if (LOCAL && (!run.used || run.seg == run.count - 1)) return;   // the whole workgroup; a row's last result is not needed
    const ScanLane w = scan_lane(p, run.n);
    const int S = p.S, D = p.H * p.E, tbeg = run.tbeg, tend = run.tend;

    ScanRows<const T, OFF> u(p.u, p.us, w, tbeg), dl(p.delta, p.ds, w, tbeg), z(p.z, p.zs, w, tbeg);
    ScanRows<T, OFF> out(p.out, p.os, w, tbeg);
    Bc rows(p, w, tbeg);
    const bool gate = !LOCAL && p.z != nullptr;
    const float bias = p.bias ? p.bias[w.d] : 0.f, Dc = p.D ? p.D[w.d] : 0.f;
    const int64_t states = (int64_t)w.d * S;   // this channel's row in [H*E, S]

    float A2[SPL], h[SPL], total = 0.f;
    load_decays<SPL>(p.A + states, S, w.q, A2);
#pragma unroll
    for (int s = 0; s < SPL; ++s) h[s] = 0.f;
    bool alive = true;   // no reset in this segment so far

    T ru[4], rd[4], rz[4], rb[Bc::kEach], rc[Bc::kEach];   // the next block as it lies in memory
    float rk = 1.f;
    // n: steps from the block's first one to the end (more than none); lanes behind it read the last one
    auto fetch = [&](int t0, int n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool full = n >= kScanBlock;
            const int at = full ? i : 0, k = full ? w.q : min(4 * i + w.q, n - 1);
            ru[i] = *u.at(at, k);
            rd[i] = *dl.at(at, k);
            if (gate) rz[i] = *z.at(at, k);
        }
        rows.fetch(rb, rc, n, !LOCAL);
        if constexpr (KEEP) {
            const int t = w.lane & 15;
            rk = t < n ? p.keep[(int64_t)w.n * p.L + t0 + t] : 1.f;
        }
    };
    if (tbeg < tend) fetch(tbeg, tend - tbeg);
    if constexpr (!LOCAL) {
        if (p.state) load_states<SPL>(p.state + w.n * (int64_t)D * S + states, S, w.q, h);
        const int64_t stride = (int64_t)D * S;
        join_segments<SPL>(p, run.first * stride + states, stride, run.seg, S, w.q, h);   // the segments in front
    }
    float *saved = nullptr;
    if (!LOCAL && p.saved)
        saved = p.saved + ((int64_t)w.n * ((p.L + kScanBlock - 1) / kScanBlock) + tbeg / kScanBlock) * D * S + states;

    for (int t0 = tbeg, buf = 0; t0 < tend; t0 += kScanBlock, buf ^= 1) {
        const int n = tend - t0;
        float uu[4], dt[4], gg[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float sig;
            uu[i] = (float)ru[i];
            dt[i] = (float)rd[i] + bias;
            if (p.softplus) dt[i] = softplus_sig(dt[i], sig);
        }
        if (n < kScanBlock) {   // behind the end: a decay of one, nothing added
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * i + w.q >= n) uu[i] = 0.f, dt[i] = 0.f;
        }
        if (gate) {
#pragma unroll
            for (int i = 0; i < 4; ++i) gg[i] = (float)rz[i], gg[i] *= sigmoid(gg[i]);
        }
        rows.stage(&bc[buf][0][0][0], rb, rc, n, !LOCAL);
        unsigned resets = 0;
        if constexpr (KEEP) {
            resets = (unsigned)__ballot(w.lane < 16 && is_reset(rk));
            alive = alive && resets == 0;
        }
        __syncthreads();
        if (n > kScanBlock) {
            u.move(kScanBlock), dl.move(kScanBlock), z.move(kScanBlock), rows.move(kScanBlock);
            fetch(t0 + kScanBlock, n - kScanBlock);
        }
        if (!w.busy) continue;
        if (saved) {
            if (w.on) store_states<SPL>(saved, S, w.q, h);
            saved += (int64_t)D * S;
        }
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float du = dt[i] * uu[i];
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float dtj = quad_lane(dt[i], j), duj = quad_lane(du, j);
                const float *Bt = &bc[buf][0][4 * i + j][w.q * SPL], *Ct = &bc[buf][1][4 * i + j][w.q * SPL];
                const bool reset = KEEP && (resets >> (4 * i + j) & 1);
#pragma unroll
                for (int s = 0; s < SPL; ++s) {
                    if constexpr (KEEP) h[s] = reset ? 0.f : h[s];
                    h[s] = fmaf(__builtin_amdgcn_exp2f(dtj * A2[s]), h[s], duj * Bt[s]);
                    if constexpr (!LOCAL) y[j] = s == 0 ? Ct[s] * h[s] : fmaf(Ct[s], h[s], y[j]);
                }
            }
            if constexpr (LOCAL) total += dt[i];
            else o[i] = fmaf(Dc, uu[i], quad_sum_scatter(y[0], y[1], y[2], y[3], w.lane));
        }
        if constexpr (!LOCAL) {
            if (gate) {
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] *= gg[i];
            }
            if (w.on) {
                if (n >= kScanBlock) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) io_store(out.at(i, w.q), o[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (4 * i + w.q < n) io_store(out.at(i, w.q), o[i]);
                }
            }
            out.move(kScanBlock);
        }
    }
    if (!w.on) return;
    if constexpr (LOCAL) {
        total = group_sum<4>(total);
        const int64_t at = (run.first + run.seg) * D * S + states;
#pragma unroll
        for (int s = 0; s < SPL; ++s) A2[s] = decay_root(total * A2[s], alive);
        store_states<SPL>(p.seg_decay + at, S, w.q, A2);
        store_states<SPL>(p.seg_state + at, S, w.q, h);
    } else {
        if (run.used && run.seg == run.count - 1) store_states<SPL>(p.last + w.n * (int64_t)D * S + states, S, w.q, h);
        if (!p.lengths) return;
        int first, behind;   // rows behind a sequence's end
        ScanLane at = w;
        at.n = blockIdx.x % p.N;
        behind_share(p, at.n, blockIdx.z, first, behind);
        ScanRows<T, OFF> rest(p.out, p.os, at, first);
        for (int t = first; t < behind; t += 4, rest.move(4))
            if (t + w.q < behind) io_store(rest.at(0, w.q), 0.f);
    }
}

template <typename T, int SPL, typename OFF>
int launch_fwd_as(const ScanParams &p, hipStream_t s) {
    const unsigned tiles = (p.H / p.G * p.E + kScanTile - 1) / kScanTile;
    const dim3 grid(tiles * p.N, p.G, p.segments), before(tiles * p.N, p.G, p.lengths ? p.segments : p.segments - 1);
    if (p.segments > 1) {
        if (p.keep) scan_fwd_kernel<T, SPL, true, true, OFF><<<before, kScanThreads, 0, s>>>(p);
        else scan_fwd_kernel<T, SPL, false, true, OFF><<<before, kScanThreads, 0, s>>>(p);
        const int r = (int)hipGetLastError();
        if (r) return r;
    }
    if (p.keep) scan_fwd_kernel<T, SPL, true, false, OFF><<<grid, kScanThreads, 0, s>>>(p);
    else scan_fwd_kernel<T, SPL, false, false, OFF><<<grid, kScanThreads, 0, s>>>(p);
    return (int)hipGetLastError();
}
template <typename T, int SPL>
int launch_fwd(const ScanParams &p, hipStream_t s) {
    const bool wide = scan_span(p, p.us, sizeof(T)) || scan_span(p, p.ds, sizeof(T)) || scan_span(p, p.zs, sizeof(T)) ||
                      scan_span(p, p.os, sizeof(T));
    return wide ? launch_fwd_as<T, SPL, int64_t>(p, s) : launch_fwd_as<T, SPL, uint32_t>(p, s);
}

// One token: a lane updates SPL states of a channel in place, for RN batch rows whose states are all asked for before the
// first is used (A, D and the bias are read once for them).  Bound by the states' memory traffic for many rows (256 rows x
// 2048 channels x 16 states: 71 MB in 18 us, 3.9 TB/s; one row a thread 23.7 us), by latency for few (one row: 3.5 us).
template <typename T, int SPL, int RN>
__global__ __launch_bounds__(kScanThreads) void scan_step_kernel(ScanParams p) {
    ScanParams at = p;
    at.N = (p.N + RN - 1) / RN;
    const ScanLane w = scan_lane(at, blockIdx.x % at.N);
    if (!w.on) return;
    const int S = p.S, n0 = w.n * RN;
    const int64_t D = (int64_t)p.H * p.E, states = (int64_t)w.d * S;
    float h[RN][SPL], A2[SPL], b[RN][SPL], c[RN][SPL], uu[RN], dt[RN], zz[RN];
    bool reset[RN];
#pragma unroll
    for (int r = 0; r < RN; ++r) {
        const int n = min(n0 + r, p.N - 1);
        load_states<SPL>(p.last + n * D * S + states, S, w.q, h[r]);
        uu[r] = io_load((const T *)p.u + n * p.us.n + w.h * p.us.h + w.e);
        dt[r] = io_load((const T *)p.delta + n * p.ds.n + w.h * p.ds.h + w.e);
        zz[r] = p.z ? io_load((const T *)p.z + n * p.zs.n + w.h * p.zs.h + w.e) : 0.f;
        load_io_states<SPL>((const T *)p.B + n * p.Bs.n + w.g * p.Bs.h, S, w.q, b[r]);
        load_io_states<SPL>((const T *)p.C + n * p.Cs.n + w.g * p.Cs.h, S, w.q, c[r]);
        reset[r] = p.keep && is_reset(p.keep[n]);
    }
    load_decays<SPL>(p.A + states, S, w.q, A2);
    const float bias = p.bias ? p.bias[w.d] : 0.f, Dc = p.D ? p.D[w.d] : 0.f;
#pragma unroll
    for (int r = 0; r < RN; ++r) {
        float d = dt[r] + bias, sig, y = 0.f;
        if (p.softplus) d = softplus_sig(d, sig);
#pragma unroll
        for (int s = 0; s < SPL; ++s) {
            h[r][s] = fmaf(__builtin_amdgcn_exp2f(d * A2[s]), reset[r] ? 0.f : h[r][s], d * uu[r] * b[r][s]);
            y = fmaf(c[r][s], h[r][s], y);
        }
        y = fmaf(Dc, uu[r], group_sum<4>(y));
        if (p.z) y *= zz[r] * sigmoid(zz[r]);
        const int n = n0 + r;
        if (n < p.N) {
            store_states<SPL>(p.last + n * D * S + states, S, w.q, h[r]);
            if (w.q == 0) io_store((T *)p.out + n * p.os.n + w.h * p.os.h + w.e, y);
        }
    }
}

template <typename T, int SPL>
int launch_step(const ScanParams &p, hipStream_t s) {
    constexpr int RN = SPL <= 4 ? 4 : SPL <= 8 ? 2 : 1;   // rows per thread where there are many
    const unsigned tiles = (p.H / p.G * p.E + kScanTile - 1) / kScanTile;
    if ((int64_t)tiles * p.G * p.N >= kScanWaves && RN > 1)
        scan_step_kernel<T, SPL, RN><<<dim3(tiles * ((p.N + RN - 1) / RN), p.G), kScanThreads, 0, s>>>(p);
    else
        scan_step_kernel<T, SPL, 1><<<dim3(tiles * p.N, p.G), kScanThreads, 0, s>>>(p);
    return (int)hipGetLastError();
}

}  // namespace

#define FW_BY_STATES(FN)                                           \
    if (p.S <= 8) return bf16 ? FN<__bf16, 2>(p, s) : FN<float, 2>(p, s);   \
    if (p.S <= 16) return bf16 ? FN<__bf16, 4>(p, s) : FN<float, 4>(p, s);  \
    if (p.S <= 32) return bf16 ? FN<__bf16, 8>(p, s) : FN<float, 8>(p, s);  \
    return bf16 ? FN<__bf16, 16>(p, s) : FN<float, 16>(p, s);

int scan_segments(int N, int H, int L, int E, int G, bool backward, int *len) {
    const int64_t waves = ((int64_t)(H / G) * E + kScanTile - 1) / kScanTile * N * G * (kScanThreads / 64);
    int64_t n = waves >= (backward ? kScanEnoughBwd : kScanEnoughFwd) ? 1 : (kScanWaves + waves - 1) / waves;
    int64_t most = (L + kScanMinSegment - 1) / kScanMinSegment;
    while (most * most > (int64_t)L * (backward ? kScanJoinBwd : kScanJoinFwd)) most = most * 7 / 8;
    if (most < 1) most = 1;
    n = n < most ? n : most;
    const int64_t fits = (kScanBwdWaves + waves - 1) / waves;
    if (backward && n > fits && L / n < kScanBwdShort) n = fits;
    int l = (int)((L + n - 1) / n);
    l = (l + kScanBlock - 1) / kScanBlock * kScanBlock;
    *len = l;
    return (L + l - 1) / l;
}

int launch_scan_fwd(const ScanParams &p, bool bf16, hipStream_t s) { FW_BY_STATES(launch_fwd) }
int launch_scan_step(const ScanParams &p, bool bf16, hipStream_t s) { FW_BY_STATES(launch_step) }

}  // namespace fw

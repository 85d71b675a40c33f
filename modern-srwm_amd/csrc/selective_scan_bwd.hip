// Selective scan, backward.  With gh the gradient of the state, gy that of y (gy = g silu(z)):
//     gh_t += C_t gy_t;   gC_t += gy_t h_t;   gB_t += dt_t u_t gh_t            (sums over the channels of the group)
//     x_t = gh_t . B_t;   w_t = gh_t a_t h_{t-1};   a_t = exp(dt_t A)
//     gA += dt_t w_t;     gdt_t = w_t . A + x_t u_t;     gu_t = x_t dt_t + D gy_t
//     gh_{t-1} = a_t gh_t   (0 where keep_t == 0)
// The states h_t are formed again from the ones that the forward saved every 16 steps.
// Bound by vector instructions like the forward (busy 82 - 85 %): 4 x 2048 steps x 2048 channels x 16 states, bf16: 61 us for
// the segments' own results, 239 us for the main pass (24.9 instructions per state and step: 5 for the states again, 8 for
// the formulas above, the rest sums over channels and what a channel has once per step), 9 us for the joins.
#include "selective_scan.h"

namespace fw {
namespace {

// One step of a reduce-scatter over lanes 8 apart, for two values: lanes 0-7 of each row of 16 end up with the sum of
// lo over the pair (l, l ^ 8), lanes 8-15 with that of hi.  A DPP add writes the banks (groups of four lanes) that it is
// told to, so the sum and the choice between the two are one instruction each.  Written as assembly because the compiler
// forms it from a select, a move and an add; the s_nop covers the wait states between a vector write and a DPP read.
__device__ __forceinline__ float scatter_add8(float lo, float hi) {
    float r;
    asm("s_nop 1\n\tv_add_f32_dpp %0, %1, %1 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
        "v_add_f32_dpp %0, %2, %2 row_ror:8 row_mask:0xf bank_mask:0xc"
        : "=&v"(r) : "v"(lo), "v"(hi));
    return r;
}
// The same over lanes 4 apart: even banks read four lanes up, odd ones four lanes down.
__device__ __forceinline__ float scatter_add4(float lo, float hi) {
    float r;
    asm("s_nop 1\n\tv_add_f32_dpp %0, %1, %1 row_shl:4 row_mask:0xf bank_mask:0x5\n\t"
        "v_add_f32_dpp %0, %2, %2 row_shr:4 row_mask:0xf bank_mask:0xa"
        : "=&v"(r) : "v"(lo), "v"(hi));
    return r;
}

// Sums R values over the 16 lanes with the same lane % 4 and leaves R / 16 of the sums on each of them: the lane with
// bits (b5, b4, b3, b2) has those from index (8 b5 + 4 b4 + 2 b3 + b2) * R / 16 on.
template <int R>
__device__ __forceinline__ void channels_sum_scatter(const float (&v)[R], float (&out)[R / 16]) {
    float a[R / 2], b[R / 4], c[R / 8];
    swap_halve<32, R>(v, a);
    swap_halve<16, R / 2>(a, b);
#pragma unroll
    for (int i = 0; i < R / 8; ++i) c[i] = scatter_add8(b[i], b[i + R / 8]);
#pragma unroll
    for (int i = 0; i < R / 16; ++i) out[i] = scatter_add4(c[i], c[i + R / 16]);
}

// v[i], i uniform: a constant after unrolling, else three selects
__device__ __forceinline__ float pick4(const float (&v)[4], int i) { return i == 0 ? v[0] : i == 1 ? v[1] : i == 2 ? v[2] : v[3]; }

// Runs the state's gradient backwards through one segment from a zero gradient behind it, for nothing but the gradient
// in front of the segment and its product of decays.
template <typename T, int SPL, bool KEEP, typename OFF>
__global__ __launch_bounds__(kScanThreads) void scan_bwd_local_kernel(ScanBwdParams b) {
    constexpr int SP = 4 * SPL;
    using Bc = ScanBc<T, SPL>;
    __shared__ float bc[2][2][kScanBlock][SP];
    const ScanParams &p = b.f;
    // a row's first result is never needed
    const ScanRun run = scan_run(p, blockIdx.x % p.N, p.lengths ? blockIdx.z : blockIdx.z + 1);
    if (!run.used || run.seg == 0) return;   // the whole workgroup
    const ScanLane w = scan_lane(p, run.n);
    const int S = p.S, D = p.H * p.E, tbeg = run.tbeg, tend = run.tend;
    const int64_t states = (int64_t)w.d * S;
    const int last = tbeg + max(tend - tbeg - 1, 0) / kScanBlock * kScanBlock;   // first step of the last block
    ScanRows<const T, OFF> dl(p.delta, p.ds, w, last), z(p.z, p.zs, w, last), go(b.go, b.gos, w, last);
    Bc rows(p, w, last);
    const bool gate = p.z != nullptr;
    const float bias = p.bias ? p.bias[w.d] : 0.f;
    float A2[SPL], gh[SPL], total = 0.f;
    load_decays<SPL>(p.A + states, S, w.q, A2);
#pragma unroll
    for (int s = 0; s < SPL; ++s) gh[s] = 0.f;
    bool alive = true;

    T rd[4], rz[4], rg[4], rb[Bc::kEach], rc[Bc::kEach];
    float rk = 1.f;
    auto fetch = [&](int t0, int n) {
        const bool full = n >= kScanBlock;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = full ? i : 0, k = full ? w.q : min(4 * i + w.q, n - 1);
            rd[i] = *dl.at(at, k);
            rg[i] = *go.at(at, k);
            if (gate) rz[i] = *z.at(at, k);
        }
        rows.fetch(rb, rc, n, true);
        if constexpr (KEEP) {
            const int t = w.lane & 15;
            rk = t < n ? p.keep[(int64_t)w.n * p.L + t0 + t] : 1.f;
        }
    };
    if (tbeg < tend) fetch(last, tend - last);
    for (int t0 = last, buf = 0; t0 >= tbeg && tbeg < tend; t0 -= kScanBlock, buf ^= 1) {
        const int n = tend - t0;
        float dt[4], gy[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float sig;
            dt[i] = (float)rd[i] + bias;
            if (p.softplus) dt[i] = softplus_sig(dt[i], sig);
            gy[i] = (float)rg[i];
        }
        if (gate) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float zz = (float)rz[i];
                gy[i] *= zz * sigmoid(zz);
            }
        }
        if (n < kScanBlock) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * i + w.q >= n) dt[i] = 0.f, gy[i] = 0.f;
        }
        rows.stage(&bc[buf][0][0][0], rb, rc, n, true);
        unsigned resets = 0;
        if constexpr (KEEP) {
            resets = (unsigned)__ballot(w.lane < 16 && is_reset(rk));
            alive = alive && resets == 0;
        }
        __syncthreads();
        if (t0 > tbeg) {
            dl.move(-kScanBlock), z.move(-kScanBlock), go.move(-kScanBlock), rows.move(-kScanBlock);
            fetch(t0 - kScanBlock, kScanBlock);
        }
        if (!w.busy) continue;
#pragma unroll
        for (int t = kScanBlock - 1; t >= 0; --t) {
            const int i = t / 4, j = t % 4;
            const float dtj = quad_lane(dt[i], j), gyj = quad_lane(gy[i], j);
            const bool reset = KEEP && (resets >> t & 1);
#pragma unroll
            for (int s = 0; s < SPL; ++s) {
                gh[s] = fmaf(bc[buf][1][t][w.q * SPL + s], gyj, gh[s]) * __builtin_amdgcn_exp2f(dtj * A2[s]);
                if constexpr (KEEP) gh[s] = reset ? 0.f : gh[s];
            }
        }
        total += (dt[0] + dt[1]) + (dt[2] + dt[3]);
    }
    if (!w.on) return;
    total = group_sum<4>(total);
    const int64_t at = (run.first + run.seg) * D * S + states;
#pragma unroll
    for (int s = 0; s < SPL; ++s) A2[s] = decay_root(total * A2[s], alive);
    store_states<SPL>(p.seg_decay + at, S, w.q, A2);
    store_states<SPL>(p.seg_state + at, S, w.q, gh);
}

// Runs 64 channels of one sequence backwards through one segment of its steps, 16 at a time: the states of a block are
// formed again from the saved one in front of it and held in registers with their decays, then the block is walked back.
template <typename T, int SPL, bool KEEP, typename OFF>
__global__ __launch_bounds__(kScanThreads, SPL <= 8 ? 2 : 1) void scan_bwd_kernel(ScanBwdParams b) {
    constexpr int SP = 4 * SPL;
    // steps whose states are held at once (32 states, 4 x 1024 x 2048: 4 of them 0.36 ms, 8 spill registers: 0.44)
    constexpr int TS = SPL <= 4 ? 16 : 4;
    constexpr int kParts = kScanBlock / TS;
    constexpr int TG = SPL >= 8 ? 1 : 8 / SPL;         // steps whose sums over channels travel together
    constexpr int R = 2 * SPL * TG;
    using Bc = ScanBc<T, SPL>;
    __shared__ float bc[2][kScanBlock][SP];
    __shared__ float red[4][kScanBlock][2][SP];
    const ScanParams &p = b.f;
    const ScanRun run = scan_run(p, blockIdx.x % p.N, blockIdx.z);
    const ScanLane w = scan_lane(p, run.n);
    const int S = p.S, D = p.H * p.E, tbeg = run.tbeg, tend = run.tend;
    const int64_t states = (int64_t)w.d * S;
    const int last = tbeg + max(tend - tbeg - 1, 0) / kScanBlock * kScanBlock;   // first step of the last block

    ScanRows<const T, OFF> u(p.u, p.us, w, last), dl(p.delta, p.ds, w, last), z(p.z, p.zs, w, last), go(b.go, b.gos, w, last);
    ScanRows<T, OFF> gu(b.gu, b.gus, w, last), gd(b.gdelta, b.gds, w, last), gz(b.gz, b.gzs, w, last);
    Bc rows(p, w, last);
    const bool gate = p.z != nullptr;
    const float bias = p.bias ? p.bias[w.d] : 0.f, Dc = p.D ? p.D[w.d] : 0.f;
    const float *saved = p.saved + ((int64_t)w.n * ((p.L + kScanBlock - 1) / kScanBlock) + last / kScanBlock) * D * S + states;
    float *part = b.part_bc + (((int64_t)w.tile * p.N + w.n) * p.G + w.g) * p.L * 2 * S;

    float A2[SPL], gh[SPL], gA[SPL];
    load_decays<SPL>(p.A + states, S, w.q, A2);
#pragma unroll
    for (int s = 0; s < SPL; ++s) gh[s] = 0.f, gA[s] = 0.f;
    float gDsum = 0.f, gbsum = 0.f;

    T ru[4], rd[4], rz[4], rg[4], rb[Bc::kEach], rc[Bc::kEach];   // the next block as it lies in memory
    float rk = 1.f, h0[SPL];
    auto fetch = [&](int t0, int n) {
        const bool full = n >= kScanBlock;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = full ? i : 0, k = full ? w.q : min(4 * i + w.q, n - 1);
            ru[i] = *u.at(at, k);
            rd[i] = *dl.at(at, k);
            rg[i] = *go.at(at, k);
            if (gate) rz[i] = *z.at(at, k);
        }
        rows.fetch(rb, rc, n, true);
        load_states<SPL>(saved, S, w.q, h0);
        if constexpr (KEEP) {
            const int t = w.lane & 15;
            rk = t < n ? p.keep[(int64_t)w.n * p.L + t0 + t] : 1.f;
        }
    };
    if (tbeg < tend) fetch(last, tend - last);
    if (b.glast) load_states<SPL>(b.glast + w.n * (int64_t)D * S + states, S, w.q, gh);
    const int64_t stride = (int64_t)D * S;
    if (run.used)
        join_segments<SPL>(p, (run.first + run.count - 1) * stride + states, -stride, run.count - 1 - run.seg, S, w.q,
                           gh);   // the segments behind
    for (int t0 = last; t0 >= tbeg && tbeg < tend; t0 -= kScanBlock) {
        const int n = tend - t0;   // steps of this block, 16 or more: all
        // what a channel needs once per step: lane q holds the steps 4i + q
        float uu[4], dt[4], sg[4], gy[4], gg[4], zz[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uu[i] = (float)ru[i];
            dt[i] = (float)rd[i] + bias;
            sg[i] = 1.f;
            if (p.softplus) dt[i] = softplus_sig(dt[i], sg[i]);
            gg[i] = (float)rg[i];
            zz[i] = gate ? (float)rz[i] : 0.f;
        }
        if (n < kScanBlock) {   // behind the end: a decay of one, nothing added, no gradient
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * i + w.q >= n) uu[i] = 0.f, dt[i] = 0.f, sg[i] = 0.f, gg[i] = 0.f, zz[i] = 0.f;
        }
        if (!w.on) {   // a lane without a channel: zeros throughout, so that it adds nothing to gB and gC
#pragma unroll
            for (int i = 0; i < 4; ++i) uu[i] = 0.f, dt[i] = 0.f, gg[i] = 0.f, zz[i] = 0.f;
#pragma unroll
            for (int s = 0; s < SPL; ++s) h0[s] = 0.f, gh[s] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            gy[i] = gg[i];
            if (gate) {   // gz = g y silu'(z): the factor of y takes the place of g
                const float q = sigmoid(zz[i]);
                gy[i] *= zz[i] * q;
                gg[i] *= q * fmaf(zz[i], 1.f - q, 1.f);
            }
            gDsum = fmaf(gy[i], uu[i], gDsum);
        }
        rows.stage(&bc[0][0][0], rb, rc, n, true);
        unsigned resets = 0;
        if constexpr (KEEP) resets = (unsigned)__ballot(w.lane < 16 && is_reset(rk));
        __syncthreads();

        float hb[SPL];   // the state in front of the block
#pragma unroll
        for (int s = 0; s < SPL; ++s) hb[s] = h0[s];
        // parts of TS steps, the last one first
#pragma unroll 1
        for (int sub = kParts - 1; sub >= 0; --sub) {
            const int tsub = sub * TS;
            float h[SPL], a[TS][SPL], hs[TS + 1][SPL];
#pragma unroll
            for (int s = 0; s < SPL; ++s) h[s] = hb[s];
            if constexpr (kParts > 1) {   // forward again up to the part
#pragma unroll 1
                for (int i = 0; i < sub * TS / 4; ++i) {
                    const float d4 = pick4(dt, i), du4 = d4 * pick4(uu, i);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float dtj = quad_lane(d4, j), duj = quad_lane(du4, j);
                        const bool reset = KEEP && (resets >> (4 * i + j) & 1);
#pragma unroll
                        for (int s = 0; s < SPL; ++s) {
                            if constexpr (KEEP) h[s] = reset ? 0.f : h[s];
                            h[s] = fmaf(__builtin_amdgcn_exp2f(dtj * A2[s]), h[s], duj * bc[0][4 * i + j][w.q * SPL + s]);
                        }
                    }
                }
            }
            // and through it, keeping its states and decays
            float y[4];
#pragma unroll
            for (int s = 0; s < SPL; ++s) hs[0][s] = h[s];
#pragma unroll
            for (int k = 0; k < TS; ++k) {
                const int t = tsub + k, i = k / 4;
                const float d4 = pick4(dt, tsub / 4 + i), u4 = pick4(uu, tsub / 4 + i);
                const float dtj = quad_lane(d4, k % 4), duj = quad_lane(d4 * u4, k % 4);
                const bool reset = KEEP && (resets >> t & 1);
#pragma unroll
                for (int s = 0; s < SPL; ++s) {
                    float as = __builtin_amdgcn_exp2f(dtj * A2[s]);
                    if constexpr (KEEP) as = reset ? 0.f : as, h[s] = reset ? 0.f : h[s];
                    h[s] = fmaf(as, h[s], duj * bc[0][t][w.q * SPL + s]);
                    a[k][s] = as;
                    hs[k + 1][s] = h[s];
                    const float c = bc[1][t][w.q * SPL + s];
                    y[k % 4] = s == 0 ? c * h[s] : fmaf(c, h[s], y[k % 4]);
                }
                if (k % 4 == 3 && gate) {
                    const float yy = fmaf(Dc, u4, quad_sum_scatter(y[0], y[1], y[2], y[3], w.lane));
                    if (tsub + 4 * i + w.q < n && w.on) io_store(gz.at(tsub / 4 + i, w.q), pick4(gg, tsub / 4 + i) * yy);
                }
            }
            if constexpr (KEEP) asm volatile("" : "+s"(resets));   // its bits are tested anew, not kept as 16 masks
            // and back
            float v[R];
            float into[4], ex[4];
#pragma unroll
            for (int k = TS - 1; k >= 0; --k) {
                // the next block's inputs come in while the second half of this one's first steps is walked back, when
                // half of the registers of the states are free
                if (k == TS / 2 - 1 && sub == 0 && t0 > tbeg) {
                    u.move(-kScanBlock), dl.move(-kScanBlock), z.move(-kScanBlock), go.move(-kScanBlock), rows.move(-kScanBlock);
                    saved -= (int64_t)D * S;
                    fetch(t0 - kScanBlock, kScanBlock);
                }
                const int t = tsub + k, i = k / 4, j = k % 4;
                const float d4 = pick4(dt, tsub / 4 + i), u4 = pick4(uu, tsub / 4 + i), g4 = pick4(gy, tsub / 4 + i);
                const float dtj = quad_lane(d4, j), duj = quad_lane(d4 * u4, j), gyj = quad_lane(g4, j);
                const bool reset = KEEP && (resets >> t & 1);
                const int o = (k % TG) * 2 * SPL;
#pragma unroll
                for (int s = 0; s < SPL; ++s) {
                    const float Bt = bc[0][t][w.q * SPL + s];
                    gh[s] = fmaf(bc[1][t][w.q * SPL + s], gyj, gh[s]);
                    into[j] = s == 0 ? gh[s] * Bt : fmaf(gh[s], Bt, into[j]);
                    v[o + s] = gh[s] * duj;
                    v[o + SPL + s] = gyj * hs[k + 1][s];
                    const float ag = a[k][s] * gh[s];
                    const float before = KEEP && reset ? 0.f : hs[k][s];
                    const float e = ag * before;
                    ex[j] = s == 0 ? e * A2[s] : fmaf(e, A2[s], ex[j]);
                    gA[s] = fmaf(e, dtj, gA[s]);
                    gh[s] = KEEP && reset ? 0.f : ag;
                }
                if (k % TG == 0) {
                    float r[R / 16];
                    channels_sum_scatter<R>(v, r);
                    const int at = (w.lane >> 2) * (R / 16);
#pragma unroll
                    for (int x = 0; x < R / 16; ++x) {
                        const int idx = at + x;
                        red[w.wave][t + idx / (2 * SPL)][idx / SPL % 2][w.q * SPL + idx % SPL] = r[x];
                    }
                }
                if (j == 0) {
                    const float in = quad_sum_scatter(into[0], into[1], into[2], into[3], w.lane);
                    const float xe = quad_sum_scatter(ex[0], ex[1], ex[2], ex[3], w.lane);
                    const float g1 = fmaf(xe, 0.693147180559945309f, in * u4) * pick4(sg, tsub / 4 + i);
                    gbsum += g1;
                    if (tsub + 4 * i + w.q < n && w.on) {
                        io_store(gu.at(tsub / 4 + i, w.q), fmaf(in, d4, Dc * g4));
                        io_store(gd.at(tsub / 4 + i, w.q), g1);
                    }
                }
            }
        }
        gu.move(-kScanBlock), gd.move(-kScanBlock), gz.move(-kScanBlock);
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * kScanBlock * SP; i += kScanThreads) {
            const int s = i % SP, c = i / SP % 2, t = i / (2 * SP);
            if (s < S && t < n)
                part[((int64_t)(t0 + t) * 2 + c) * S + s] = (red[0][t][c][s] + red[1][t][c][s]) + (red[2][t][c][s] + red[3][t][c][s]);
        }
    }
    gDsum = group_sum<4>(gDsum);
    gbsum = group_sum<4>(gbsum);
    if (!w.on) return;
    // a share of the sums of gA, gD and gbias from every workgroup, of zeros from one without steps
    float *pa = b.part_a + ((int64_t)blockIdx.z * p.N + blockIdx.x % p.N) * scan_part_a_row(D, S);
    store_states<SPL>(pa + states, S, w.q, gA);
    if (w.q == 0) {
        pa[(int64_t)D * S + w.d] = gDsum;
        pa[(int64_t)D * (S + 1) + w.d] = gbsum;
    }
    if (b.gstate && run.used && run.seg == 0) store_states<SPL>(b.gstate + w.n * (int64_t)D * S + states, S, w.q, gh);
    if (!p.lengths) return;
    int first, behind;   // rows behind a sequence's end
    ScanLane at = w;
    at.n = blockIdx.x % p.N;
    behind_share(p, at.n, blockIdx.z, first, behind);
    ScanRows<T, OFF> qu(b.gu, b.gus, at, first), qd(b.gdelta, b.gds, at, first), qz(b.gz, b.gzs, at, first);
    for (int t = first; t < behind; t += 4, qu.move(4), qd.move(4), qz.move(4))
        if (t + w.q < behind) {
            io_store(qu.at(0, w.q), 0.f);
            io_store(qd.at(0, w.q), 0.f);
            if (gate) io_store(qz.at(0, w.q), 0.f);
        }
}

// Joins the partial sums, in a fixed order: those of gB and gC over the tiles of a group (an element per thread), those
// of gA, gD and gbias over batch and segments (32 columns per workgroup, 8 threads over the rows of each).
template <typename T>
__global__ __launch_bounds__(256) void scan_bwd_join_kernel(ScanBwdParams b, int tiles, unsigned blocks_bc) {
    __shared__ float sums[8][32];
    const ScanParams &p = b.f;
    const int S = p.S;
    if (blockIdx.x < blocks_bc) {
        const int64_t per = (int64_t)p.N * p.G * p.L * 2 * S;
        const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
        if (i >= per) return;
        const int s = i % S, c = i / S % 2;
        const int64_t r = i / (2 * S);
        const int t = r % p.L, g = r / p.L % p.G, n = r / p.L / p.G;
        float v = 0.f;
        if (!p.lengths || t < p.lengths[n]) {
#pragma unroll 8
            for (int k = 0; k < tiles; ++k) v += b.part_bc[k * per + i];
        }
        if (c) io_store((T *)b.gC + n * b.gCs.n + g * b.gCs.h + t * b.gCs.l + s, v);
        else io_store((T *)b.gB + n * b.gBs.n + g * b.gBs.h + t * b.gBs.l + s, v);
        return;
    }
    const int64_t D = (int64_t)p.H * p.E, row = scan_part_a_row(D, S);
    const int c = threadIdx.x % 32, r = threadIdx.x / 32, rows = p.N * p.segments;
    const int64_t i = (int64_t)(blockIdx.x - blocks_bc) * 32 + c;
    float *dst = nullptr;
    if (i < D * S) dst = b.gA + i;
    else if (i < D * (S + 1)) dst = b.gD ? b.gD + (i - D * S) : nullptr;
    else if (i < D * (S + 2)) dst = b.gbias ? b.gbias + (i - D * (S + 1)) : nullptr;
    float v = 0.f;
    if (dst) {
#pragma unroll 8
        for (int n = r; n < rows; n += 8) v += b.part_a[n * row + i];
    }
    sums[r][c] = v;
    __syncthreads();
    if (r == 0 && dst) {
        v = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) v += sums[k][c];
        *dst = v;
    }
}

template <typename T, int SPL, typename OFF>
int launch_bwd_as(const ScanBwdParams &b, hipStream_t s) {
    const ScanParams &p = b.f;
    const unsigned tiles = (p.H / p.G * p.E + kScanTile - 1) / kScanTile;
    const dim3 grid(tiles * p.N, p.G, p.segments), behind(tiles * p.N, p.G, p.lengths ? p.segments : p.segments - 1);
    int r = 0;
    if (p.segments > 1) {
        if (p.keep) scan_bwd_local_kernel<T, SPL, true, OFF><<<behind, kScanThreads, 0, s>>>(b);
        else scan_bwd_local_kernel<T, SPL, false, OFF><<<behind, kScanThreads, 0, s>>>(b);
        if ((r = (int)hipGetLastError())) return r;
    }
    if (p.keep) scan_bwd_kernel<T, SPL, true, OFF><<<grid, kScanThreads, 0, s>>>(b);
    else scan_bwd_kernel<T, SPL, false, OFF><<<grid, kScanThreads, 0, s>>>(b);
    if ((r = (int)hipGetLastError())) return r;
    const int64_t nbc = ((int64_t)p.N * p.G * p.L * 2 * p.S + 255) / 256;
    const int64_t na = ((int64_t)p.H * p.E * (p.S + 2) + 31) / 32;
    scan_bwd_join_kernel<T><<<(unsigned)(nbc + na), 256, 0, s>>>(b, (int)tiles, (unsigned)nbc);
    return (int)hipGetLastError();
}
template <typename T, int SPL>
int launch_bwd(const ScanBwdParams &b, hipStream_t s) {
    const ScanParams &p = b.f;
    const bool wide = scan_span(p, p.us, sizeof(T)) || scan_span(p, p.ds, sizeof(T)) || scan_span(p, p.zs, sizeof(T)) ||
                      scan_span(p, b.gos, sizeof(T)) || scan_span(p, b.gus, sizeof(T)) || scan_span(p, b.gds, sizeof(T)) ||
                      scan_span(p, b.gzs, sizeof(T));
    return wide ? launch_bwd_as<T, SPL, int64_t>(b, s) : launch_bwd_as<T, SPL, uint32_t>(b, s);
}

}  // namespace

int launch_scan_bwd(const ScanBwdParams &b, bool bf16, hipStream_t s) {
    const int S = b.f.S;
    if (S <= 8) return bf16 ? launch_bwd<__bf16, 2>(b, s) : launch_bwd<float, 2>(b, s);
    if (S <= 16) return bf16 ? launch_bwd<__bf16, 4>(b, s) : launch_bwd<float, 4>(b, s);
    if (S <= 32) return bf16 ? launch_bwd<__bf16, 8>(b, s) : launch_bwd<float, 8>(b, s);
    return bf16 ? launch_bwd<__bf16, 16>(b, s) : launch_bwd<float, 16>(b, s);
}

}  // namespace fw

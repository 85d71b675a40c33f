// Selective scan, backward.  With gh the gradient of the state, gy that of y (gy = g silu(z)):
//     gh_t += C_t gy_t;   gC_t += gy_t h_t;   gB_t += dt_t u_t gh_t            (sums over the channels of the group)
//     x_t = gh_t . B_t;   w_t = gh_t a_t h_{t-1};   a_t = exp(dt_t A)
//     gA += dt_t w_t;     gdt_t = w_t . A + x_t u_t;     gu_t = x_t dt_t + D gy_t
//     gh_{t-1} = a_t gh_t   (0 where keep_t == 0)
// The states h_t are formed again from the ones that the forward saved every 16 steps.
#include "selective_scan.h"

namespace fw {
namespace {

// Value of lane ^ 4 (within a row of 16: the even banks read four lanes up, the odd ones four lanes down).
__device__ __forceinline__ float xor4(float v) {
    const int x = __builtin_bit_cast(int, v);
    int r = __builtin_amdgcn_update_dpp(0, x, 0x104, 0xF, 0x5, true);
    r = __builtin_amdgcn_update_dpp(r, x, 0x114, 0xF, 0xA, false);
    return __builtin_bit_cast(float, r);
}

// Sums R values over the 16 lanes with the same lane % 4 and leaves R / 16 of the sums on each of them: the lane with
// bits (b5, b4, b3, b2) has those from index (8 b5 + 4 b4 + 2 b3 + b2) * R / 16 on.
template <int R>
__device__ __forceinline__ void channels_sum_scatter(const float (&v)[R], float (&out)[R / 16], int lane) {
    float a[R / 2], b[R / 4], c[R / 8];
    swap_halve<32, R>(v, a);
    swap_halve<16, R / 2>(a, b);
    const bool b3 = lane & 8, b2 = lane & 4;
#pragma unroll
    for (int i = 0; i < R / 8; ++i) c[i] = (b3 ? b[i + R / 8] : b[i]) + dpp_mov<kDppRor8>(b3 ? b[i] : b[i + R / 8]);
#pragma unroll
    for (int i = 0; i < R / 16; ++i) out[i] = (b2 ? c[i + R / 16] : c[i]) + xor4(b2 ? c[i] : c[i + R / 16]);
}

template <typename T, int SPL, bool KEEP>
__global__ __launch_bounds__(kScanThreads) void scan_bwd_kernel(ScanBwdParams b) {
    constexpr int SP = 4 * SPL;
    constexpr int TS = SPL <= 4 ? 16 : 64 / SPL;       // steps whose states are held in registers at once
    constexpr int TG = SPL >= 8 ? 1 : 8 / SPL;         // steps whose sums over channels travel together
    constexpr int R = 2 * SPL * TG;
    __shared__ float bc[2][kScanBlock][SP];
    __shared__ float red[4][kScanBlock][2][SP];
    const ScanParams &p = b.f;
    const int n = blockIdx.x % p.N, tile = blockIdx.x / p.N, g = blockIdx.y;
    const ScanLane w = scan_lane(p.H, p.E, p.G, tile, g);
    const int S = p.S, D = p.H * p.E;
    int Ln = p.L;
    if (p.lengths) Ln = min(max(p.lengths[n], 0), p.L);

    const T *u = (const T *)p.u + n * p.us.n + w.h * p.us.h + w.e;
    const T *dl = (const T *)p.delta + n * p.ds.n + w.h * p.ds.h + w.e;
    const T *z = p.z ? (const T *)p.z + n * p.zs.n + w.h * p.zs.h + w.e : nullptr;
    const T *go = (const T *)b.go + n * b.gos.n + w.h * b.gos.h + w.e;
    T *gu = (T *)b.gu + n * b.gus.n + w.h * b.gus.h + w.e;
    T *gd = (T *)b.gdelta + n * b.gds.n + w.h * b.gds.h + w.e;
    T *gz = z ? (T *)b.gz + n * b.gzs.n + w.h * b.gzs.h + w.e : nullptr;
    const T *Bp = (const T *)p.B + n * p.Bs.n + g * p.Bs.h;
    const T *Cp = (const T *)p.C + n * p.Cs.n + g * p.Cs.h;
    const float bias = p.bias ? p.bias[w.d] : 0.f, Dc = p.D ? p.D[w.d] : 0.f;

    float A2[SPL], gh[SPL], gA[SPL];
    load_states<SPL>(p.A + (int64_t)w.d * S, S, w.q, A2);
#pragma unroll
    for (int s = 0; s < SPL; ++s) A2[s] *= kLog2e, gh[s] = 0.f, gA[s] = 0.f;
    if (b.glast) load_states<SPL>(b.glast + ((int64_t)n * D + w.d) * S, S, w.q, gh);
    float gDsum = 0.f, gbsum = 0.f;

    if (w.on)
        for (int64_t t = Ln + w.q; t < p.L; t += 4) {
            io_store(gu + t * b.gus.l, 0.f);
            io_store(gd + t * b.gds.l, 0.f);
            if (z) io_store(gz + t * b.gzs.l, 0.f);
        }

    const int nblk = (Ln + kScanBlock - 1) / kScanBlock, nsave = (p.L + kScanBlock - 1) / kScanBlock;
    float *part = b.part_bc + (((int64_t)tile * p.N + n) * p.G + g) * p.L * 2 * S;
    for (int blk = nblk - 1; blk >= 0; --blk) {
        const int t0 = blk * kScanBlock;
        for (int i = threadIdx.x; i < 2 * kScanBlock * SP; i += kScanThreads) {
            const int s = i % SP, t = i / SP % kScanBlock, c = i / (SP * kScanBlock);
            float v = 0.f;
            if (s < S && t0 + t < Ln) v = c ? io_load(Cp + (t0 + t) * p.Cs.l + s) : io_load(Bp + (t0 + t) * p.Bs.l + s);
            bc[c][t][s] = v;
        }
        unsigned resets = 0;
        if constexpr (KEEP) {
            const int t = t0 + (w.lane & 15);
            resets = (unsigned)__ballot(w.lane < 16 && t < Ln && is_reset(p.keep[(int64_t)n * p.L + min(t, p.L - 1)]));
        }
        __syncthreads();

        // what a channel needs once per step: lane q holds the steps 4i + q
        float uu[4], dt[4], du[4], sg[4], gg[4], zz[4], gy[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t t = t0 + 4 * i + w.q;
            uu[i] = dt[i] = sg[i] = gg[i] = zz[i] = 0.f;
            if (t < Ln) {
                uu[i] = io_load(u + t * p.us.l);
                gg[i] = w.on ? io_load(go + t * b.gos.l) : 0.f;   // a lane without a channel adds nothing to gB and gC
                dt[i] = io_load(dl + t * p.ds.l) + bias;
                if (z) zz[i] = io_load(z + t * p.zs.l);
                sg[i] = 1.f;
                if (p.softplus) dt[i] = softplus_sig(dt[i], sg[i]);
            }
            du[i] = dt[i] * uu[i];
            gy[i] = z ? gg[i] * zz[i] * sigmoid(zz[i]) : gg[i];
            gDsum = fmaf(gy[i], uu[i], gDsum);
        }

        float h0[SPL];
        load_states<SPL>(p.saved + (((int64_t)n * nsave + blk) * D + w.d) * S, S, w.q, h0);
#pragma unroll
        for (int sub = kScanBlock / TS - 1; sub >= 0; --sub) {
            float h[SPL], a[TS][SPL], hs[TS + 1][SPL];
#pragma unroll
            for (int s = 0; s < SPL; ++s) h[s] = h0[s];
            // forward again, keeping what the last TS steps need
            float y[4];
#pragma unroll
            for (int t = 0; t < (sub + 1) * TS; ++t) {
                const int i = t / 4, j = t % 4, k = t - sub * TS;
                const float dtj = quad_lane(dt[i], j), duj = quad_lane(du[i], j);
                const bool reset = KEEP && (resets >> t & 1);
                if (k == 0) {
#pragma unroll
                    for (int s = 0; s < SPL; ++s) hs[0][s] = h[s];
                }
                y[j] = 0.f;
#pragma unroll
                for (int s = 0; s < SPL; ++s) {
                    float as = __builtin_amdgcn_exp2f(dtj * A2[s]);
                    if constexpr (KEEP) as = reset ? 0.f : as, h[s] = reset ? 0.f : h[s];
                    h[s] = fmaf(as, h[s], duj * bc[0][t][w.q * SPL + s]);
                    if (k >= 0) {
                        a[k < 0 ? 0 : k][s] = as;
                        hs[(k < 0 ? 0 : k) + 1][s] = h[s];
                        y[j] = fmaf(bc[1][t][w.q * SPL + s], h[s], y[j]);
                    }
                }
                if (k >= 0 && j == 3 && z) {
                    const float yy = quad_sum_scatter(y[0], y[1], y[2], y[3], w.lane) + Dc * uu[i];
                    const float q = sigmoid(zz[i]);
                    const int64_t tt = t0 + 4 * i + w.q;
                    if (tt < Ln && w.on) io_store(gz + tt * b.gzs.l, gg[i] * yy * q * (1.f + zz[i] * (1.f - q)));
                }
            }
            // and back
            float v[R];
            float into[4], ex[4];
#pragma unroll
            for (int k = TS - 1; k >= 0; --k) {
                const int t = sub * TS + k, i = t / 4, j = t % 4;
                const float dtj = quad_lane(dt[i], j), duj = quad_lane(du[i], j), gyj = quad_lane(gy[i], j);
                const bool reset = KEEP && (resets >> t & 1);
                into[j] = ex[j] = 0.f;
                const int o = (t % TG) * 2 * SPL;
#pragma unroll
                for (int s = 0; s < SPL; ++s) {
                    gh[s] = fmaf(bc[1][t][w.q * SPL + s], gyj, gh[s]);
                    into[j] = fmaf(gh[s], bc[0][t][w.q * SPL + s], into[j]);
                    v[o + s] = w.on ? gh[s] * duj : 0.f;
                    v[o + SPL + s] = gyj * hs[k + 1][s];
                    const float ag = a[k][s] * gh[s];
                    const float before = KEEP && reset ? 0.f : hs[k][s];
                    const float e = ag * before;
                    ex[j] = fmaf(e, A2[s], ex[j]);
                    gA[s] = fmaf(e, dtj, gA[s]);
                    gh[s] = KEEP && reset ? 0.f : ag;
                }
                if (t % TG == 0) {
                    float r[R / 16];
                    channels_sum_scatter<R>(v, r, w.lane);
                    const int first = (w.lane >> 2) % 16;
                    // bits of the lane's place, most significant first: b5, b4, b3, b2
                    const int at = ((first >> 3 & 1) * 8 + (first >> 2 & 1) * 4 + (first >> 1 & 1) * 2 + (first & 1)) * (R / 16);
#pragma unroll
                    for (int x = 0; x < R / 16; ++x) {
                        const int idx = at + x;
                        red[w.wave][t + idx / (2 * SPL)][idx / SPL % 2][w.q * SPL + idx % SPL] = r[x];
                    }
                }
                if (j == 0) {
                    const float in = quad_sum_scatter(into[0], into[1], into[2], into[3], w.lane);
                    const float xe = quad_sum_scatter(ex[0], ex[1], ex[2], ex[3], w.lane);
                    const float g1 = fmaf(xe, 0.693147180559945309f, in * uu[i]) * sg[i];
                    const int64_t tt = t0 + 4 * i + w.q;
                    gbsum += g1;
                    if (tt < Ln && w.on) {
                        io_store(gu + tt * b.gus.l, fmaf(in, dt[i], Dc * gy[i]));
                        io_store(gd + tt * b.gds.l, g1);
                    }
                }
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * kScanBlock * SP; i += kScanThreads) {
            const int s = i % SP, c = i / SP % 2, t = i / (2 * SP);
            if (s < S && t0 + t < Ln)
                part[((int64_t)(t0 + t) * 2 + c) * S + s] = (red[0][t][c][s] + red[1][t][c][s]) + (red[2][t][c][s] + red[3][t][c][s]);
        }
    }
    gDsum = group_sum<4>(gDsum);
    gbsum = group_sum<4>(gbsum);
    if (w.on) {
        if (b.gstate) store_states<SPL>(b.gstate + ((int64_t)n * D + w.d) * S, S, w.q, gh);
        float *pa = b.part_a + n * scan_part_a_row(D, S);
        store_states<SPL>(pa + (int64_t)w.d * S, S, w.q, gA);
        if (w.q == 0) {
            pa[(int64_t)D * S + w.d] = gDsum;
            pa[(int64_t)D * (S + 1) + w.d] = gbsum;
        }
    }
}

// Joins the partial sums: those of gB and gC over the tiles of a group, those of gA, gD and gbias over the batch.
template <typename T>
__global__ __launch_bounds__(256) void scan_bwd_join_kernel(ScanBwdParams b, int tiles, unsigned blocks_bc) {
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
        if (!p.lengths || t < p.lengths[n])
            for (int k = 0; k < tiles; ++k) v += b.part_bc[k * per + i];
        if (c) io_store((T *)b.gC + n * b.gCs.n + g * b.gCs.h + t * b.gCs.l + s, v);
        else io_store((T *)b.gB + n * b.gBs.n + g * b.gBs.h + t * b.gBs.l + s, v);
        return;
    }
    const int64_t D = (int64_t)p.H * p.E, row = scan_part_a_row(D, S);
    const int64_t i = (int64_t)(blockIdx.x - blocks_bc) * 256 + threadIdx.x;
    if (i >= D * (S + 2)) return;
    float *dst = i < D * S ? b.gA + i : i < D * (S + 1) ? (b.gD ? b.gD + (i - D * S) : nullptr)
                                                        : (b.gbias ? b.gbias + (i - D * (S + 1)) : nullptr);
    if (!dst) return;
    float v = 0.f;
    for (int n = 0; n < p.N; ++n) v += b.part_a[n * row + i];
    *dst = v;
}

template <typename T, int SPL>
int launch_bwd(const ScanBwdParams &b, hipStream_t s) {
    const ScanParams &p = b.f;
    const int Dg = p.H / p.G * p.E, tiles = (Dg + kScanTile - 1) / kScanTile;
    const dim3 grid(tiles * p.N, p.G);
    if (p.keep) scan_bwd_kernel<T, SPL, true><<<grid, kScanThreads, 0, s>>>(b);
    else scan_bwd_kernel<T, SPL, false><<<grid, kScanThreads, 0, s>>>(b);
    const int r = (int)hipGetLastError();
    if (r) return r;
    const int64_t nbc = ((int64_t)p.N * p.G * p.L * 2 * p.S + 255) / 256;
    const int64_t na = ((int64_t)p.H * p.E * (p.S + 2) + 255) / 256;
    scan_bwd_join_kernel<T><<<(unsigned)(nbc + na), 256, 0, s>>>(b, tiles, (unsigned)nbc);
    return (int)hipGetLastError();
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

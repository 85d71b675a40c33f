// Root-mean-square norm with the residual's addition:  s = x + r;  out = s rsqrt(mean(s^2) + eps) weight,
// with `out` in the type of x or in e4m3 with one scale per row, and the backward pass.  One wave per row up to 2048
// elements, one workgroup of 4 waves per row beyond; a row stays in registers up to 32 elements per lane and is read a
// second time beyond that.  Memory-bound, every element once: 8192 rows of 1024 (bf16, fp32 residual) forward 101 MB in
// 21 us (4.8 TB/s), backward 134 MB in 27.5 us (4.9) and 7 us for the join of the weight's gradient; to e4m3, 12 001 rows,
// 135 MB in 23.7 us (5.7); one row 3.6 us, which is a launch.
#include "common.h"
#include "vec_io.h"
#include "xlane.h"

namespace fw {
namespace {

constexpr int kNormThreads = 256;
constexpr int kNormBlocks = 1024;   // workgroups of the backward, each with a share of the weight's gradient
constexpr float kE4m3Max = 448.f;

// Sum (or maximum) over the TPR lanes of a row.
template <int TPR, class Op>
__device__ __forceinline__ float row_reduce(float v, float *lds) {
    v = group_allreduce<64, Op>(v);
    if constexpr (TPR == 256) {
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[wave] = v;
        __syncthreads();
        v = Op::f(Op::f(lds[0], lds[1]), Op::f(lds[2], lds[3]));
    }
    return v;
}

template <typename TX, typename TR, int V>
__device__ __forceinline__ void load_sum(const TX *x, const TR *r, int64_t at, float (&v)[V]) {
    load_vec<V>(x + at, v);
    if (r) {
        float a[V];
        load_vec<V>(r + at, a);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] += a[i];
    }
}

__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xFFFFu;
}
template <int V>
__device__ __forceinline__ void store_e4m3(uint8_t *p, const float (&v)[V]) {
    if constexpr (V == 4) {
        *reinterpret_cast<uint32_t *>(p) = e4m3_pair(v[0], v[1]) | e4m3_pair(v[2], v[3]) << 16;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = (uint8_t)e4m3_pair(v[i], 0.f);
    }
}

// NV vectors of V elements per lane in registers; NV == 0: the row is read again instead of being held.
template <typename TX, typename TR, int V, int TPR, int NV, bool E4M3>
__global__ __launch_bounds__(kNormThreads) void norm_fwd_kernel(NormParams p) {
    __shared__ float lds[4];
    const int lane = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (kNormThreads / TPR) + threadIdx.x / TPR;
    if (row >= p.rows) return;   // whole waves; with TPR == 256 the grid has no such row
    const int64_t base = row * p.D;
    const TX *x = (const TX *)p.x + base;
    const TR *r = p.residual ? (const TR *)p.residual + base : nullptr;
    TR *sum = p.sum ? (TR *)p.sum + base : nullptr;
    float keep[NV > 0 ? NV : 1][V];
    float sq = 0.f;
    auto first = [&](int d, float (&v)[V]) {
        load_sum<TX, TR, V>(x, r, d, v);
        if (sum) store_vec<V>(sum + d, v);
#pragma unroll
        for (int i = 0; i < V; ++i) sq = fmaf(v[i], v[i], sq);
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int d = (k * TPR + lane) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) keep[k][i] = 0.f;
            if (d < p.D) first(d, keep[k]);
        }
    } else {
        for (int d = lane * V; d < p.D; d += TPR * V) first(d, keep[0]);
    }
    sq = row_reduce<TPR, OpSum>(sq, lds);
    const float rstd = 1.f / sqrtf(sq / (float)p.D + p.eps);
    if (p.rstd && lane == 0) p.rstd[row] = rstd;
    auto normed = [&](int d, const float (&v)[V], float (&y)[V]) {
        float w[V];
        load_vec<V>(p.weight + d, w);
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] = v[i] * rstd * w[i];
    };
    float inv = 1.f, lift = 1.f, by = 1.f;
    if constexpr (E4M3) {
        float top = 0.f;
        auto look = [&](int d, const float (&v)[V]) {
            float y[V];
            normed(d, v, y);
#pragma unroll
            for (int i = 0; i < V; ++i) top = fmaxf(top, fabsf(y[i]));
        };
        if constexpr (NV > 0) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int d = (k * TPR + lane) * V;
                if (d < p.D) look(d, keep[k]);
            }
        } else {
            for (int d = lane * V; d < p.D; d += TPR * V) {
                load_sum<TX, TR, V>(x, r, d, keep[0]);
                look(d, keep[0]);
            }
        }
        top = row_reduce<TPR, OpMax>(top, lds);
        float scale = top > 0.f ? top / kE4m3Max : 1.f;
        // below the normal numbers max / 448 may be off by half of itself: rounded up, or the quotients would pass 448
        if (scale < 0x1p-126f && scale * kE4m3Max < top) scale += 0x1p-149f;
        // a small scale is lifted, so that neither its reciprocal nor the quotients' remainders leave the normal numbers
        lift = scale < 1e-20f ? 0x1p64f : 1.f;
        by = scale * lift;
        inv = 1.f / by;
        if (inv == 0.f) by = 0.f;   // an infinite scale: quotients of zero (or NaN) without a remainder
        if (lane == 0) p.scale[row] = scale;
    }
    auto write = [&](int d, const float (&v)[V]) {
        float y[V];
        normed(d, v, y);
        if constexpr (E4M3) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                // y / scale: the product with the reciprocal may be a rounding beside a border of two e4m3 values, the remainder
                // puts it right (equal to the division for every scale's mantissa and all floats around each border; with a
                // division a call of 12 001 rows of 1024 takes 29.2 us in place of 27.3)
                const float a = y[i] * lift, q = a * inv;
                y[i] = fmaf(fmaf(-q, by, a), inv, q);
            }
            store_e4m3<V>((uint8_t *)p.out + base + d, y);
        } else {
            store_vec<V>((TX *)p.out + base + d, y);
        }
    };
    if constexpr (NV > 0) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int d = (k * TPR + lane) * V;
            if (d < p.D) write(d, keep[k]);
        }
    } else {
        for (int d = lane * V; d < p.D; d += TPR * V) {
            load_sum<TX, TR, V>(x, r, d, keep[0]);
            write(d, keep[0]);
        }
    }
}

// With hat = s rstd and m = mean(g w hat):  gs = rstd (g w - hat m) + gsum,  gw = sum over rows of g hat.
// A workgroup takes every blocks-th group of rows and leaves its share of gw in part[block].
template <typename TX, typename TR, int V, int TPR, int NV>
__global__ __launch_bounds__(kNormThreads) void norm_bwd_kernel(NormBwdParams p) {
    __shared__ float lds[4];
    constexpr int RPB = kNormThreads / TPR;
    const int lane = threadIdx.x % TPR;
    float gw[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) gw[k][i] = 0.f;
    for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; row < p.rows; row += (int64_t)p.blocks * RPB) {
        const int64_t base = row * p.D;
        const float rstd = p.rstd[row];
        float hat[NV][V], g[NV][V], s[NV][V], m = 0.f;
        if (p.gsum) {   // asked for in front of the row's reduction, used behind it
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int d = (k * TPR + lane) * V;
                if (d < p.D) load_vec<V>((const TR *)p.gsum + base + d, s[k]);
            }
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int d = (k * TPR + lane) * V;
            if (d < p.D) {
                float w[V];
                load_vec<V>((const TR *)p.sum + base + d, hat[k]);
                load_vec<V>((const TX *)p.go + base + d, g[k]);
                load_vec<V>(p.weight + d, w);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    hat[k][i] *= rstd;
                    gw[k][i] = fmaf(g[k][i], hat[k][i], gw[k][i]);
                    g[k][i] *= w[i];
                    m = fmaf(g[k][i], hat[k][i], m);
                }
            }
        }
        m = row_reduce<TPR, OpSum>(m, lds) / (float)p.D;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int d = (k * TPR + lane) * V;
            if (d < p.D) {
                float v[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    v[i] = rstd * fmaf(-hat[k][i], m, g[k][i]);
                    if (p.gsum) v[i] += s[k][i];
                }
                store_vec<V>((TX *)p.gx + base + d, v);
                if (p.gres) store_vec<V>((TR *)p.gres + base + d, v);
            }
        }
    }
    // the rows of a workgroup's waves, in a fixed order
    float *part = p.part + (int64_t)blockIdx.x * p.D;
    if constexpr (TPR == 64) {
        __shared__ float sums[4][NV * 64 * V];
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) sums[threadIdx.x >> 6][(k * 64 + lane) * V + i] = gw[k][i];
        __syncthreads();
        for (int d = threadIdx.x; d < p.D; d += kNormThreads) part[d] = (sums[0][d] + sums[1][d]) + (sums[2][d] + sums[3][d]);
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int d = (k * TPR + lane) * V;
            if (d < p.D) store_vec<V>(part + d, gw[k]);
        }
    }
}

// gweight[d] = sum of part[k][d]: 32 columns per workgroup, 8 threads over the rows of each, joined in a fixed order.
__global__ __launch_bounds__(256) void norm_join_kernel(const float *part, float *gweight, int D, int blocks) {
    __shared__ float sums[8][32];
    const int c = threadIdx.x % 32, r = threadIdx.x / 32, d = blockIdx.x * 32 + c;
    float v = 0.f;
    if (d < D) {
#pragma unroll 8
        for (int k = r; k < blocks; k += 8) v += part[(int64_t)k * D + d];
    }
    sums[r][c] = v;
    __syncthreads();
    if (r == 0 && d < D) {
        v = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) v += sums[k][c];
        gweight[d] = v;
    }
}

template <typename TX, typename TR, int V, bool E4M3>
int fwd_by_size(const NormParams &p, hipStream_t s) {
    const unsigned waves = (unsigned)((p.rows + 3) / 4), groups = (unsigned)p.rows;
    const int per = (p.D + 64 * V - 1) / (64 * V);   // vectors per lane of one wave
#define FW_NORM(TPR, NV, GRID) norm_fwd_kernel<TX, TR, V, TPR, NV, E4M3><<<GRID, kNormThreads, 0, s>>>(p)
    constexpr int M = 32 / V;
    if (per <= M / 8) FW_NORM(64, M / 8, waves);
    else if (per <= M / 4) FW_NORM(64, M / 4, waves);
    else if (per <= M / 2) FW_NORM(64, M / 2, waves);
    else if (per <= M) FW_NORM(64, M, waves);
    else if (per <= 2 * M) FW_NORM(256, M / 2, groups);
    else if (per <= 4 * M) FW_NORM(256, M, groups);
    else FW_NORM(256, 0, groups);
#undef FW_NORM
    return (int)hipGetLastError();
}

template <typename TX, typename TR, int V>
int bwd_by_size(const NormBwdParams &p, hipStream_t s) {
    const int per = (p.D + 64 * V - 1) / (64 * V);
    constexpr int M = 32 / V;
#define FW_NORM(TPR, NV) norm_bwd_kernel<TX, TR, V, TPR, NV><<<(unsigned)p.blocks, kNormThreads, 0, s>>>(p)
    if (per <= M / 4) FW_NORM(64, M / 4);
    else if (per <= M / 2) FW_NORM(64, M / 2);
    else if (per <= M) FW_NORM(64, M);
    else if (per <= 2 * M) FW_NORM(256, M / 2);
    else if (per <= 4 * M) FW_NORM(256, M);
    else if (per <= 8 * M) FW_NORM(256, 2 * M);
    else return -1;
#undef FW_NORM
    const int r = (int)hipGetLastError();
    if (r) return r;
    norm_join_kernel<<<(unsigned)((p.D + 31) / 32), 256, 0, s>>>(p.part, p.gweight, p.D, p.blocks);
    return (int)hipGetLastError();
}

bool al(const void *p) { return ((uintptr_t)p & 15) == 0; }

template <typename TX, typename TR>
int fwd_types(const NormParams &p, bool e4m3, hipStream_t s) {
    const bool vec = p.D % 4 == 0 && al(p.x) && al(p.residual) && al(p.weight) && al(p.out) && al(p.sum);
    if (e4m3) return vec ? fwd_by_size<TX, TR, 4, true>(p, s) : fwd_by_size<TX, TR, 1, true>(p, s);
    return vec ? fwd_by_size<TX, TR, 4, false>(p, s) : fwd_by_size<TX, TR, 1, false>(p, s);
}
template <typename TX, typename TR>
int bwd_types(const NormBwdParams &p, hipStream_t s) {
    const bool vec = p.D % 4 == 0 && al(p.sum) && al(p.weight) && al(p.go) && al(p.gsum) && al(p.gx) && al(p.gres) && al(p.part);
    return vec ? bwd_by_size<TX, TR, 4>(p, s) : bwd_by_size<TX, TR, 1>(p, s);
}

}  // namespace

int norm_bwd_blocks(int64_t rows, int D) {
    const int64_t groups = D <= 2048 ? (rows + 3) / 4 : rows;
    return (int)(groups < kNormBlocks ? groups : kNormBlocks);
}

int launch_norm_fwd(const NormParams &p, bool x_bf16, bool r_bf16, bool e4m3, hipStream_t s) {
    if (!x_bf16) return fwd_types<float, float>(p, e4m3, s);
    return r_bf16 ? fwd_types<__bf16, __bf16>(p, e4m3, s) : fwd_types<__bf16, float>(p, e4m3, s);
}
int launch_norm_bwd(const NormBwdParams &p, bool x_bf16, bool r_bf16, hipStream_t s) {
    if (!x_bf16) return bwd_types<float, float>(p, s);
    return r_bf16 ? bwd_types<__bf16, __bf16>(p, s) : bwd_types<__bf16, float>(p, s);
}

}  // namespace fw

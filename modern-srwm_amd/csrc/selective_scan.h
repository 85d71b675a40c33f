// Shared by the selective-scan kernels (selective_scan.hip, selective_scan_bwd.hip): the parameter block, the layout of
// a channel over lanes, and the elementary functions.
//
// Recurrence of one channel (state of S numbers, diagonal decay that depends on the step):
//     dt_t = softplus(delta_t + bias)
//     h_t  = exp(dt_t A) h_{t-1} + dt_t u_t B_t          (h_{t-1} := 0 where keep_t == 0)
//     y_t  = C_t . h_t + D u_t,      out_t = y_t silu(z_t)
// B_t and C_t are shared by all channels of a group of heads; the sums over s run inside a channel, those of the
// gradients of B and C over channels.
//
// Layout: a channel sits on the four lanes of a quad, SPL = S / 4 of its states on each (sizes in between are padded
// with zero states).  Three things decide for four: the reduction over s is two DPP steps, a wave covers 16 channels so
// that a single sequence already fills many waves, and the work that a channel has once per step (softplus, gate,
// addresses, loads, stores) is spread over time instead -- lane j of the quad does it for the steps 4i + j and hands
// the results round by DPP, so it is paid once per step and not four times.
#pragma once

#include <hip/hip_runtime.h>

#include "common.h"
#include "gates.h"
#include "vec_io.h"
#include "xlane.h"

namespace fw {

constexpr int kScanBlock = 16;      // steps between two saved states, and per stage of B and C in LDS
constexpr int kScanThreads = 256;   // 4 waves
// Times in these files: single figures are of long runs (300 passes).  Figures that compare two forms are of runs of about ten
// passes, at lower clocks, which makes those of the scan up to a fifth longer; where they are of long runs they say so.
//
// A call of few waves is cut into segments until it has kScanWaves (four on each SIMD), at the price of the pass that
// forms the segments' own results, 0.6 of the forward and 0.2 of the backward.  2048 channels and 16 states, long runs, ms
// without / with: forward 16 x 1024 steps (2 048 waves) 0.186 / 0.219, 8 x 2048 (1 024 waves) 0.245 / 0.232, 4 x 2048 (512
// waves) 0.244 / 0.132; backward 16 x 1024 0.475 / 0.540, 8 x 2048 0.694 / 0.567.  At 1 024 waves the forward gains a
// twentieth by segments, and the call would need their workspace: it is left whole.
constexpr int kScanWaves = 4096, kScanEnoughFwd = 1024, kScanEnoughBwd = 2048;
// The backward's main pass runs kScanBwdWaves at a time (two on each SIMD).  Segments shorter than kScanBwdShort are not
// worth a second round of them, long ones are, as their rounds overlap (both kernels of the pass, us with segments for two
// rounds / one: 32 x 100 steps x 8 groups of 32 channels 46.7 / 43.0, 4 x 512 x 2048 with 64 states 507 / 482; 4 x 2048 x
// 2048 328 / 332, 8 x 1000 x 16 groups of 32 155 / 162).
constexpr int kScanBwdWaves = 2048, kScanBwdShort = 96;
// Shortest segment.  A segment also joins those in front of it one after the other, so their number n is bounded by their
// length: n^2 <= steps forward, 4 steps backward (1 x 100000 steps of 64 channels, the two kernels of a pass, ms: n^2 <=
// steps 0.130 + 0.236, 4 steps 0.139 + 0.224, 16 steps 0.189 + 0.254).
// Rows of different lengths keep both bounds, by the longest of them (64 channels, 12001 steps and 31 rows of 64, forward and
// with the backward: up to 751 segments of the long row 141 and 344 us, within the bounds 54 and 190; 100000 steps and three
// rows of one 198 and 517 against 131 and 412).

// From four values per lane to one: lane j of each quad ends up with the quad's sum of v[j].
__device__ __forceinline__ float quad_sum_scatter(float v0, float v1, float v2, float v3, int lane) {
    const bool b0 = lane & 1, b1 = lane & 2;
    const float r0 = (b0 ? v1 : v0) + dpp_mov<kDppXor1>(b0 ? v0 : v1);
    const float r1 = (b0 ? v3 : v2) + dpp_mov<kDppXor1>(b0 ? v2 : v3);
    return (b1 ? r1 : r0) + dpp_mov<kDppXor2>(b1 ? r0 : r1);
}
// The value of lane j of the quad (j a constant after unrolling).
__device__ __forceinline__ float quad_lane(float v, int j) {
    return j == 0 ? quad_broadcast<0>(v) : j == 1 ? quad_broadcast<1>(v) : j == 2 ? quad_broadcast<2>(v) : quad_broadcast<3>(v);
}

// A workgroup's place in the grid: x = batch row and tile of 64 channels, y = group, z = segment of the steps.
// One lane's place in it: its channel and its states [q * SPL, q * SPL + SPL).
struct ScanLane {
    int n, tile, g, h0;   // of the workgroup; h0: head of its first channel
    int h, e, d;          // head, channel of the head, channel of the tensor [H*E]
    int q, lane, wave;
    bool on;              // false: a lane behind the group's last channel (reads the last one, writes nothing)
    // false: a wave without a channel, which only helps to stage B and C (8 x 1000 steps, 16 groups of 32 channels: forward 74.6
    // -> 60.2 us).  The backward's main pass walks it through all the same: leaving it out gained 2 % there.
    bool busy;
};
__device__ __forceinline__ ScanLane scan_lane(const ScanParams &p, int n) {
    ScanLane r;
    r.n = n, r.tile = blockIdx.x / p.N, r.g = blockIdx.y;
    r.lane = threadIdx.x & 63;
    r.wave = threadIdx.x >> 6;
    r.q = r.lane & 3;
    const int Dg = (p.H / p.G) * p.E;
    int c = r.tile * kScanTile + r.wave * 16 + (r.lane >> 2);
    r.on = c < Dg;
    r.busy = __builtin_amdgcn_readfirstlane(r.tile * kScanTile + r.wave * 16) < Dg;
    c = r.on ? c : Dg - 1;
    r.d = r.g * Dg + c;
    r.h = r.d / p.E;
    r.e = r.d % p.E;
    r.h0 = (r.g * Dg + r.tile * kScanTile) / p.E;
    return r;
}
__device__ __forceinline__ int row_length(const ScanParams &p, int n) {
    return p.lengths ? min(max(p.lengths[n], 0), p.L) : p.L;
}

// A workgroup's run of steps: segment `seg` of the `count` that row n is cut into, steps [tbeg, tend); the segments'
// results stand side by side from slot `first` on.
struct ScanRun {
    int n, len, seg, count, tbeg, tend;   // len: steps of the row
    int64_t first;
    bool used;
};
// Rows of one length: every row has p.segments segments.  Rows of different lengths: the segments are of one length over
// all rows, so that no workgroup of a short row stands idle beside those of a long one; (slots - N) of them cover all steps,
// and N more what is left over at the rows' ends.  Longer segments, where the longest row would join too many, leave slots
// empty.  Every wave works this out for itself (n, seg: the workgroup's place).
__device__ __forceinline__ ScanRun scan_run(const ScanParams &p, int n, int seg) {
    ScanRun r;
    r.used = true;
    if (!p.lengths || p.segments == 1) {
        r.n = n, r.seg = seg, r.count = p.segments, r.len = row_length(p, n);
        r.first = (int64_t)n * p.segments;
        r.tbeg = seg * p.seg_len, r.tend = min(r.tbeg + p.seg_len, r.len);
        return r;
    }
    const int lane = threadIdx.x & 63;
    int64_t total = 0;
    int longest = 0;
    for (int b = 0; b < p.N; b += 64) {
        const int v = b + lane < p.N ? row_length(p, b + lane) : 0;
        int64_t s = v;
        int most = v;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            s += __shfl_xor((long long)s, off, kWave);
            most = max(most, __shfl_xor(most, off, kWave));
        }
        total += s;
        longest = max(longest, most);
    }
    const int64_t slots = (int64_t)p.N * p.segments - p.N;
    int64_t sl = (total + slots - 1) / slots;
    sl = max((sl + kScanBlock - 1) / kScanBlock * kScanBlock, (int64_t)kScanMinSegment);
    while (sl * sl * p.seg_join < longest) sl += kScanBlock;   // (longest / sl)^2 <= seg_join * longest
    const int seg_len = __builtin_amdgcn_readfirstlane((int)sl);   // the same in every lane: in a scalar register
    int at = seg * p.N + n;
    r.used = false, r.n = 0, r.seg = 0, r.count = 1, r.len = 0, r.first = 0, r.tbeg = 0, r.tend = 0;
    int64_t before = 0;   // slots of the rows in front of this batch of 64
    for (int b = 0; b < p.N && !r.used; b += 64) {
        const int v = b + lane < p.N ? row_length(p, b + lane) : 0;
        const int c = b + lane < p.N ? max((v + seg_len - 1) / seg_len, 1) : 0;
        int incl = c;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int t = __shfl_up(incl, off, kWave);
            incl += lane >= off ? t : 0;
        }
        const unsigned long long hit = __ballot(incl > at - before);
        if (hit) {
            const int f = __ffsll((long long)hit) - 1;
            r.used = true;
            r.n = b + f;
            r.count = __builtin_amdgcn_readlane(c, f);
            r.len = __builtin_amdgcn_readlane(v, f);
            r.first = before + __builtin_amdgcn_readlane(incl, f) - r.count;
            r.seg = (int)(at - r.first);
            r.tbeg = r.seg * seg_len, r.tend = min(r.tbeg + seg_len, r.len);
        }
        before += __builtin_amdgcn_readlane(incl, 63);
    }
    return r;
}
// The share of the steps behind row n's end that the workgroups at its places (n, seg) fill with zeros, seg of p.segments,
// whatever run they had: the rows with the most steps behind their end have the fewest runs (4 rows of 64 channels, 100000
// steps and three of 1: forward 1187 -> 198 us, with the backward 2776 -> 517).
__device__ __forceinline__ void behind_share(const ScanParams &p, int n, int seg, int &from, int &to) {
    const int len = row_length(p, n), each = (p.L - len + p.segments - 1) / p.segments;
    from = (int)min((int64_t)len + (int64_t)seg * each, (int64_t)p.L), to = min(from + each, p.L);
}

// Elements (t, channel) of a strided [N,H,L,E] tensor as one address per workgroup and step (scalar registers) plus one
// offset per lane that never changes: a load is then one instruction without address arithmetic in the vector unit.
// OFF: unsigned 32-bit byte offsets, or int64_t where a workgroup's channels and 16 steps span 2 GiB or more.
template <typename T, typename OFF>
struct ScanRows {
    char *base;     // element (n, h0, t, 0) of the block's first step t; uniform
    int64_t step;   // bytes between two steps; uniform
    OFF off;        // of this lane's channel
    __device__ __forceinline__ ScanRows(const void *p, const Strided3 &s, const ScanLane &w, int t)
        : base((char *)p + (w.n * s.n + w.h0 * s.h + t * s.l) * (int64_t)sizeof(T)), step(s.l * (int64_t)sizeof(T)),
          off((OFF)(((w.h - w.h0) * s.h + w.e) * (int64_t)sizeof(T))) {}
    __device__ __forceinline__ void move(int steps) { base += steps * step; }
    // the element of step 4i + k (i uniform; k >= 0: the lane's share)
    __device__ __forceinline__ T *at(int i, int k) const { return (T *)(base + 4 * i * step + (OFF)(off + (OFF)(k * step))); }
};

// The elements of B and C that a thread stages in LDS: row r + R * k' of a block of 16, element s.
template <typename T, int SPL>
struct ScanBc {
    static constexpr int SP = 4 * SPL, kRows = kScanThreads / SP;      // rows of B or C per pass of the workgroup
    static constexpr int kEach = kRows >= kScanBlock ? 1 : kScanBlock / kRows;
    static constexpr bool kSplit = kRows > kScanBlock;                 // half of the workgroup stages B, the other half C
    const T *b, *c;
    int64_t bs, cs;
    int row, s;
    bool pad;
    __device__ __forceinline__ ScanBc(const ScanParams &p, const ScanLane &w, int t) {
        const int i = threadIdx.x;
        s = i % SP, row = i / SP % kScanBlock;
        pad = s >= p.S;
        const int sc = pad ? 0 : s;
        b = (const T *)p.B + w.n * p.Bs.n + w.g * p.Bs.h + t * p.Bs.l + sc;
        c = (const T *)p.C + w.n * p.Cs.n + w.g * p.Cs.h + t * p.Cs.l + sc;
        bs = p.Bs.l, cs = p.Cs.l;
        if (kSplit && i / SP >= kScanBlock) b = c, bs = cs;
    }
    __device__ __forceinline__ void move(int steps) { b += steps * bs, c += steps * cs; }
    // n: steps from the block's first one to the sequence's end; rows behind it read the last one
    __device__ __forceinline__ void fetch(T (&vb)[kEach], T (&vc)[kEach], int n, bool with_c) const {
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int t = min(row + k * kRows, n - 1);
            vb[k] = b[t * bs];
            if (!kSplit && with_c) vc[k] = c[t * cs];
        }
    }
    // dst: [2][16][SP]; rows behind the end are staged as zeros
    __device__ __forceinline__ void stage(float *dst, const T (&vb)[kEach], const T (&vc)[kEach], int n, bool with_c) const {
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const bool none = pad || row + k * kRows >= n;
            const int i = threadIdx.x + k * kScanThreads;
            dst[i] = none ? 0.f : (float)vb[k];
            if (!kSplit && with_c) dst[kScanBlock * SP + i] = none ? 0.f : (float)vc[k];
        }
    }
};

// A segment's product of decays 2^e is handed on as its root: the product itself may leave float32's range where the state that
// it is applied to, in two steps, does not.  After a reset in the segment nothing of the state in front passes, not even NaN.
// No power of two has these bits.
constexpr float kDropped = -0.f;
__device__ __forceinline__ float decay_root(float e, bool alive) { return alive ? __builtin_amdgcn_exp2f(0.5f * e) : kDropped; }
// A state of zero passes as zero through decays whose product overflows all the same.
__device__ __forceinline__ float carried(float root, float x, float result) {
    return __float_as_uint(root) == 0x80000000u || x == 0.f ? result : fmaf(root * x, root, result);
}

// Whether a workgroup's lanes lie 2 GiB or more apart in rows of these strides (64 channels, 16 steps).
inline bool scan_span(const ScanParams &p, const Strided3 &s, int64_t bytes) {
    const auto mag = [](int64_t x) { return x < 0 ? -x : x; };
    const int64_t heads = (kScanTile + p.E - 2) / p.E;   // heads that a tile reaches beyond its first
    return (heads * mag(s.h) + kScanBlock * mag(s.l) + p.E) * bytes >= ((int64_t)1 << 31) || s.h < 0 || s.l < 0;
}

// SPL consecutive states of a row of S; those behind S read as zero and are not written
template <int SPL>
__device__ __forceinline__ void load_states(const float *row, int S, int q, float (&v)[SPL]) {
    if (S == 4 * SPL && SPL % 4 == 0) {
#pragma unroll
        for (int i = 0; i < SPL; i += 4) {
            const float4 r = *reinterpret_cast<const float4 *>(row + q * SPL + i);
            v[i] = r.x, v[(i + 1) % SPL] = r.y, v[(i + 2) % SPL] = r.z, v[(i + 3) % SPL] = r.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < SPL; ++i) v[i] = q * SPL + i < S ? row[q * SPL + i] : 0.f;
    }
}
// A channel's decays, in units of log2(e).  An infinite one is kept finite, so that the steps behind a row's end (dt = 0)
// pass the state on there too.
template <int SPL>
__device__ __forceinline__ void load_decays(const float *row, int S, int q, float (&v)[SPL]) {
    load_states<SPL>(row, S, q, v);
#pragma unroll
    for (int i = 0; i < SPL; ++i) {
        const float a = v[i] * kLog2e;
        v[i] = a < -3e38f ? -3e38f : a > 3e38f ? 3e38f : a;
    }
}
// states (or B, C) from a row of fp32 or bf16 elements that may start anywhere
template <int SPL, typename T>
__device__ __forceinline__ void load_io_states(const T *row, int S, int q, float (&v)[SPL]) {
    if (S == 4 * SPL && ((uintptr_t)row & (sizeof(T) * SPL - 1)) == 0 && sizeof(T) * SPL <= 16) {
        load_vec<SPL>(row + q * SPL, v);
    } else {
#pragma unroll
        for (int i = 0; i < SPL; ++i) v[i] = q * SPL + i < S ? io_load(row + q * SPL + i) : 0.f;
    }
}
template <int SPL>
__device__ __forceinline__ void store_states(float *row, int S, int q, const float (&v)[SPL]) {
    if (S == 4 * SPL && SPL % 4 == 0) {
#pragma unroll
        for (int i = 0; i < SPL; i += 4)
            *reinterpret_cast<float4 *>(row + q * SPL + i) = make_float4(v[i], v[(i + 1) % SPL], v[(i + 2) % SPL], v[(i + 3) % SPL]);
    } else {
#pragma unroll
        for (int i = 0; i < SPL; ++i)
            if (q * SPL + i < S) row[q * SPL + i] = v[i];
    }
}

// Carries a state (or its gradient) over `count` segments from the one at `at` on, `stride` floats from one to the next:
// x = root^2 x + result.  Four segments are asked for at a time (two above 16 states; eight take the forward from five to
// three waves a SIMD): one after the other would cost a trip to memory each, as they were written by other dies.
template <int SPL>
__device__ __forceinline__ void join_segments(const ScanParams &p, int64_t at, int64_t stride, int count, int S, int q, float (&x)[SPL]) {
    constexpr int U = SPL <= 4 ? 4 : 2;
    int k = 0;
    if (S == 4 * SPL && SPL % 4 == 0) {
        for (; k + U <= count; k += U) {
            float4 pr[U][(SPL + 3) / 4], r[U][(SPL + 3) / 4];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int64_t o = at + (k + i) * stride + q * SPL;
#pragma unroll
                for (int s = 0; s < SPL / 4; ++s) {
                    pr[i][s] = reinterpret_cast<const float4 *>(p.seg_decay + o)[s];
                    r[i][s] = reinterpret_cast<const float4 *>(p.seg_state + o)[s];
                }
            }
#pragma unroll
            for (int i = 0; i < U; ++i)
#pragma unroll
                for (int s = 0; s < SPL; ++s) {
                    const float d = (&pr[i][s / 4].x)[s % 4], v = (&r[i][s / 4].x)[s % 4];
                    x[s] = carried(d, x[s], v);
                }
        }
    }
    for (; k < count; ++k) {
        float pr[SPL], r[SPL];
        load_states<SPL>(p.seg_decay + at + k * stride, S, q, pr);
        load_states<SPL>(p.seg_state + at + k * stride, S, q, r);
#pragma unroll
        for (int s = 0; s < SPL; ++s) x[s] = carried(pr[s], x[s], r[s]);
    }
}

}  // namespace fw

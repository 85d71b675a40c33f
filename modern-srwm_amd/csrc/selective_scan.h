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

// One lane's place: its channel, its states [q * SPL, q * SPL + SPL), and where they live.
struct ScanLane {
    int h, e, d;        // head, channel of the head, channel of the tensor [H*E]
    int q, lane, wave;
    bool on;            // false: a lane behind the group's last channel (reads the last one, writes nothing)
};
__device__ __forceinline__ ScanLane scan_lane(int H, int E, int G, int tile, int g) {
    ScanLane r;
    r.lane = threadIdx.x & 63;
    r.wave = threadIdx.x >> 6;
    r.q = r.lane & 3;
    const int Dg = (H / G) * E;
    int c = tile * kScanTile + r.wave * 16 + (r.lane >> 2);
    r.on = c < Dg;
    c = r.on ? c : Dg - 1;
    r.d = g * Dg + c;
    r.h = r.d / E;
    r.e = r.d % E;
    return r;
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

}  // namespace fw

// selective_scan.cuh -- what the forward and the backward of the selective
// scan share: the tiling, the staging of a warp's time steps, the kernel block.
//
//   dt = softplus(delta + bias),  u = dt x,  a[n] = exp(dt A[n])
//   h[n] <- a[n] h[n] + u B[n],   y = sum_n C[n] h[n] + D x,   out = y z sigmoid(z)
//
// Tiling.  A thread owns 4 neighbouring states of 2 neighbouring features; NL
// lanes side by side cover up to 4 NL states and the 32 / NL lane groups 64 / NL
// features.  So B and C (one row of states per time step, shared by the
// features) cost one 16-byte shared-memory load each per 8 state updates, dt and
// u another, and the sums over the states are log2(NL) lane exchanges.
//
// Time.  The warps of a block hold consecutive runs of 8 steps of the same
// features.  Each computes its run's exponentials once and keeps them in
// registers, runs the recurrence from h = 0, and publishes the run's product of
// decays P and end state E: h_out = P h_in + E.  After one barrier every warp
// chains the runs before its own and runs its steps again from the true state
// with the decays that it kept.  The exponentials, which bound the kernel (16
// per SM and cycle), are computed once each whatever the number of warps.
#pragma once

#include "seq_device.cuh"
#include "seq_kernels.h"

namespace sdtw {

constexpr int kScanSteps = 8;                        // time steps of a warp's run
constexpr int kScanWarps = kScanChunk / kScanSteps;  // 4
constexpr int kScanThreads = 32 * kScanWarps;
constexpr int kCT = 2;  // features per thread
constexpr float kL2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <int NL>
struct ScanTile {
    static constexpr int CL = 32 / NL;     // lane groups over features
    static constexpr int CH = CL * kCT;    // features per block
    static constexpr int NP = 4 * NL;      // states, padded
    static constexpr int VX = CH / 4;      // features of a staging lane (4 lanes per time step)
    static constexpr int VN = NL;          // states of a staging lane
};

struct ScanP {
    sdtw_scan_args a;
    int dg;       // features per group
    int tiles_g;  // blocks per group
    int nchunk;
    bool vec_x, vec_delta, vec_z, vec_B, vec_C, vec_y, vec_dy, vec_dx, vec_ddelta, vec_dz;
    bool vec_n;   // the states of a thread are 16 bytes aligned
    float* part_bc;   // (tiles, batch, length, 2, NP) partial dB, dC
    float* part_par;  // (batch, dim * nstate + 2 * dim) partial dA, dD, ddelta_bias
};

// The block's place: batch entry, first feature and how many of them exist.
template <int NL>
struct ScanPlace {
    int b, tile, g, c0, nc;
    __device__ __forceinline__ explicit ScanPlace(const ScanP& p) {
        const int tiles = p.tiles_g * p.a.groups;
        b = blockIdx.x / tiles;
        tile = blockIdx.x % tiles;
        g = tile / p.tiles_g;
        const int first = (tile % p.tiles_g) * ScanTile<NL>::CH;
        c0 = g * p.dg + first;
        nc = min(ScanTile<NL>::CH, p.dg - first);
    }
};

// A thread's 4 states of 2 features, as pairs [feature][pair].
struct St {
    f2 v[kCT][2];
};
__device__ __forceinline__ void st_set(St& s, float x) {
#pragma unroll
    for (int i = 0; i < kCT; ++i) s.v[i][0] = s.v[i][1] = pk(x, x);
}
// s <- P s + E with the run's P and E in shared memory ([feature][lane]).
__device__ __forceinline__ void st_chain(St& s, const ulonglong2 (*P)[32], const ulonglong2 (*E)[32], int lane) {
#pragma unroll
    for (int i = 0; i < kCT; ++i) {
        const ulonglong2 q = P[i][lane], e = E[i][lane];
        s.v[i][0] = fma2(f2{q.x}, s.v[i][0], f2{e.x});
        s.v[i][1] = fma2(f2{q.y}, s.v[i][1], f2{e.y});
    }
}
__device__ __forceinline__ void st_put(ulonglong2 (*d)[32], int lane, const St& s) {
#pragma unroll
    for (int i = 0; i < kCT; ++i) d[i][lane] = make_ulonglong2(s.v[i][0].v, s.v[i][1].v);
}
__device__ __forceinline__ void st_get(St& s, const ulonglong2 (*d)[32], int lane) {
#pragma unroll
    for (int i = 0; i < kCT; ++i) {
        const ulonglong2 q = d[i][lane];
        s.v[i][0].v = q.x;
        s.v[i][1].v = q.y;
    }
}
// States n0 .. n0 + 4 of features f and f + 1 of a (features, S) table; those
// that do not exist read as 0 and are not written.
__device__ __forceinline__ void st_load(St& s, const float* tab, int f, int nf, int S, int n0, bool vec) {
#pragma unroll
    for (int i = 0; i < kCT; ++i) {
        Vec<float, 4> r;
        const int n = f + i < nf ? min(max(S - n0, 0), 4) : 0;
        r.load_n(tab + static_cast<long long>(f + i) * S + n0, n, vec);
        s.v[i][0] = pk(r.get(0), r.get(1));
        s.v[i][1] = pk(r.get(2), r.get(3));
    }
}
__device__ __forceinline__ void st_store(const St& s, float* tab, int f, int nf, int S, int n0, bool vec) {
#pragma unroll
    for (int i = 0; i < kCT; ++i) {
        Vec<float, 4> r;
        float v[4];
        upk(s.v[i][0], v[0], v[1]);
        upk(s.v[i][1], v[2], v[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) r.set(j, v[j]);
        const int n = f + i < nf ? min(max(S - n0, 0), 4) : 0;
        r.store_n(tab + static_cast<long long>(f + i) * S + n0, n, vec);
    }
}

template <typename T, int NL>
inline void scan_params(ScanP& p, const sdtw_scan_args& a) {
    using K = ScanTile<NL>;
    p.a = a;
    p.dg = a.dim / a.groups;
    p.tiles_g = (p.dg + K::CH - 1) / K::CH;
    p.nchunk = (a.length + kScanChunk - 1) / kScanChunk;
    const bool d = p.dg % K::VX == 0 && a.dim % K::VX == 0;
    const long long ds = a.dim;
    p.vec_x = d && vec_ok<T, K::VX>(a.x, a.x_batch, a.x_time);
    p.vec_delta = d && vec_ok<T, K::VX>(a.delta, a.delta_batch, a.delta_time);
    p.vec_z = d && vec_ok<T, K::VX>(a.z, a.z_batch, a.z_time);
    p.vec_y = d && vec_ok<T, K::VX>(a.y, ds, 0);
    p.vec_dy = d && vec_ok<T, K::VX>(a.dy, a.dy_batch, a.dy_time);
    p.vec_dx = d && vec_ok<T, K::VX>(a.dx, ds, 0);
    p.vec_ddelta = d && vec_ok<T, K::VX>(a.ddelta, ds, 0);
    p.vec_dz = d && vec_ok<T, K::VX>(a.dz, ds, 0);
    const bool n = a.nstate % K::VN == 0;
    p.vec_B = n && vec_ok<T, K::VN>(a.B, a.B_batch, a.B_time, a.B_group);
    p.vec_C = n && vec_ok<T, K::VN>(a.C, a.C_batch, a.C_time, a.C_group);
    p.vec_n = a.nstate % 4 == 0 && vec_ok<float, 4>(a.A, 0, 0) && vec_ok<float, 4>(a.state_in, a.state_in_batch, 0) &&
              vec_ok<float, 4>(a.state_out, a.state_out_batch, 0) && vec_ok<float, 4>(a.saved, 0, 0) &&
              vec_ok<float, 4>(a.dstate_in, 0, 0) && vec_ok<float, 4>(a.dstate_out, 0, 0);
}

// Lanes over the states of a feature.
inline int scan_lanes(int nstate) {
    int nl = 1;
    while (4 * nl < nstate) nl *= 2;
    return nl;
}

template <int NL>
inline long long scan_blocks(const ScanP& p) {
    return static_cast<long long>(p.tiles_g) * p.a.groups * p.a.batch;
}

}  // namespace sdtw

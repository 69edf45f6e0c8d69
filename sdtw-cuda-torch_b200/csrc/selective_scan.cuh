// selective_scan.cuh -- what the forward and the backward of the selective
// scan share: the tiling, the split of the time axis, the kernel block.
//
//   dt = softplus(delta + bias),  u = dt x,  a[n] = exp(dt A[n])
//   h[n] <- a[n] h[n] + u B[n],   y = sum_n C[n] h[n] + D x,   out = y z sigmoid(z)
//
// Tiling.  A thread owns 4 neighbouring states of 2 neighbouring features; NL
// lanes side by side cover up to 4 NL states and the 32 / NL lane groups 64 / NL
// features.  So B and C (one row of states per time step, shared by the
// features) cost one 16-byte shared-memory load each per 8 state updates, dt and
// u another, and the sums over the states are log2(NL) lane exchanges.  A warp
// walks over the time steps; dt, u, B and C of TS steps at a time are staged in
// shared memory, the elementwise functions computed once per element there.
//
// Time.  When there are too few warps to fill the GPU, the time axis is cut into
// segments: a first kernel runs each from h = 0 and keeps its end state E and
// the sum of its dt (whose exponential with A is the product of the decays), and
// the main kernel's warps chain the segments before their own,
// h <- exp(A sum dt) h + E, before they start.  The exponentials are then
// computed twice.
#pragma once

#include "seq_device.cuh"
#include "seq_kernels.h"

namespace sdtw {

constexpr int kScanWarps = 4;
constexpr int kScanThreads = 32 * kScanWarps;
constexpr int kCT = 2;     // features per thread
constexpr int kRun = 8;    // time steps held in registers
constexpr float kL2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <int NL>
struct ScanTile {
    static constexpr int CL = 32 / NL;               // lane groups over features
    static constexpr int CH = CL * kCT;              // features per warp
    static constexpr int NP = 4 * NL;                // states, padded
    static constexpr int TS = scan_stage_steps(NL);  // staged time steps
    static constexpr int LR = 32 / TS;               // staging lanes per time step
    static constexpr int VX = CH / LR;               // features of a staging lane
    static constexpr int VN = NP / LR;               // states of a staging lane
};

struct ScanP {
    sdtw_scan_args a;
    int dg;        // features per group
    int tiles_g;   // warps' tiles per group
    int nchunk;    // stored states per series
    int nseg, seglen;
    bool vec_x, vec_delta, vec_z, vec_B, vec_C, vec_y, vec_dy, vec_dx, vec_ddelta, vec_dz;
    bool vec_n;    // the states of a thread are 16 bytes aligned
    float* seg_dt;    // (batch, nseg, dim) sums of dt
    float* seg_E;     // (batch, nseg, dim, nstate) end states of the segments run from 0
    float* part_bc;   // backward: (blocks over features, batch, length, 2, NP) partial dB, dC
    float* part_par;  // backward: (batch, nseg, dim * nstate + 2 * dim) partial dA, dD, ddelta_bias
};

// A warp's place.  `tile` counts the warps over the features, all groups.
template <int NL>
struct ScanPlace {
    int b, seg, g, c0, nc;
    int t0, t1;  // the segment
    __device__ __forceinline__ ScanPlace(const ScanP& p, int batch, int segment, int group, int tile_in_group) {
        b = batch;
        seg = segment;
        g = group;
        const int first = tile_in_group * ScanTile<NL>::CH;
        c0 = g * p.dg + first;
        nc = max(0, min(ScanTile<NL>::CH, p.dg - first));
        t0 = seg * p.seglen;
        t1 = min(t0 + p.seglen, p.a.length);
    }
    __device__ static __forceinline__ ScanPlace of_warp(const ScanP& p, long long i) {
        const int tiles = p.tiles_g * p.a.groups;
        const int tile = static_cast<int>(i % tiles);
        const long long bs = i / tiles;
        return ScanPlace(p, static_cast<int>(bs / p.nseg), static_cast<int>(bs % p.nseg), tile / p.tiles_g, tile % p.tiles_g);
    }
};

// A thread's 4 states of 2 features, as pairs [feature][pair].  Lanes with an
// odd state group hold their two features swapped (see pair_exchange).
struct St {
    f2 v[kCT][2];
};
__device__ __forceinline__ void st_set(St& s, float x) {
#pragma unroll
    for (int i = 0; i < kCT; ++i) s.v[i][0] = s.v[i][1] = pk(x, x);
}
// States n0 .. n0 + 4 of features f + (0 ^ swap) and f + (1 ^ swap) of a
// (features, S) table; those that do not exist read as 0 and are not written.
__device__ __forceinline__ void st_load(St& s, const float* tab, int f, int swap, int nf, int S, int n0, bool vec) {
#pragma unroll
    for (int i = 0; i < kCT; ++i) {
        const int c = f + (i ^ swap);
        Vec<float, 4> r;
        const int n = c < nf ? min(max(S - n0, 0), 4) : 0;
        r.load_n(tab + static_cast<long long>(c) * S + n0, n, vec);
        s.v[i][0] = pk(r.get(0), r.get(1));
        s.v[i][1] = pk(r.get(2), r.get(3));
    }
}
__device__ __forceinline__ void st_store(const St& s, float* tab, int f, int swap, int nf, int S, int n0, bool vec) {
#pragma unroll
    for (int i = 0; i < kCT; ++i) {
        const int c = f + (i ^ swap);
        Vec<float, 4> r;
        float v[4];
        upk(s.v[i][0], v[0], v[1]);
        upk(s.v[i][1], v[2], v[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) r.set(j, v[j]);
        const int n = c < nf ? min(max(S - n0, 0), 4) : 0;
        r.store_n(tab + static_cast<long long>(c) * S + n0, n, vec);
    }
}
// h <- exp(A sum dt) h + E over one segment.
__device__ __forceinline__ void st_chain(St& h, const ScanP& p, const St& A2, int b, int seg, int f, int swap, int nf, int n0) {
    const long long row = static_cast<long long>(b) * p.nseg + seg;
    St E;
    st_load(E, p.seg_E + row * p.a.dim * p.a.nstate, f, swap, nf, p.a.nstate, n0, p.vec_n);
#pragma unroll
    for (int i = 0; i < kCT; ++i) {
        const int c = f + (i ^ swap);
        const float d = c < nf ? __ldg(p.seg_dt + row * p.a.dim + c) : 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) h.v[i][j] = fma2(ex22(mul2(pk(d, d), A2.v[i][j])), h.v[i][j], E.v[i][j]);
    }
}
__device__ __forceinline__ void st_scale(St& s, float k) {
#pragma unroll
    for (int i = 0; i < kCT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) s.v[i][j] = mul2(s.v[i][j], pk(k, k));
}

template <typename T, int NL>
inline void scan_params(ScanP& p, const sdtw_scan_args& a) {
    using K = ScanTile<NL>;
    p.a = a;
    p.dg = a.dim / a.groups;
    p.tiles_g = (p.dg + K::CH - 1) / K::CH;
    p.nchunk = (a.length + K::TS - 1) / K::TS;
    const bool d = p.dg % K::VX == 0;
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

// The segments' tables at the start of a workspace, and their floats.
inline size_t scan_segment_floats(int batch, int nseg, int dim, int nstate) {
    return nseg > 1 ? static_cast<size_t>(batch) * nseg * dim * (nstate + 1) : 0;
}
inline void scan_segment_tables(ScanP& p, const ScanSplit& s, void* ws) {
    p.nseg = s.nseg;
    p.seglen = s.seglen;
    // The states first: their 16-byte pieces stay aligned.
    p.seg_E = static_cast<float*>(ws);
    p.seg_dt = p.seg_E + static_cast<size_t>(p.a.batch) * s.nseg * p.a.dim * p.a.nstate;
}

// The segments' first kernel: forward (u B added up) or backward over time
// (gy C added up, with gy = dy or dy z sigmoid(z)).
cudaError_t launch_scan_segments(const ScanP& p, bool reverse, cudaStream_t st);

}  // namespace sdtw

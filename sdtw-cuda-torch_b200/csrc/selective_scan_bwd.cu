// selective_scan_bwd.cu -- gradient of the selective scan (formulas and tiling:
// selective_scan.cuh).
//
// With gy = dL/dy before the gate and r the gradient that flows into a state
// from later steps, backwards over time:
//   gh[n] = gy C[n] + r[n],                    r[n] <- a[n] gh[n]
//   dC[n] = sum over features of gy h[n],      dB[n] = sum over features of gh[n] u
//   q = sum_n gh[n] B[n]                       (dL/du)
//   s = sum_n gh[n] a[n] h_prev[n] A[n]        (dL/d dt through the decays)
//   dA[n] += gh[n] a[n] h_prev[n] dt,          ddelta = (s + q x) softplus'(delta + bias)
//   dx = q dt + gy D,   dD += gy x,            dz = dout y (sigmoid(z) (1 + z (1 - sigmoid(z))))
//
// A warp walks over its staged pieces of TS steps from the last to the first,
// from the states that the forward stored at their starts.  It runs 8 steps
// forward, keeping their decays and states in registers (64 each per thread),
// then the same 8 backward; the first half of a 16-step piece is run forward
// once more in front of the second.  Reductions: the sums over the states of a
// feature and over the features of dB and dC are lane exchanges that halve the
// values at every step, mostly without selects, because the lanes hold their
// two features, and their four states, in an order that depends on the lane
// (two copies of dt, u and gy and four of B and C in shared memory provide it).
// The 4 warps of a block take neighbouring features of one group, add up their
// dB and dC in shared memory behind one barrier per piece, and share the staging
// of B and C; what is left per block goes to a partial table that a second
// kernel adds up in a fixed order, so results do not change from call to call.
#include <algorithm>

#include "selective_scan.cuh"

namespace sdtw {
namespace {

template <int NL>
struct BwdSmem {
    using K = ScanTile<NL>;
    static constexpr int NQ = K::CL < 4 ? K::CL : 4;  // copies of B and C: states permuted by n ^ q within fours
    float4 U[kScanWarps][2][K::TS][K::CH / 2];        // (dt, u) of two features; copy 1 swapped
    float2 G[kScanWarps][2][K::TS][K::CH / 2];        // gy
    // Per element, for the last step of a piece: x, softplus', dout times the gate's derivative ...
    float X[kScanWarps][K::TS][K::CH], D[kScanWarps][K::TS][K::CH], Z[kScanWarps][K::TS][K::CH];
    // ... and the sums q, s and y.
    float Q[kScanWarps][K::TS][K::CH], R[kScanWarps][K::TS][K::CH], Y[kScanWarps][K::TS][K::CH];
    // One more row than steps, so that the copies start in different banks.
    float B[2][NQ][K::TS + 1][K::NP], C[2][NQ][K::TS + 1][K::NP];
    float acc[2][kScanWarps][K::TS][2][K::NP];  // the warps' dB, dC
};

template <typename T, int NL>
__global__ void __launch_bounds__(kScanThreads, 2) scan_bwd_kernel(const ScanP p) {
    using K = ScanTile<NL>;
    using M = BwdSmem<NL>;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    M& sm = *reinterpret_cast<M*>(smem_raw);
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int quads = (p.tiles_g + kScanWarps - 1) / kScanWarps;  // blocks over a group's features
    const int gq = blockIdx.x % (quads * p.a.groups);
    const int bs = blockIdx.x / (quads * p.a.groups);
    const ScanPlace<NL> at(p, bs / p.nseg, bs % p.nseg, gq / quads, gq % quads * kScanWarps + w);
    const int nl = lane % NL, cl = lane / NL, swap = nl & 1, n0 = nl * 4, perm = cl & (M::NQ - 1);
    const int S = p.a.nstate, L = p.a.length, dim = p.a.dim;
    const int len = seq_len(p.a.lengths, at.b, L);
    const int f0 = at.c0 + cl * kCT, fend = at.c0 + at.nc;
    const int row = lane / K::LR, col = lane % K::LR * K::VX;
    const int nx = min(max(at.nc - col, 0), K::VX);
    // Staging of B and C: the block's 128 threads over TS rows.
    constexpr int BR = kScanThreads / K::TS, BN = (K::NP + BR - 1) / BR;
    const int brow = threadIdx.x / BR, bcol = threadIdx.x % BR * BN;

    St A2, dA, r;
    st_load(A2, p.a.A, f0, swap, fend, S, n0, p.vec_n);
    st_scale(A2, kL2e);
    // States in this lane's order: register j holds state n0 + (j ^ perm).
    auto permute = [&](St& s) {
#pragma unroll
        for (int i = 0; i < kCT; ++i) {
            float v[4], o[4];
            upk(s.v[i][0], v[0], v[1]);
            upk(s.v[i][1], v[2], v[3]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float a = perm & 1 ? v[j ^ 1] : v[j], b = perm & 1 ? v[j ^ 3] : v[j ^ 2];
                o[j] = perm & 2 ? b : a;
            }
            s.v[i][0] = pk(o[0], o[1]);
            s.v[i][1] = pk(o[2], o[3]);
        }
    };
    permute(A2);
    st_set(dA, 0.f);
    st_set(r, 0.f);
    if (p.a.dstate_out) {
        st_load(r, p.a.dstate_out + static_cast<long long>(at.b) * dim * S, f0, swap, fend, S, n0, p.vec_n);
        permute(r);
    }
    if (p.nseg > 1) {
        pdl_wait();
        permute(A2);
        permute(r);
        for (int q = p.nseg - 1; q > at.seg; --q) st_chain(r, p, A2, at.b, q, f0, swap, fend, n0);
        permute(A2);
        permute(r);
    }
    float dD[K::VX], dbias[K::VX];
#pragma unroll
    for (int e = 0; e < K::VX; ++e) dD[e] = dbias[e] = 0.f;
    const T* xp = static_cast<const T*>(p.a.x) + at.b * p.a.x_batch + at.c0 + col;
    const T* dp = static_cast<const T*>(p.a.delta) + at.b * p.a.delta_batch + at.c0 + col;
    const T* zp = static_cast<const T*>(p.a.z) + at.b * p.a.z_batch + at.c0 + col;
    const T* gp = static_cast<const T*>(p.a.dy) + at.b * p.a.dy_batch + at.c0 + col;
    const T* Bp = static_cast<const T*>(p.a.B) + at.b * p.a.B_batch + at.g * p.a.B_group;
    const T* Cp = static_cast<const T*>(p.a.C) + at.b * p.a.C_batch + at.g * p.a.C_group;
    const float* bias = p.a.delta_bias ? p.a.delta_bias + at.c0 + col : nullptr;
    const float* skip = p.a.D ? p.a.D + at.c0 + col : nullptr;
    const long long out0 = static_cast<long long>(at.b) * L * dim + at.c0 + col;

    Vec<T, K::VX> rx, rd, rz, rg;
    St h0;
    auto fetch = [&](int tc) {
        const int t = tc + row, n = t < len ? nx : 0;
        rx.load_n(xp + t * p.a.x_time, n, p.vec_x);
        rd.load_n(dp + t * p.a.delta_time, n, p.vec_delta);
        rg.load_n(gp + t * p.a.dy_time, n, p.vec_dy);
        if (p.a.z) rz.load_n(zp + t * p.a.z_time, n, p.vec_z);
        st_load(h0, p.a.saved + (static_cast<long long>(at.b) * p.nchunk + tc / K::TS) * dim * S, f0, swap, fend, S, n0, p.vec_n);
    };
    auto stage_bc = [&](int buf, int tc) {
        const int t = tc + brow;
#pragma unroll
        for (int e = 0; e < BN; ++e) {
            const int n = bcol + e;
            if (n < K::NP) {
                const bool in = t < len && n < S;
                const float b = in ? to_f(Bp[t * p.a.B_time + n]) : 0.f, c = in ? to_f(Cp[t * p.a.C_time + n]) : 0.f;
#pragma unroll
                for (int q = 0; q < M::NQ; ++q) {
                    sm.B[buf][q][brow][n ^ q] = b;
                    sm.C[buf][q][brow][n ^ q] = c;
                }
            }
        }
    };
    // The block's dB, dC of a piece.
    auto put_bc = [&](int buf, int tc) {
        float* d = p.part_bc + ((static_cast<long long>(gq) * p.a.batch + at.b) * L + tc) * 2 * K::NP;
        const int rows = min(K::TS, min(at.t1, len) - tc);
        for (int i = threadIdx.x; i < rows * 2 * K::NP; i += kScanThreads) {
            float s = 0.f;
#pragma unroll
            for (int q = 0; q < kScanWarps; ++q) s += (&sm.acc[buf][q][0][0][0])[i];
            d[i] = s;
        }
    };

    const int tend = min(at.t1, len), pieces = tend > at.t0 ? (tend - at.t0 + K::TS - 1) / K::TS : 0;
    if (pieces > 0) {
        fetch(at.t0 + (pieces - 1) * K::TS);
        stage_bc(0, at.t0 + (pieces - 1) * K::TS);
    }
    for (int k = 0; k < pieces; ++k) {
        const int tc = at.t0 + (pieces - 1 - k) * K::TS, buf = k & 1, t = tc + row;
        const bool in = t < len;
        St hs = h0;
        __syncwarp();
#pragma unroll
        for (int e = 0; e < K::VX; e += 2) {
            float dt[2], u[2], g[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float x = rx.get(e + i);
                float ds = 1.f, zf = 0.f;
                dt[i] = rd.get(e + i) + (bias && e + i < nx ? __ldg(bias + e + i) : 0.f);
                if (p.a.softplus) dt[i] = softplusf(dt[i], &ds);
                if (!in) dt[i] = ds = 0.f;
                g[i] = rg.get(e + i);
                if (p.a.z) {
                    const float z = rz.get(e + i), sg = sigmoidf(z);
                    zf = g[i] * sg * fmaf(z, 1.f - sg, 1.f);
                    g[i] *= z * sg;
                }
                u[i] = dt[i] * x;
                sm.X[w][row][col + e + i] = x;
                sm.D[w][row][col + e + i] = ds;
                sm.Z[w][row][col + e + i] = zf;
            }
            sm.U[w][0][row][(col + e) / 2] = make_float4(dt[0], u[0], dt[1], u[1]);
            sm.U[w][1][row][(col + e) / 2] = make_float4(dt[1], u[1], dt[0], u[0]);
            sm.G[w][0][row][(col + e) / 2] = make_float2(g[0], g[1]);
            sm.G[w][1][row][(col + e) / 2] = make_float2(g[1], g[0]);
        }
        // Behind this barrier: B and C of this piece, and the warps' dB and dC
        // of the one before.  The buffers alternate, so one barrier is enough.
        __syncthreads();
        if (k > 0) put_bc(buf ^ 1, tc + K::TS);
        permute(hs);

        f2 a[kRun][kCT][2], h[kRun][kCT][2];
        // 8 steps forward from hs; `keep` stores the decays and the states.
        auto forward = [&](int sb, St& s0, bool keep) {
#pragma unroll
            for (int s = 0; s < kRun; ++s) {
                const float4 du = sm.U[w][swap][sb + s][cl];
                const ulonglong2 bv = *reinterpret_cast<const ulonglong2*>(&sm.B[buf][perm][sb + s][n0]);
#pragma unroll
                for (int i = 0; i < kCT; ++i) {
                    const float dt = i ? du.z : du.x, u = i ? du.w : du.y;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const f2 d = ex22(mul2(pk(dt, dt), A2.v[i][j]));
                        s0.v[i][j] = fma2(d, s0.v[i][j], mul2(pk(u, u), f2{j ? bv.y : bv.x}));
                        if (keep) {
                            a[s][i][j] = d;
                            h[s][i][j] = s0.v[i][j];
                        }
                    }
                }
            }
        };
        St hm = hs;
        if constexpr (K::TS > kRun) forward(0, hm, false);
#pragma unroll 1
        for (int sb = K::TS - kRun; sb >= 0; sb -= kRun) {
            St hin;
#pragma unroll
            for (int i = 0; i < kCT; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) hin.v[i][j].v = sb > 0 ? hm.v[i][j].v : hs.v[i][j].v;
            St run = hin;
            forward(sb, run, true);
            float vq[2 * kCT], vr[2 * kCT], vy[2 * kCT];
#pragma unroll
            for (int s = kRun - 1; s >= 0; --s) {
                const float4 du = sm.U[w][swap][sb + s][cl];
                const float2 gy = sm.G[w][swap][sb + s][cl];
                const ulonglong2 bv = *reinterpret_cast<const ulonglong2*>(&sm.B[buf][perm][sb + s][n0]);
                const ulonglong2 cv = *reinterpret_cast<const ulonglong2*>(&sm.C[buf][perm][sb + s][n0]);
                f2 aB[2], aC[2];
#pragma unroll
                for (int i = 0; i < kCT; ++i) {
                    const float dt = i ? du.z : du.x, u = i ? du.w : du.y, g = i ? gy.y : gy.x;
                    f2 q, sa, y;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const f2 b2{j ? bv.y : bv.x}, c2{j ? cv.y : cv.x};
                        const f2 gh = fma2(pk(g, g), c2, r.v[i][j]);
                        r.v[i][j] = mul2(a[s][i][j], gh);
                        const f2 hp = s > 0 ? h[s > 0 ? s - 1 : 0][i][j] : hin.v[i][j];
                        const f2 kk = mul2(r.v[i][j], hp);
                        dA.v[i][j] = fma2(pk(dt, dt), kk, dA.v[i][j]);
                        aC[j] = i ? fma2(pk(g, g), h[s][i][j], aC[j]) : mul2(pk(g, g), h[s][i][j]);
                        aB[j] = i ? fma2(pk(u, u), gh, aB[j]) : mul2(pk(u, u), gh);
                        q = j ? fma2(gh, b2, q) : mul2(gh, b2);
                        sa = j ? fma2(kk, A2.v[i][j], sa) : mul2(kk, A2.v[i][j]);
                        y = j ? fma2(c2, h[s][i][j], y) : mul2(c2, h[s][i][j]);
                    }
                    // Pairs of registers (step of an even pair, feature): see pair_exchange.
                    vq[(s & 1) * kCT + i] = sum2(q);
                    vr[(s & 1) * kCT + i] = sum2(sa);
                    vy[(s & 1) * kCT + i] = sum2(y);
                }
                // dB, dC over the lanes' features: register j is state n0 + (j ^ perm).
                float vb[4], vc[4];
                upk(aB[0], vb[0], vb[1]);
                upk(aB[1], vb[2], vb[3]);
                upk(aC[0], vc[0], vc[1]);
                upk(aC[1], vc[2], vc[3]);
                float* acc = &sm.acc[buf][w][sb + s][0][n0];
                if constexpr (M::NQ == 4) {
                    float b1[2], c1[2], b0[1], c0[1];
                    pair_exchange(vb, b1, NL);  // state bit 0
                    pair_exchange(vc, c1, NL);
                    pair_exchange(b1, b0, 2 * NL);  // state bit 1
                    pair_exchange(c1, c0, 2 * NL);
                    // dB to the lanes without bit 4 NL, dC to those with it (none for 8 lanes per feature: both).
                    if constexpr (K::CL >= 8) {
                        const bool up = lane & (4 * NL);
                        float v = (up ? c0[0] : b0[0]) + __shfl_xor_sync(0xffffffffu, up ? b0[0] : c0[0], 4 * NL);
#pragma unroll
                        for (int m = 8 * NL; m < 32; m *= 2) v += __shfl_xor_sync(0xffffffffu, v, m);
                        if (lane < 8 * NL) acc[(up ? K::NP : 0) + perm] = v;
                    } else {
                        acc[perm] = b0[0];
                        acc[K::NP + perm] = c0[0];
                    }
                } else {  // two lane groups: state bit 0 only
                    float b1[2], c1[2];
                    pair_exchange(vb, b1, NL);
                    pair_exchange(vc, c1, NL);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        acc[2 * j + perm] = b1[j];
                        acc[K::NP + 2 * j + perm] = c1[j];
                    }
                }
                if ((s & 1) == 0) {  // q, s, y over the lanes' states, two steps at a time
                    auto put = [&](float(&v)[2 * kCT], float (*out)[K::CH]) {
                        if constexpr (NL == 1) {
#pragma unroll
                            for (int i = 0; i < 2 * kCT; ++i) out[sb + s + i / kCT][cl * kCT + i % kCT] = v[i];
                        } else {
                            float o[2];
                            pair_exchange(v, o, 1);
                            using Sum = LaneSum<2, 2, NL / 2>;
                            Sum::run(o, lane);
                            if (Sum::owner(lane)) {
                                const int slot = Sum::slot(lane);
#pragma unroll
                                for (int i = 0; i < Sum::kept; ++i) out[sb + s + slot + i][cl * kCT + swap] = o[i];
                            }
                        }
                    };
                    put(vq, sm.Q[w]);
                    put(vr, sm.R[w]);
                    put(vy, sm.Y[w]);
                }
            }
        }
        if (k + 1 < pieces) {  // on their way during what follows
            fetch(tc - K::TS);
            stage_bc(buf ^ 1, tc - K::TS);
        }
        __syncwarp();
        Vec<T, K::VX> ox, od, oz;
#pragma unroll
        for (int e = 0; e < K::VX; ++e) {
            const float2 du = reinterpret_cast<const float2*>(sm.U[w][0][row])[col + e];
            const float gy = reinterpret_cast<const float*>(sm.G[w][0][row])[col + e];
            const float q = sm.Q[w][row][col + e], x = sm.X[w][row][col + e];
            const float Df = skip && e < nx ? __ldg(skip + e) : 0.f;
            const float dd = fmaf(q, x, kLn2 * sm.R[w][row][col + e]) * sm.D[w][row][col + e];
            dbias[e] += dd;
            dD[e] = fmaf(gy, x, dD[e]);
            ox.set(e, fmaf(q, du.x, gy * Df));
            od.set(e, dd);
            oz.set(e, sm.Z[w][row][col + e] * fmaf(Df, x, sm.Y[w][row][col + e]));
        }
        const int no = t < at.t1 ? nx : 0;
        const long long o = out0 + static_cast<long long>(t) * dim;
        if (p.a.dx) ox.store_n(static_cast<T*>(p.a.dx) + o, no, p.vec_dx);
        if (p.a.ddelta) od.store_n(static_cast<T*>(p.a.ddelta) + o, no, p.vec_ddelta);
        if (p.a.z && p.a.dz) oz.store_n(static_cast<T*>(p.a.dz) + o, no, p.vec_dz);
    }
    for (int t = at.t0 + pieces * K::TS + row; t < at.t1; t += K::TS) {
        Vec<T, K::VX> o;
        o.zero();
        const long long at_t = out0 + static_cast<long long>(t) * dim;
        if (p.a.dx) o.store_n(static_cast<T*>(p.a.dx) + at_t, nx, p.vec_dx);
        if (p.a.ddelta) o.store_n(static_cast<T*>(p.a.ddelta) + at_t, nx, p.vec_ddelta);
        if (p.a.z && p.a.dz) o.store_n(static_cast<T*>(p.a.dz) + at_t, nx, p.vec_dz);
    }
    __syncthreads();
    if (pieces > 0) put_bc((pieces - 1) & 1, at.t0);
    permute(dA);
    permute(r);
    if (at.seg == 0 && p.a.dstate_in)
        st_store(r, p.a.dstate_in + static_cast<long long>(at.b) * dim * S, f0, swap, fend, S, n0, p.vec_n);
    // The segment's dA, dD and ddelta_bias.
    float* par = p.part_par + (static_cast<long long>(at.b) * p.nseg + at.seg) * dim * (S + 2);
    st_store(dA, par, f0, swap, fend, S, n0, p.vec_n && dim % 2 == 0);
#pragma unroll
    for (int e = 0; e < K::VX; ++e) {
#pragma unroll
        for (int m = K::LR; m < 32; m *= 2) {
            dD[e] += __shfl_xor_sync(0xffffffffu, dD[e], m);
            dbias[e] += __shfl_xor_sync(0xffffffffu, dbias[e], m);
        }
        if (row == 0 && e < nx) {
            par[static_cast<long long>(dim) * S + at.c0 + col + e] = dD[e];
            par[static_cast<long long>(dim) * (S + 1) + at.c0 + col + e] = dbias[e];
        }
    }
}

// Adds the partial sums in a fixed order: blocks below nbc one element of dB or
// dC per thread (over the group's blocks of features), the others one of dA, dD
// and ddelta_bias (over the batch and its segments).
template <typename T>
__global__ void __launch_bounds__(256) scan_sum_kernel(const ScanP p, long long nbc, int NP, int quads) {
    pdl_wait();
    const int S = p.a.nstate, G = p.a.groups, dim = p.a.dim, L = p.a.length;
    if (blockIdx.x < nbc) {
        const long long i = blockIdx.x * 256ll + threadIdx.x;  // (b, t, g, which, n)
        const int n = static_cast<int>(i % NP), which = static_cast<int>(i / NP % 2);
        const long long rowg = i / (2 * NP);
        const int g = static_cast<int>(rowg % G);
        const long long bt = rowg / G;
        if (bt >= static_cast<long long>(p.a.batch) * L || n >= S) return;
        const int b = static_cast<int>(bt / L), t = static_cast<int>(bt % L);
        void* out = which ? p.a.dC : p.a.dB;
        if (!out) return;
        float s = 0.f;
        if (t < seq_len(p.a.lengths, b, L)) {
            const long long part = static_cast<long long>(p.a.batch) * L * 2 * NP;
            const float* q = p.part_bc + g * quads * part + bt * 2 * NP + which * NP + n;
#pragma unroll 8
            for (int k = 0; k < quads; ++k) s += q[k * part];
        }
        static_cast<T*>(out)[rowg * S + n] = from_f<T>(s);
        return;
    }
    const long long i = (blockIdx.x - nbc) * 256 + threadIdx.x, cols = static_cast<long long>(dim) * (S + 2);
    if (i >= cols) return;
    float s = 0.f;
    const int rows = p.a.batch * p.nseg;
#pragma unroll 8
    for (int b = 0; b < rows; ++b) s += p.part_par[b * cols + i];
    const long long dA = static_cast<long long>(dim) * S;
    if (i < dA) {
        if (p.a.dA) p.a.dA[i] = s;
    } else if (i < dA + dim) {
        if (p.a.dD) p.a.dD[i - dA] = s;
    } else if (p.a.ddelta_bias) {
        p.a.ddelta_bias[i - dA - dim] = s;
    }
}

int scan_quads(int dim, int groups, int nstate) {
    const int ch = 32 / scan_lanes(nstate) * kCT * kScanWarps;
    return (dim / groups + ch - 1) / ch;
}
size_t bc_floats(int batch, int length, int dim, int groups, int nstate) {
    return static_cast<size_t>(groups) * scan_quads(dim, groups, nstate) * batch * length * 2 * 4 * scan_lanes(nstate);
}
size_t up4(size_t n) { return (n + 3) / 4 * 4; }  // whole 16-byte pieces

template <typename T, int NL>
cudaError_t run_scan_bwd(const sdtw_scan_args& a, cudaStream_t st) {
    ScanP p{};
    scan_params<T, NL>(p, a);
    const ScanSplit split = scan_split(a.batch, a.length, a.dim, a.groups, a.nstate, true);
    p.part_bc = static_cast<float*>(a.workspace);
    float* seg = p.part_bc + bc_floats(a.batch, a.length, a.dim, a.groups, a.nstate);
    scan_segment_tables(p, split, seg);
    p.part_par = seg + up4(scan_segment_floats(a.batch, split.nseg, a.dim, a.nstate));
    const int quads = scan_quads(a.dim, a.groups, a.nstate);
    const long long blocks = static_cast<long long>(quads) * a.groups * a.batch * p.nseg;
    const long long nbc = (static_cast<long long>(a.batch) * a.length * a.groups * 2 * 4 * NL + 255) / 256;
    const long long npar = (static_cast<long long>(a.dim) * (a.nstate + 2) + 255) / 256;
    if (blocks > 0x7fffffffll || nbc + npar > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    const int smem = static_cast<int>(sizeof(BwdSmem<NL>));
    cudaError_t e = cudaFuncSetAttribute(scan_bwd_kernel<T, NL>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (p.nseg > 1 && (e = launch_scan_segments(p, true, st)) != cudaSuccess) return e;
    e = launch_pdl(p.nseg > 1, scan_bwd_kernel<T, NL>, dim3(static_cast<unsigned>(blocks)), dim3(kScanThreads), smem, st, p);
    if (e != cudaSuccess) return e;
    return launch_pdl(true, scan_sum_kernel<T>, dim3(static_cast<unsigned>(nbc + npar)), dim3(256), 0, st, p, nbc, 4 * NL, quads);
}

template <typename T>
cudaError_t run_scan_bwd_t(const sdtw_scan_args& a, cudaStream_t st) {
    switch (scan_lanes(a.nstate)) {
        case 1: return run_scan_bwd<T, 1>(a, st);
        case 2: return run_scan_bwd<T, 2>(a, st);
        case 4: return run_scan_bwd<T, 4>(a, st);
        case 8: return run_scan_bwd<T, 8>(a, st);
        default: return run_scan_bwd<T, 16>(a, st);
    }
}

}  // namespace

size_t scan_bwd_ws(int batch, int length, int dim, int groups, int nstate) {
    const int nseg = scan_split(batch, length, dim, groups, nstate, true).nseg;
    return (bc_floats(batch, length, dim, groups, nstate) + up4(scan_segment_floats(batch, nseg, dim, nstate)) +
            static_cast<size_t>(batch) * nseg * dim * (nstate + 2)) *
           sizeof(float);
}

cudaError_t launch_scan_bwd(const sdtw_scan_args& a, cudaStream_t st) {
    if (a.dtype == SDTW_F32) return run_scan_bwd_t<float>(a, st);
    if (a.dtype == SDTW_F16) return run_scan_bwd_t<__half>(a, st);
    return run_scan_bwd_t<__nv_bfloat16>(a, st);
}

}  // namespace sdtw

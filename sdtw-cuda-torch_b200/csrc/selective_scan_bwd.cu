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
// A block walks over its chunks from the last to the first, from the states that
// the forward stored at the chunks' starts.  As in the forward each warp keeps
// the decays of its 8 steps in registers and runs the recurrence twice: from 0,
// which gives the run's product P and end E, and with the states chained over
// the warps; the reverse recurrence r has the same product P, so that both are
// chained behind one barrier.  Every exponential is computed once.  The states
// of the 8 steps stay in registers too (64 registers each for decays and states
// per thread).  Sums over the states of a feature and over the features of dB
// and dC are lane exchanges that halve the values at every step; what is left of
// dB and dC per block goes to a partial table that a second kernel adds up in a
// fixed order, so results do not change from call to call.
#include "selective_scan.cuh"

namespace sdtw {
namespace {

template <int NL>
struct BwdSmem {
    using K = ScanTile<NL>;
    float2 U[kScanWarps][kScanSteps][K::CH];  // (dt, u)
    float G[kScanWarps][kScanSteps][K::CH];   // gy
    float Q[kScanWarps][kScanSteps][K::CH], R[kScanWarps][kScanSteps][K::CH], Y[kScanWarps][kScanSteps][K::CH];
    float B[kScanWarps][kScanSteps][K::NP], C[kScanWarps][kScanSteps][K::NP];
    ulonglong2 P[2][kScanWarps][kCT][32], E[2][kScanWarps][kCT][32], R0[2][kScanWarps][kCT][32], carry[2][kCT][32];
};

template <typename T, int NL>
__global__ void __launch_bounds__(kScanThreads, 2) scan_bwd_kernel(const ScanP p) {
    using K = ScanTile<NL>;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    BwdSmem<NL>& sm = *reinterpret_cast<BwdSmem<NL>*>(smem_raw);
    const ScanPlace<NL> at(p);
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nl = lane % NL, cl = lane / NL;
    const int S = p.a.nstate, L = p.a.length, dim = p.a.dim;
    const int len = seq_len(p.a.lengths, at.b, L);
    const int f0 = at.c0 + cl * kCT, fend = at.c0 + at.nc;
    const int row = lane >> 2, col = (lane & 3) * K::VX, bcol = (lane & 3) * K::VN;
    const int nx = min(max(at.nc - col, 0), K::VX), nb = min(max(S - bcol, 0), K::VN);

    St A2, dA;
    st_load(A2, p.a.A, f0, fend, S, nl * 4, p.vec_n);
#pragma unroll
    for (int i = 0; i < kCT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) A2.v[i][j] = mul2(A2.v[i][j], pk(kL2e, kL2e));
    st_set(dA, 0.f);
    float dD[K::VX], dbias[K::VX];
#pragma unroll
    for (int e = 0; e < K::VX; ++e) dD[e] = dbias[e] = 0.f;
    if (w == 0) {
        St r;
        st_set(r, 0.f);
        if (p.a.dstate_out) st_load(r, p.a.dstate_out + static_cast<long long>(at.b) * dim * S, f0, fend, S, nl * 4, p.vec_n);
        st_put(sm.carry[0], lane, r);
    }
    const T* xp = static_cast<const T*>(p.a.x) + at.b * p.a.x_batch + at.c0 + col;
    const T* dp = static_cast<const T*>(p.a.delta) + at.b * p.a.delta_batch + at.c0 + col;
    const T* zp = static_cast<const T*>(p.a.z) + at.b * p.a.z_batch + at.c0 + col;
    const T* gp = static_cast<const T*>(p.a.dy) + at.b * p.a.dy_batch + at.c0 + col;
    const T* Bp = static_cast<const T*>(p.a.B) + at.b * p.a.B_batch + at.g * p.a.B_group + bcol;
    const T* Cp = static_cast<const T*>(p.a.C) + at.b * p.a.C_batch + at.g * p.a.C_group + bcol;
    const long long out0 = static_cast<long long>(at.b) * L * dim + at.c0 + col;

    const int nck = (len + kScanChunk - 1) / kScanChunk;
    for (int ck = nck - 1; ck >= 0; --ck) {
        const int buf = (nck - 1 - ck) & 1;
        const int t = ck * kScanChunk + w * kScanSteps + row;  // the step that this lane stages
        const bool in = t < len;
        Vec<T, K::VX> rx, rd, rz, rg;
        Vec<T, K::VN> rB, rC;
        rx.load_n(xp + t * p.a.x_time, in ? nx : 0, p.vec_x);
        rd.load_n(dp + t * p.a.delta_time, in ? nx : 0, p.vec_delta);
        rg.load_n(gp + t * p.a.dy_time, in ? nx : 0, p.vec_dy);
        if (p.a.z) rz.load_n(zp + t * p.a.z_time, in ? nx : 0, p.vec_z);
        rB.load_n(Bp + t * p.a.B_time, in ? nb : 0, p.vec_B);
        rC.load_n(Cp + t * p.a.C_time, in ? nb : 0, p.vec_C);
        St hin;
        st_load(hin, p.a.saved + (static_cast<long long>(at.b) * p.nchunk + ck) * dim * S, f0, fend, S, nl * 4, p.vec_n);
        __syncwarp();
#pragma unroll
        for (int e = 0; e < K::VX; ++e) {
            float dt = rd.get(e) + (p.a.delta_bias && e < nx ? __ldg(p.a.delta_bias + at.c0 + col + e) : 0.f);
            if (p.a.softplus) dt = softplusf(dt);
            if (!in) dt = 0.f;
            float gy = rg.get(e);
            if (p.a.z) {
                const float z = rz.get(e);
                gy *= z * sigmoidf(z);
            }
            sm.U[w][row][col + e] = make_float2(dt, dt * rx.get(e));
            sm.G[w][row][col + e] = gy;
        }
#pragma unroll
        for (int e = 0; e < K::VN; ++e) {
            sm.B[w][row][bcol + e] = rB.get(e);
            sm.C[w][row][bcol + e] = rC.get(e);
        }
        __syncwarp();

        f2 a[kScanSteps][kCT][2], h[kScanSteps][kCT][2];
        St P, E;
        st_set(E, 0.f);
        st_set(P, 1.f);
#pragma unroll
        for (int s = 0; s < kScanSteps; ++s) {
            const float4 du = *reinterpret_cast<const float4*>(&sm.U[w][s][cl * kCT]);
            const ulonglong2 bv = *reinterpret_cast<const ulonglong2*>(&sm.B[w][s][nl * 4]);
#pragma unroll
            for (int i = 0; i < kCT; ++i) {
                const float dt = i ? du.z : du.x, u = i ? du.w : du.y;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    a[s][i][j] = ex22(mul2(pk(dt, dt), A2.v[i][j]));
                    E.v[i][j] = fma2(a[s][i][j], E.v[i][j], mul2(pk(u, u), f2{j ? bv.y : bv.x}));
                    h[s][i][j] = E.v[i][j];
                    P.v[i][j] = mul2(P.v[i][j], a[s][i][j]);
                }
            }
        }
        st_put(sm.P[buf][w], lane, P);
        st_put(sm.E[buf][w], lane, E);
        St r;
        st_set(r, 0.f);
#pragma unroll
        for (int s = kScanSteps - 1; s >= 0; --s) {
            const float2 gy = *reinterpret_cast<const float2*>(&sm.G[w][s][cl * kCT]);
            const ulonglong2 cv = *reinterpret_cast<const ulonglong2*>(&sm.C[w][s][nl * 4]);
#pragma unroll
            for (int i = 0; i < kCT; ++i) {
                const float g = i ? gy.y : gy.x;
#pragma unroll
                for (int j = 0; j < 2; ++j) r.v[i][j] = mul2(a[s][i][j], fma2(pk(g, g), f2{j ? cv.y : cv.x}, r.v[i][j]));
            }
        }
        st_put(sm.R0[buf][w], lane, r);
        __syncthreads();  // one per chunk: the buffers alternate
        for (int q = 0; q < w; ++q) st_chain(hin, sm.P[buf][q], sm.E[buf][q], lane);
        st_get(r, sm.carry[buf], lane);
        for (int q = kScanWarps - 1; q > w; --q) st_chain(r, sm.P[buf][q], sm.R0[buf][q], lane);
        if (w == 0) {
            St c = r;
            st_chain(c, sm.P[buf][0], sm.R0[buf][0], lane);
            st_put(sm.carry[buf ^ 1], lane, c);
        }
        // The states from the true start: h = (h from 0) + (product of decays) hin.
        St pc = hin;
#pragma unroll
        for (int s = 0; s < kScanSteps; ++s)
#pragma unroll
            for (int i = 0; i < kCT; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    pc.v[i][j] = mul2(pc.v[i][j], a[s][i][j]);
                    h[s][i][j] = add2(h[s][i][j], pc.v[i][j]);
                }
        using SumF = LaneSum<2 * kCT, 1, NL>;      // over the states of a feature, 2 steps at a time
        using SumN = LaneSum<8, NL, 32 / NL>;      // over the features: 4 states of dB, 4 of dC
        float vq[2 * kCT], vr[2 * kCT], vy[2 * kCT];
#pragma unroll
        for (int s = kScanSteps - 1; s >= 0; --s) {
            const float4 du = *reinterpret_cast<const float4*>(&sm.U[w][s][cl * kCT]);
            const float2 gy = *reinterpret_cast<const float2*>(&sm.G[w][s][cl * kCT]);
            const ulonglong2 bv = *reinterpret_cast<const ulonglong2*>(&sm.B[w][s][nl * 4]);
            const ulonglong2 cv = *reinterpret_cast<const ulonglong2*>(&sm.C[w][s][nl * 4]);
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
                    const f2 k = mul2(r.v[i][j], hp);
                    dA.v[i][j] = fma2(pk(dt, dt), k, dA.v[i][j]);
                    aC[j] = i ? fma2(pk(g, g), h[s][i][j], aC[j]) : mul2(pk(g, g), h[s][i][j]);
                    aB[j] = i ? fma2(pk(u, u), gh, aB[j]) : mul2(pk(u, u), gh);
                    q = j ? fma2(gh, b2, q) : mul2(gh, b2);
                    sa = j ? fma2(k, A2.v[i][j], sa) : mul2(k, A2.v[i][j]);
                    y = j ? fma2(c2, h[s][i][j], y) : mul2(c2, h[s][i][j]);
                }
                vq[(s & 1) * kCT + i] = sum2(q);
                vr[(s & 1) * kCT + i] = sum2(sa);
                vy[(s & 1) * kCT + i] = sum2(y);
            }
            float v[8];
            upk(aB[0], v[0], v[1]);
            upk(aB[1], v[2], v[3]);
            upk(aC[0], v[4], v[5]);
            upk(aC[1], v[6], v[7]);
            SumN::run(v, lane);
            const int ts = ck * kScanChunk + w * kScanSteps + s;
            if (ts < len && SumN::owner(lane)) {
                const int k0 = SumN::slot(lane);  // 0-3: dB, 4-7: dC
                float* d = p.part_bc +
                           ((static_cast<long long>(at.tile) * p.a.batch + at.b) * L + ts) * 2 * K::NP + (k0 / 4) * K::NP + nl * 4 + k0 % 4;
#pragma unroll
                for (int k = 0; k < SumN::kept; ++k) d[k % 4 + k / 4 * K::NP] = v[k];
            }
            if ((s & 1) == 0) {
                SumF::run(vq, lane);
                SumF::run(vr, lane);
                SumF::run(vy, lane);
                if (SumF::owner(lane)) {
                    const int slot = SumF::slot(lane);
#pragma unroll
                    for (int k = 0; k < SumF::kept; ++k) {
                        const int ss = s + (slot + k) / kCT, c = cl * kCT + (slot + k) % kCT;
                        sm.Q[w][ss][c] = vq[k];
                        sm.R[w][ss][c] = vr[k];
                        sm.Y[w][ss][c] = vy[k];
                    }
                }
            }
        }
        __syncwarp();
        Vec<T, K::VX> ox, od, oz;
#pragma unroll
        for (int e = 0; e < K::VX; ++e) {
            const float dt = sm.U[w][row][col + e].x, gy = sm.G[w][row][col + e], q = sm.Q[w][row][col + e];
            const float x = rx.get(e);
            const float Df = p.a.D && e < nx ? __ldg(p.a.D + at.c0 + col + e) : 0.f;
            float dd = fmaf(q, x, kLn2 * sm.R[w][row][col + e]);
            if (p.a.softplus) dd *= sigmoidf(rd.get(e) + (p.a.delta_bias && e < nx ? __ldg(p.a.delta_bias + at.c0 + col + e) : 0.f));
            if (!in) dd = 0.f;
            dbias[e] += dd;
            dD[e] = fmaf(gy, x, dD[e]);
            ox.set(e, fmaf(q, dt, gy * Df));
            od.set(e, dd);
            if (p.a.z) {
                const float z = rz.get(e), sg = sigmoidf(z);
                const float y = fmaf(Df, x, sm.Y[w][row][col + e]);
                oz.set(e, rg.get(e) * y * (sg * (1.f + z * (1.f - sg))));
            }
        }
        const int no = t < L ? nx : 0;
        const long long o = out0 + static_cast<long long>(t) * dim;
        if (p.a.dx) ox.store_n(static_cast<T*>(p.a.dx) + o, no, p.vec_dx);
        if (p.a.ddelta) od.store_n(static_cast<T*>(p.a.ddelta) + o, no, p.vec_ddelta);
        if (p.a.z && p.a.dz) oz.store_n(static_cast<T*>(p.a.dz) + o, no, p.vec_dz);
    }
    for (int t = nck * kScanChunk + w * kScanSteps + row; t < L; t += kScanChunk) {
        Vec<T, K::VX> o;
        o.zero();
        const long long at_t = out0 + static_cast<long long>(t) * dim;
        if (p.a.dx) o.store_n(static_cast<T*>(p.a.dx) + at_t, nx, p.vec_dx);
        if (p.a.ddelta) o.store_n(static_cast<T*>(p.a.ddelta) + at_t, nx, p.vec_ddelta);
        if (p.a.z && p.a.dz) o.store_n(static_cast<T*>(p.a.dz) + at_t, nx, p.vec_dz);
    }
    __syncthreads();
    if (w == 0 && p.a.dstate_in) {
        St r;
        st_get(r, sm.carry[nck & 1], lane);
        st_store(r, p.a.dstate_in + static_cast<long long>(at.b) * dim * S, f0, fend, S, nl * 4, p.vec_n);
    }
    // This batch entry's dA, dD and ddelta_bias: the warps' sums in a fixed order.
    float* par = p.part_par + static_cast<long long>(at.b) * dim * (S + 2);
    st_put(sm.P[0][w], lane, dA);
#pragma unroll
    for (int e = 0; e < K::VX; ++e) {
#pragma unroll
        for (int m = 4; m < 32; m *= 2) {
            dD[e] += __shfl_xor_sync(0xffffffffu, dD[e], m);
            dbias[e] += __shfl_xor_sync(0xffffffffu, dbias[e], m);
        }
        if (row == 0) {
            sm.Q[w][0][col + e] = dD[e];
            sm.R[w][0][col + e] = dbias[e];
        }
    }
    __syncthreads();
    if (w == 0) {
#pragma unroll
        for (int q = 1; q < kScanWarps; ++q) {
            St o;
            st_get(o, sm.P[0][q], lane);
#pragma unroll
            for (int i = 0; i < kCT; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) dA.v[i][j] = add2(dA.v[i][j], o.v[i][j]);
        }
        st_store(dA, par, f0, fend, S, nl * 4, p.vec_n && dim % 2 == 0);
    } else if (w == 1) {
        for (int c = lane; c < at.nc; c += 32) {
            float d = 0.f, s = 0.f;
#pragma unroll
            for (int q = 0; q < kScanWarps; ++q) {
                d += sm.Q[q][0][c];
                s += sm.R[q][0][c];
            }
            par[static_cast<long long>(dim) * S + at.c0 + c] = d;
            par[static_cast<long long>(dim) * (S + 1) + at.c0 + c] = s;
        }
    }
}

// Adds the partial sums in a fixed order: blocks below nbc one element of dB or
// dC per thread (over the group's tiles), the others one of dA, dD and
// ddelta_bias (over the batch).
template <typename T>
__global__ void __launch_bounds__(256) scan_sum_kernel(const ScanP p, long long nbc, int NP) {
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
            const long long tile = static_cast<long long>(p.a.batch) * L * 2 * NP;
            const float* q = p.part_bc + g * p.tiles_g * tile + bt * 2 * NP + which * NP + n;
#pragma unroll 8
            for (int k = 0; k < p.tiles_g; ++k) s += q[k * tile];
        }
        static_cast<T*>(out)[rowg * S + n] = from_f<T>(s);
        return;
    }
    const long long i = (blockIdx.x - nbc) * 256 + threadIdx.x, cols = static_cast<long long>(dim) * (S + 2);
    if (i >= cols) return;
    float s = 0.f;
#pragma unroll 8
    for (int b = 0; b < p.a.batch; ++b) s += p.part_par[b * cols + i];
    const long long dA = static_cast<long long>(dim) * S;
    if (i < dA) {
        if (p.a.dA) p.a.dA[i] = s;
    } else if (i < dA + dim) {
        if (p.a.dD) p.a.dD[i - dA] = s;
    } else if (p.a.ddelta_bias) {
        p.a.ddelta_bias[i - dA - dim] = s;
    }
}

size_t bc_floats(int batch, int length, int dim, int groups, int nstate) {
    const int nl = scan_lanes(nstate), ch = 32 / nl * kCT, dg = dim / groups;
    return static_cast<size_t>(groups) * ((dg + ch - 1) / ch) * batch * length * 2 * 4 * nl;
}

template <typename T, int NL>
cudaError_t run_scan_bwd(const sdtw_scan_args& a, cudaStream_t st) {
    ScanP p{};
    scan_params<T, NL>(p, a);
    p.part_bc = static_cast<float*>(a.workspace);
    p.part_par = p.part_bc + bc_floats(a.batch, a.length, a.dim, a.groups, a.nstate);
    const long long blocks = scan_blocks<NL>(p);
    const long long nbc = (static_cast<long long>(a.batch) * a.length * a.groups * 2 * 4 * NL + 255) / 256;
    const long long npar = (static_cast<long long>(a.dim) * (a.nstate + 2) + 255) / 256;
    if (blocks > 0x7fffffffll || nbc + npar > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    const int smem = static_cast<int>(sizeof(BwdSmem<NL>));
    cudaError_t e = cudaFuncSetAttribute(scan_bwd_kernel<T, NL>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    scan_bwd_kernel<T, NL><<<static_cast<unsigned>(blocks), kScanThreads, smem, st>>>(p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_pdl(true, scan_sum_kernel<T>, dim3(static_cast<unsigned>(nbc + npar)), dim3(256), 0, st, p, nbc, 4 * NL);
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
    return (bc_floats(batch, length, dim, groups, nstate) + static_cast<size_t>(batch) * dim * (nstate + 2)) * sizeof(float);
}

cudaError_t launch_scan_bwd(const sdtw_scan_args& a, cudaStream_t st) {
    if (a.dtype == SDTW_F32) return run_scan_bwd_t<float>(a, st);
    if (a.dtype == SDTW_F16) return run_scan_bwd_t<__half>(a, st);
    return run_scan_bwd_t<__nv_bfloat16>(a, st);
}

}  // namespace sdtw

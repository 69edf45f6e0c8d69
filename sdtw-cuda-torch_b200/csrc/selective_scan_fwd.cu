// selective_scan_fwd.cu -- forward of the selective scan (see
// selective_scan.cuh for the formulas and the tiling) and its single-step form.
#include "selective_scan.cuh"

namespace sdtw {
namespace {

template <typename T, int NL>
__global__ void __launch_bounds__(kScanThreads, 3) scan_fwd_kernel(const ScanP p) {
    using K = ScanTile<NL>;
    __shared__ __align__(16) float2 sU[kScanWarps][kScanSteps][K::CH];  // (dt, u); later y
    __shared__ __align__(16) float sB[kScanWarps][kScanSteps][K::NP], sC[kScanWarps][kScanSteps][K::NP];
    __shared__ ulonglong2 sP[2][kScanWarps][kCT][32], sE[2][kScanWarps][kCT][32], sCarry[2][kCT][32];
    const ScanPlace<NL> at(p);
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nl = lane % NL, cl = lane / NL;
    const int S = p.a.nstate, L = p.a.length, dim = p.a.dim;
    const int len = seq_len(p.a.lengths, at.b, L);
    const int f0 = at.c0 + cl * kCT, fend = at.c0 + at.nc;  // this thread's first feature, the block's last + 1
    // Staging: 4 lanes per time step.
    const int row = lane >> 2, col = (lane & 3) * K::VX, bcol = (lane & 3) * K::VN;
    const int nx = min(max(at.nc - col, 0), K::VX), nb = min(max(S - bcol, 0), K::VN);

    St A2;
    st_load(A2, p.a.A, f0, fend, S, nl * 4, p.vec_n);
#pragma unroll
    for (int i = 0; i < kCT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) A2.v[i][j] = mul2(A2.v[i][j], pk(kL2e, kL2e));
    float bias[K::VX], skip[K::VX];
#pragma unroll
    for (int e = 0; e < K::VX; ++e) {
        bias[e] = p.a.delta_bias && e < nx ? __ldg(p.a.delta_bias + at.c0 + col + e) : 0.f;
        skip[e] = p.a.D && e < nx ? __ldg(p.a.D + at.c0 + col + e) : 0.f;
    }
    if (w == 0) {
        St h;
        st_set(h, 0.f);
        if (p.a.state_in) st_load(h, p.a.state_in + at.b * p.a.state_in_batch, f0, fend, S, nl * 4, p.vec_n);
        st_put(sCarry[0], lane, h);
    }
    const T* xp = static_cast<const T*>(p.a.x) + at.b * p.a.x_batch + at.c0 + col;
    const T* dp = static_cast<const T*>(p.a.delta) + at.b * p.a.delta_batch + at.c0 + col;
    const T* zp = static_cast<const T*>(p.a.z) + at.b * p.a.z_batch + at.c0 + col;
    const T* Bp = static_cast<const T*>(p.a.B) + at.b * p.a.B_batch + at.g * p.a.B_group + bcol;
    const T* Cp = static_cast<const T*>(p.a.C) + at.b * p.a.C_batch + at.g * p.a.C_group + bcol;
    T* yp = static_cast<T*>(p.a.y) + static_cast<long long>(at.b) * L * dim + at.c0 + col;

    Vec<T, K::VX> rx, rd;
    Vec<T, K::VN> rB, rC;
    auto fetch = [&](int t) {
        const bool in = t < len;
        rx.load_n(xp + t * p.a.x_time, in ? nx : 0, p.vec_x);
        rd.load_n(dp + t * p.a.delta_time, in ? nx : 0, p.vec_delta);
        rB.load_n(Bp + t * p.a.B_time, in ? nb : 0, p.vec_B);
        rC.load_n(Cp + t * p.a.C_time, in ? nb : 0, p.vec_C);
    };
    const int nck = (len + kScanChunk - 1) / kScanChunk;
    fetch(w * kScanSteps + row);
    for (int ck = 0; ck < nck; ++ck) {
        const int buf = ck & 1;
        const int t = ck * kScanChunk + w * kScanSteps + row;  // the step that this lane stages
        const Vec<T, K::VX> xk = rx;
        __syncwarp();
#pragma unroll
        for (int e = 0; e < K::VX; ++e) {
            float dt = rd.get(e) + bias[e];
            if (p.a.softplus) dt = softplusf(dt);
            if (t >= len) dt = 0.f;  // the state stays as it is
            sU[w][row][col + e] = make_float2(dt, dt * rx.get(e));
        }
#pragma unroll
        for (int e = 0; e < K::VN; ++e) {
            sB[w][row][bcol + e] = rB.get(e);
            sC[w][row][bcol + e] = rC.get(e);
        }
        __syncwarp();

        f2 a[kScanSteps][kCT][2];
        St h, P;
        st_set(h, 0.f);
        st_set(P, 1.f);
#pragma unroll
        for (int s = 0; s < kScanSteps; ++s) {
            const float4 du = *reinterpret_cast<const float4*>(&sU[w][s][cl * kCT]);
            const ulonglong2 bv = *reinterpret_cast<const ulonglong2*>(&sB[w][s][nl * 4]);
#pragma unroll
            for (int i = 0; i < kCT; ++i) {
                const float dt = i ? du.z : du.x, u = i ? du.w : du.y;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    a[s][i][j] = ex22(mul2(pk(dt, dt), A2.v[i][j]));
                    h.v[i][j] = fma2(a[s][i][j], h.v[i][j], mul2(pk(u, u), f2{j ? bv.y : bv.x}));
                    P.v[i][j] = mul2(P.v[i][j], a[s][i][j]);
                }
            }
        }
        st_put(sP[buf][w], lane, P);
        st_put(sE[buf][w], lane, h);
        if (ck + 1 < nck) fetch(t + kScanChunk);
        Vec<T, K::VX> rz;
        if (p.a.z) rz.load_n(zp + t * p.a.z_time, t < len ? nx : 0, p.vec_z);
        // One barrier per chunk: the buffers alternate, and a warp that is a
        // chunk ahead has passed the barrier behind this chunk's reads.
        __syncthreads();
        St hin;
        st_get(hin, sCarry[buf], lane);
        if (w == 0 && p.a.saved)
            st_store(hin, p.a.saved + (static_cast<long long>(at.b) * p.nchunk + ck) * dim * S, f0, fend, S, nl * 4, p.vec_n);
        for (int q = 0; q < w; ++q) st_chain(hin, sP[buf][q], sE[buf][q], lane);
        if (w == kScanWarps - 1) {
            St c = hin;
            st_chain(c, sP[buf][w], sE[buf][w], lane);
            st_put(sCarry[buf ^ 1], lane, c);
        }
        float v[kScanSteps * kCT];
#pragma unroll
        for (int s = 0; s < kScanSteps; ++s) {
            const float4 du = *reinterpret_cast<const float4*>(&sU[w][s][cl * kCT]);
            const ulonglong2 bv = *reinterpret_cast<const ulonglong2*>(&sB[w][s][nl * 4]);
            const ulonglong2 cv = *reinterpret_cast<const ulonglong2*>(&sC[w][s][nl * 4]);
#pragma unroll
            for (int i = 0; i < kCT; ++i) {
                const float u = i ? du.w : du.y;
#pragma unroll
                for (int j = 0; j < 2; ++j) hin.v[i][j] = fma2(a[s][i][j], hin.v[i][j], mul2(pk(u, u), f2{j ? bv.y : bv.x}));
                v[s * kCT + i] = sum2(fma2(f2{cv.y}, hin.v[i][1], mul2(f2{cv.x}, hin.v[i][0])));
            }
        }
        using Sum = LaneSum<kScanSteps * kCT, 1, NL>;
        Sum::run(v, lane);
        float* sY = reinterpret_cast<float*>(sU[w]);  // (dt, u) has been read
        __syncwarp();
        const int slot = Sum::slot(lane);
#pragma unroll
        for (int k = 0; k < Sum::kept; ++k) sY[(slot + k) / kCT * K::CH + cl * kCT + (slot + k) % kCT] = v[k];
        __syncwarp();
        Vec<T, K::VX> o;
#pragma unroll
        for (int e = 0; e < K::VX; ++e) {
            float y = fmaf(skip[e], xk.get(e), sY[row * K::CH + col + e]);
            if (p.a.z) {
                const float z = rz.get(e);
                y *= z * sigmoidf(z);
            }
            o.set(e, t < len ? y : 0.f);
        }
        o.store_n(yp + static_cast<long long>(t) * dim, t < L ? nx : 0, p.vec_y);
    }
    for (int t = nck * kScanChunk + w * kScanSteps + row; t < L; t += kScanChunk) {
        Vec<T, K::VX> o;
        o.zero();
        o.store_n(yp + static_cast<long long>(t) * dim, nx, p.vec_y);
    }
    if (p.a.state_out) {
        __syncthreads();
        if (w == 0) {
            St h;
            st_get(h, sCarry[nck & 1], lane);
            st_store(h, p.a.state_out + at.b * p.a.state_out_batch, f0, fend, S, nl * 4, p.vec_n);
        }
    }
}

// One new step of every series: NL lanes per feature, 4 states each, read and
// written once (the state is all of the traffic).
template <typename T, int NL>
__global__ void __launch_bounds__(128) scan_step_kernel(const ScanP p) {
    const long long i = (static_cast<long long>(blockIdx.x) * 128 + threadIdx.x) / NL;
    const int nl = threadIdx.x % NL, S = p.a.nstate, n0 = nl * 4;
    const bool in = i < static_cast<long long>(p.a.batch) * p.a.dim;
    float y = 0.f, x = 0.f;
    int b = 0, f = 0;
    if (in) {
        b = static_cast<int>(i / p.a.dim);
        f = static_cast<int>(i % p.a.dim);
        const int g = f / p.dg, n = min(max(S - n0, 0), 4);
        Vec<float, 4> A, h;
        A.load_n(p.a.A + static_cast<long long>(f) * S + n0, n, p.vec_n);
        // Plain loads: state_out may be the same tensor.
        const float* hp = p.a.state_in + b * p.a.state_in_batch + static_cast<long long>(f) * S + n0;
        h.zero();
        if (p.vec_n) {
            if (n > 0) {
                const float4 q = *reinterpret_cast<const float4*>(hp);
                h.set(0, q.x);
                h.set(1, q.y);
                h.set(2, q.z);
                h.set(3, q.w);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < n) h.set(j, hp[j]);
        }
        x = to_f(static_cast<const T*>(p.a.x)[b * p.a.x_batch + f]);
        float dt = to_f(static_cast<const T*>(p.a.delta)[b * p.a.delta_batch + f]);
        if (p.a.delta_bias) dt += __ldg(p.a.delta_bias + f);
        if (p.a.softplus) dt = softplusf(dt);
        const T* Bp = static_cast<const T*>(p.a.B) + b * p.a.B_batch + g * p.a.B_group + n0;
        const T* Cp = static_cast<const T*>(p.a.C) + b * p.a.C_batch + g * p.a.C_group + n0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < n) {
                h.set(j, fmaf(ex2f(dt * (A.get(j) * kL2e)), h.get(j), dt * x * to_f(Bp[j])));
                y = fmaf(to_f(Cp[j]), h.get(j), y);
            }
        h.store_n(p.a.state_out + b * p.a.state_out_batch + static_cast<long long>(f) * S + n0, n, p.vec_n);
    }
#pragma unroll
    for (int m = 1; m < NL; m *= 2) y += __shfl_xor_sync(0xffffffffu, y, m);
    if (in && nl == 0) {
        if (p.a.D) y = fmaf(__ldg(p.a.D + f), x, y);
        if (p.a.z) {
            const float z = to_f(static_cast<const T*>(p.a.z)[b * p.a.z_batch + f]);
            y *= z * sigmoidf(z);
        }
        static_cast<T*>(p.a.y)[i] = from_f<T>(y);
    }
}

template <typename T, int NL>
cudaError_t run_scan_fwd(const sdtw_scan_args& a, bool step, cudaStream_t st) {
    ScanP p{};
    scan_params<T, NL>(p, a);
    const long long blocks = step ? (static_cast<long long>(a.batch) * a.dim * NL + 127) / 128 : scan_blocks<NL>(p);
    if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    if (step)
        scan_step_kernel<T, NL><<<static_cast<unsigned>(blocks), 128, 0, st>>>(p);
    else
        scan_fwd_kernel<T, NL><<<static_cast<unsigned>(blocks), kScanThreads, 0, st>>>(p);
    return cudaGetLastError();
}

template <typename T>
cudaError_t run_scan_fwd_t(const sdtw_scan_args& a, bool step, cudaStream_t st) {
    switch (scan_lanes(a.nstate)) {
        case 1: return run_scan_fwd<T, 1>(a, step, st);
        case 2: return run_scan_fwd<T, 2>(a, step, st);
        case 4: return run_scan_fwd<T, 4>(a, step, st);
        case 8: return run_scan_fwd<T, 8>(a, step, st);
        default: return run_scan_fwd<T, 16>(a, step, st);
    }
}

cudaError_t run_scan_fwd_any(const sdtw_scan_args& a, bool step, cudaStream_t st) {
    if (a.dtype == SDTW_F32) return run_scan_fwd_t<float>(a, step, st);
    if (a.dtype == SDTW_F16) return run_scan_fwd_t<__half>(a, step, st);
    return run_scan_fwd_t<__nv_bfloat16>(a, step, st);
}

}  // namespace

size_t scan_states(int batch, int length, int dim, int nstate) {
    return static_cast<size_t>(batch) * ((length + kScanChunk - 1) / kScanChunk) * dim * nstate;
}
cudaError_t launch_scan_fwd(const sdtw_scan_args& a, cudaStream_t st) { return run_scan_fwd_any(a, false, st); }
cudaError_t launch_scan_step(const sdtw_scan_args& a, cudaStream_t st) { return run_scan_fwd_any(a, true, st); }

}  // namespace sdtw

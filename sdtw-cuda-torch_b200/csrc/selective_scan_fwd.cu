// selective_scan_fwd.cu -- forward of the selective scan (see
// selective_scan.cuh for the formulas and the tiling) and its single-step form.
#include <algorithm>
#include <type_traits>

#include "selective_scan.cuh"

namespace sdtw {
namespace {

// One warp per (series, segment, tile of features); the warps of a block do not
// wait for one another.
template <typename T, int NL>
__global__ void __launch_bounds__(kScanThreads) scan_fwd_kernel(const ScanP p, long long warps) {
    using K = ScanTile<NL>;
    // (dt, u) of two features, and once more with the two swapped; later y in the first.
    __shared__ float4 sU[kScanWarps][2][K::TS][K::CH / 2];
    __shared__ __align__(16) float sB[kScanWarps][K::TS][K::NP], sC[kScanWarps][K::TS][K::NP];
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long wi = static_cast<long long>(blockIdx.x) * kScanWarps + w;
    if (wi >= warps) return;
    const ScanPlace<NL> at = ScanPlace<NL>::of_warp(p, wi);
    const int nl = lane % NL, cl = lane / NL, swap = nl & 1, n0 = nl * 4;
    const int S = p.a.nstate, L = p.a.length, dim = p.a.dim;
    const int len = seq_len(p.a.lengths, at.b, L);
    const int f0 = at.c0 + cl * kCT, fend = at.c0 + at.nc;
    const int row = lane / K::LR, col = lane % K::LR * K::VX, bcol = lane % K::LR * K::VN;
    const int nx = min(max(at.nc - col, 0), K::VX), nb = min(max(S - bcol, 0), K::VN);

    St A2, h;
    st_load(A2, p.a.A, f0, swap, fend, S, n0, p.vec_n);
    st_scale(A2, kL2e);
    st_set(h, 0.f);
    if (p.a.state_in) st_load(h, p.a.state_in + at.b * p.a.state_in_batch, f0, swap, fend, S, n0, p.vec_n);
    if (p.nseg > 1) {
        pdl_wait();
        for (int q = 0; q < at.seg; ++q) st_chain(h, p, A2, at.b, q, f0, swap, fend, n0);
    }
    const T* xp = static_cast<const T*>(p.a.x) + at.b * p.a.x_batch + at.c0 + col;
    const T* dp = static_cast<const T*>(p.a.delta) + at.b * p.a.delta_batch + at.c0 + col;
    const T* zp = static_cast<const T*>(p.a.z) + at.b * p.a.z_batch + at.c0 + col;
    const T* Bp = static_cast<const T*>(p.a.B) + at.b * p.a.B_batch + at.g * p.a.B_group + bcol;
    const T* Cp = static_cast<const T*>(p.a.C) + at.b * p.a.C_batch + at.g * p.a.C_group + bcol;
    T* yp = static_cast<T*>(p.a.y) + static_cast<long long>(at.b) * L * dim + at.c0 + col;
    const float* bias = p.a.delta_bias ? p.a.delta_bias + at.c0 + col : nullptr;
    const float* skip = p.a.D ? p.a.D + at.c0 + col : nullptr;

    Vec<T, K::VX> rx, rd;
    Vec<T, K::VN> rB, rC;
    auto fetch = [&](int t) {
        const bool in = t < len;
        rx.load_n(xp + t * p.a.x_time, in ? nx : 0, p.vec_x);
        rd.load_n(dp + t * p.a.delta_time, in ? nx : 0, p.vec_delta);
        rB.load_n(Bp + t * p.a.B_time, in ? nb : 0, p.vec_B);
        rC.load_n(Cp + t * p.a.C_time, in ? nb : 0, p.vec_C);
    };
    const int tend = min(at.t1, len);
    if (at.t0 < tend) fetch(at.t0 + row);
    int tc = at.t0;
    for (; tc < tend; tc += K::TS) {
        const int t = tc + row;  // the step that this lane stages
        const Vec<T, K::VX> xk = rx;
        Vec<T, K::VX> rz;
        if (p.a.z) rz.load_n(zp + t * p.a.z_time, t < len ? nx : 0, p.vec_z);
        __syncwarp();
#pragma unroll
        for (int e = 0; e < K::VX; e += 2) {
            float dt[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                dt[k] = rd.get(e + k) + (bias && e + k < nx ? __ldg(bias + e + k) : 0.f);
                if (p.a.softplus) dt[k] = softplusf(dt[k]);
                if (t >= len) dt[k] = 0.f;  // the state stays as it is
            }
            const float u0 = dt[0] * rx.get(e), u1 = dt[1] * rx.get(e + 1);
            sU[w][0][row][(col + e) / 2] = make_float4(dt[0], u0, dt[1], u1);
            sU[w][1][row][(col + e) / 2] = make_float4(dt[1], u1, dt[0], u0);
        }
#pragma unroll
        for (int e = 0; e < K::VN; ++e) {
            sB[w][row][bcol + e] = rB.get(e);
            sC[w][row][bcol + e] = rC.get(e);
        }
        if (tc + K::TS < tend) fetch(t + K::TS);
        __syncwarp();
        if (p.a.saved)
            st_store(h, p.a.saved + (static_cast<long long>(at.b) * p.nchunk + tc / K::TS) * dim * S, f0, swap, fend, S, n0, p.vec_n);
#pragma unroll 1
        for (int sb = 0; sb < K::TS; sb += kRun) {
            float v[kRun * kCT];
#pragma unroll
            for (int s = 0; s < kRun; ++s) {
                const float4 du = sU[w][swap][sb + s][cl];
                const ulonglong2 bv = *reinterpret_cast<const ulonglong2*>(&sB[w][sb + s][n0]);
                const ulonglong2 cv = *reinterpret_cast<const ulonglong2*>(&sC[w][sb + s][n0]);
#pragma unroll
                for (int i = 0; i < kCT; ++i) {
                    const float dt = i ? du.z : du.x, u = i ? du.w : du.y;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const f2 a = ex22(mul2(pk(dt, dt), A2.v[i][j]));
                        h.v[i][j] = fma2(a, h.v[i][j], mul2(pk(u, u), f2{j ? bv.y : bv.x}));
                    }
                    v[s * kCT + i] = sum2(fma2(f2{cv.y}, h.v[i][1], mul2(f2{cv.x}, h.v[i][0])));
                }
            }
            if constexpr (NL == 1) {
                __syncwarp();
#pragma unroll
                for (int s = 0; s < kRun; ++s)
                    *reinterpret_cast<float2*>(reinterpret_cast<float*>(sU[w][0][sb + s]) + cl * kCT) = make_float2(v[2 * s], v[2 * s + 1]);
            } else {
                float y[kRun];  // per step, of the lane's first feature
                pair_exchange(v, y, 1);
                using Sum = LaneSum<kRun, 2, NL / 2>;
                Sum::run(y, lane);
                __syncwarp();
                const int slot = Sum::slot(lane);
#pragma unroll
                for (int k = 0; k < Sum::kept; ++k)
                    reinterpret_cast<float*>(sU[w][0][sb + slot + k])[cl * kCT + swap] = y[k];
            }
        }
        __syncwarp();
        Vec<T, K::VX> o;
        const float* sY = reinterpret_cast<const float*>(sU[w][0][row]) + col;
#pragma unroll
        for (int e = 0; e < K::VX; ++e) {
            float y = fmaf(skip && e < nx ? __ldg(skip + e) : 0.f, xk.get(e), sY[e]);
            if (p.a.z) {
                const float z = rz.get(e);
                y *= z * sigmoidf(z);
            }
            o.set(e, t < len ? y : 0.f);
        }
        o.store_n(yp + static_cast<long long>(t) * dim, t < at.t1 ? nx : 0, p.vec_y);
    }
    for (int t = tc + row; t < at.t1; t += K::TS) {
        Vec<T, K::VX> o;
        o.zero();
        o.store_n(yp + static_cast<long long>(t) * dim, nx, p.vec_y);
    }
    if (p.a.state_out && at.seg == p.nseg - 1)
        st_store(h, p.a.state_out + at.b * p.a.state_out_batch, f0, swap, fend, S, n0, p.vec_n);
}

// End state and sum of dt of a segment run from 0: see launch_scan_segments.
template <typename T, int NL, bool REV>
__global__ void __launch_bounds__(kScanThreads) scan_segment_kernel(const ScanP p, long long warps) {
    using K = ScanTile<NL>;
    __shared__ float4 sU[kScanWarps][2][K::TS][K::CH / 2];
    __shared__ __align__(16) float sB[kScanWarps][K::TS][K::NP];
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long wi = static_cast<long long>(blockIdx.x) * kScanWarps + w;
    if (wi >= warps) return;
    const ScanPlace<NL> at = ScanPlace<NL>::of_warp(p, wi);
    const int nl = lane % NL, cl = lane / NL, swap = nl & 1, n0 = nl * 4;
    const int S = p.a.nstate, dim = p.a.dim;
    const int len = seq_len(p.a.lengths, at.b, p.a.length);
    const int f0 = at.c0 + cl * kCT, fend = at.c0 + at.nc;
    const int row = lane / K::LR, col = lane % K::LR * K::VX, bcol = lane % K::LR * K::VN;
    const int nx = min(max(at.nc - col, 0), K::VX), nb = min(max(S - bcol, 0), K::VN);
    const long long out = static_cast<long long>(at.b) * p.nseg + at.seg;
    St A2, h;
    st_load(A2, p.a.A, f0, swap, fend, S, n0, p.vec_n);
    st_scale(A2, kL2e);
    st_set(h, 0.f);
    float sum[kCT] = {};
    const T* xp = static_cast<const T*>(REV ? p.a.dy : p.a.x) + at.b * (REV ? p.a.dy_batch : p.a.x_batch) + at.c0 + col;
    const T* dp = static_cast<const T*>(p.a.delta) + at.b * p.a.delta_batch + at.c0 + col;
    const T* zp = static_cast<const T*>(p.a.z) + at.b * p.a.z_batch + at.c0 + col;
    const T* Bp = static_cast<const T*>(REV ? p.a.C : p.a.B) + at.b * (REV ? p.a.C_batch : p.a.B_batch) +
                  at.g * (REV ? p.a.C_group : p.a.B_group) + bcol;
    const long long x_time = REV ? p.a.dy_time : p.a.x_time, B_time = REV ? p.a.C_time : p.a.B_time;
    const bool vec_x = REV ? p.vec_dy : p.vec_x, vec_B = REV ? p.vec_C : p.vec_B;
    const float* bias = p.a.delta_bias ? p.a.delta_bias + at.c0 + col : nullptr;
    const int tend = min(at.t1, len), n = tend > at.t0 ? (tend - at.t0 + K::TS - 1) / K::TS : 0;
    for (int k = 0; k < n; ++k) {
        const int t = at.t0 + (REV ? n - 1 - k : k) * K::TS + row;
        const bool in = t < len;
        Vec<T, K::VX> rx, rd, rz;
        Vec<T, K::VN> rB;
        rx.load_n(xp + t * x_time, in ? nx : 0, vec_x);
        rd.load_n(dp + t * p.a.delta_time, in ? nx : 0, p.vec_delta);
        if (REV && p.a.z) rz.load_n(zp + t * p.a.z_time, in ? nx : 0, p.vec_z);
        rB.load_n(Bp + t * B_time, in ? nb : 0, vec_B);
        __syncwarp();
#pragma unroll
        for (int e = 0; e < K::VX; e += 2) {
            float dt[2], u[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                dt[q] = rd.get(e + q) + (bias && e + q < nx ? __ldg(bias + e + q) : 0.f);
                if (p.a.softplus) dt[q] = softplusf(dt[q]);
                if (!in) dt[q] = 0.f;
                u[q] = rx.get(e + q);
                if (!REV) u[q] *= dt[q];
                if (REV && p.a.z) u[q] *= rz.get(e + q) * sigmoidf(rz.get(e + q));
            }
            sU[w][0][row][(col + e) / 2] = make_float4(dt[0], u[0], dt[1], u[1]);
            sU[w][1][row][(col + e) / 2] = make_float4(dt[1], u[1], dt[0], u[0]);
        }
#pragma unroll
        for (int e = 0; e < K::VN; ++e) sB[w][row][bcol + e] = rB.get(e);
        __syncwarp();
#pragma unroll 8
        for (int i8 = 0; i8 < K::TS; ++i8) {
            const int s = REV ? K::TS - 1 - i8 : i8;
            const float4 du = sU[w][swap][s][cl];
            const ulonglong2 bv = *reinterpret_cast<const ulonglong2*>(&sB[w][s][n0]);
#pragma unroll
            for (int i = 0; i < kCT; ++i) {
                const float dt = i ? du.z : du.x, u = i ? du.w : du.y;
                sum[i] += dt;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const f2 a = ex22(mul2(pk(dt, dt), A2.v[i][j])), b{j ? bv.y : bv.x};
                    h.v[i][j] = REV ? mul2(a, fma2(pk(u, u), b, h.v[i][j])) : fma2(a, h.v[i][j], mul2(pk(u, u), b));
                }
            }
        }
    }
    st_store(h, p.seg_E + out * dim * S, f0, swap, fend, S, n0, p.vec_n);
    if (nl == 0) {
#pragma unroll
        for (int i = 0; i < kCT; ++i)
            if (f0 + i < fend) p.seg_dt[out * dim + f0 + i] = sum[i];
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

// Dispatch over the types and the lanes per feature.
template <typename F>
cudaError_t scan_dispatch(const sdtw_scan_args& a, F&& f) {
    auto lanes = [&](auto type) -> cudaError_t {
        switch (scan_lanes(a.nstate)) {
            case 1: return f(type, std::integral_constant<int, 1>{});
            case 2: return f(type, std::integral_constant<int, 2>{});
            case 4: return f(type, std::integral_constant<int, 4>{});
            case 8: return f(type, std::integral_constant<int, 8>{});
            default: return f(type, std::integral_constant<int, 16>{});
        }
    };
    if (a.dtype == SDTW_F32) return lanes(float{});
    if (a.dtype == SDTW_F16) return lanes(__half{});
    return lanes(__nv_bfloat16{});
}

bool grid_of(long long warps, unsigned* blocks) {
    const long long n = (warps + kScanWarps - 1) / kScanWarps;
    *blocks = static_cast<unsigned>(n);
    return n <= 0x7fffffffll;
}

}  // namespace

// Segments of the time axis: none while there are two warps per SM
// sub-partition or nearly so; else enough for that, of 64 steps at least.
ScanSplit scan_split(int batch, int length, int dim, int groups, int nstate, bool backward) {
    const int nl = scan_lanes(nstate), ch = 32 / nl * kCT, ts = scan_stage_steps(nl), dg = dim / groups;
    const long long warps = static_cast<long long>(batch) * groups * ((dg + ch - 1) / ch);
    (void)backward;
    long long n = 1184 / warps;
    n = std::min<long long>(n, length / 64);
    if (n < 3) n = 1;
    ScanSplit s;
    s.seglen = static_cast<int>(((length + n - 1) / n + ts - 1) / ts * ts);
    s.nseg = (length + s.seglen - 1) / s.seglen;
    return s;
}

size_t scan_states(int batch, int length, int dim, int nstate) {
    const int ts = scan_stage_steps(scan_lanes(nstate));
    return static_cast<size_t>(batch) * ((length + ts - 1) / ts) * dim * nstate;
}
size_t scan_fwd_ws(int batch, int length, int dim, int groups, int nstate) {
    return scan_segment_floats(batch, scan_split(batch, length, dim, groups, nstate, false).nseg, dim, nstate) * sizeof(float);
}

cudaError_t launch_scan_segments(const ScanP& p, bool reverse, cudaStream_t st) {
    return scan_dispatch(p.a, [&](auto type, auto lanes) -> cudaError_t {
        using T = decltype(type);
        constexpr int NL = decltype(lanes)::value;
        const long long warps = static_cast<long long>(p.a.batch) * p.nseg * p.tiles_g * p.a.groups;
        unsigned blocks;
        if (!grid_of(warps, &blocks)) return cudaErrorInvalidConfiguration;
        if (reverse)
            scan_segment_kernel<T, NL, true><<<blocks, kScanThreads, 0, st>>>(p, warps);
        else
            scan_segment_kernel<T, NL, false><<<blocks, kScanThreads, 0, st>>>(p, warps);
        return cudaGetLastError();
    });
}

cudaError_t launch_scan_fwd(const sdtw_scan_args& a, cudaStream_t st) {
    return scan_dispatch(a, [&](auto type, auto lanes) -> cudaError_t {
        using T = decltype(type);
        constexpr int NL = decltype(lanes)::value;
        ScanP p{};
        scan_params<T, NL>(p, a);
        scan_segment_tables(p, scan_split(a.batch, a.length, a.dim, a.groups, a.nstate, false), a.workspace);
        const long long warps = static_cast<long long>(a.batch) * p.nseg * p.tiles_g * a.groups;
        unsigned blocks;
        if (!grid_of(warps, &blocks)) return cudaErrorInvalidConfiguration;
        if (p.nseg > 1) {
            const cudaError_t e = launch_scan_segments(p, false, st);
            if (e != cudaSuccess) return e;
        }
        return launch_pdl(p.nseg > 1, scan_fwd_kernel<T, NL>, dim3(blocks), dim3(kScanThreads), 0, st, p, warps);
    });
}

cudaError_t launch_scan_step(const sdtw_scan_args& a, cudaStream_t st) {
    return scan_dispatch(a, [&](auto type, auto lanes) -> cudaError_t {
        using T = decltype(type);
        constexpr int NL = decltype(lanes)::value;
        ScanP p{};
        scan_params<T, NL>(p, a);
        const long long blocks = (static_cast<long long>(a.batch) * a.dim * NL + 127) / 128;
        if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
        scan_step_kernel<T, NL><<<static_cast<unsigned>(blocks), 128, 0, st>>>(p);
        return cudaGetLastError();
    });
}

}  // namespace sdtw

// causal_conv.cu -- causal convolution of each feature over time, and its gradient.
//
//   v[t] = bias + sum_k w[k] s[t + k],  y = v or v sigmoid(v),  k < W
// with s = (the W - 1 inputs before the series) followed by x, so that x[t] is
// s[t + W - 1].  With gv = dL/dv (dy, or dy times the derivative of v sigmoid(v)):
//   dL/ds[i] = sum_k w[k] gv[i - k],   dw[k] = sum_t gv[t] s[t + k],   dbias = sum_t gv[t]
//
// Memory bound (a forward reads x and writes y, a backward reads x and dy and
// writes dx; W + 1 multiply-adds per element).  A thread owns VEC neighbouring
// features and walks over a tile of time steps with the last W - 1 steps in
// registers, so each element is read once and only the W - 1 steps before (and,
// in the backward, behind) a tile twice.  The backward computes v again from x
// instead of storing it, and keeps the thread's dw and dbias in registers; the
// blocks' partial sums are added by a second kernel in a fixed order.
#include <algorithm>

#include "seq_device.cuh"
#include "seq_kernels.h"

namespace sdtw {
namespace {

constexpr int kThreads = 128;
constexpr int kU = 4;  // time steps whose loads are issued together

struct ConvP {
    sdtw_conv_args a;
    int cx;      // threads over features (a power of two); kThreads / cx tiles per block
    int tt;      // time steps per tile, a multiple of kU and >= 16
    int nch;     // groups of VEC features
    int nchb;    // blocks over features
    int ntb;     // blocks over time
    bool vec_x, vec_y, vec_s, vec_so, vec_dy, vec_dx, vec_dso;
    float* part;
};

// Tile length: long tiles re-read less; shorter ones when there would be too
// few threads to fill the GPU (148 SMs x 1024).
int conv_tile(int batch, int length, int nch) {
    int tt = 64;
    while (tt > 16 && static_cast<long long>(batch) * ((length + tt - 1) / tt) * nch < 148ll * 1024) tt /= 2;
    return tt;
}
constexpr int kBwdVec = 4;  // 8 features' windows of x and gv, weights and dw would not fit in registers

void conv_geometry(ConvP& p, int vec) {
    p.nch = (p.a.dim + vec - 1) / vec;
    p.cx = 1;
    while (p.cx < 32 && p.cx < p.nch) p.cx *= 2;
    p.tt = conv_tile(p.a.batch, p.a.length, p.nch);
    const int tiles = (p.a.length + p.tt - 1) / p.tt, ry = kThreads / p.cx;
    p.nchb = (p.nch + p.cx - 1) / p.cx;
    p.ntb = (tiles + ry - 1) / ry;
}

// WT is the width, or 0 for a width that is not 2, 3 or 4 (arrays of kConvMaxWidth).
template <int WT>
struct Width {
    static constexpr int kMax = WT ? WT : kConvMaxWidth;
    __device__ static __forceinline__ int get(int w) { return WT ? WT : w; }
};

// s[i] for i < W - 1 + len: a step before the series or of it.
template <typename T, int VEC>
__device__ __forceinline__ void load_s(const ConvP& p, int b, int c, int n, int i, int W, int len, Vec<T, VEC>& v) {
    const int t = i - (W - 1);
    if (t >= 0 && t < len)
        v.load_n(static_cast<const T*>(p.a.x) + b * p.a.x_batch + t * p.a.x_time + c, n, p.vec_x);
    else if (t < 0 && p.a.state_in)
        v.load_n(static_cast<const T*>(p.a.state_in) + b * p.a.state_in_batch + static_cast<long long>(i) * p.a.dim + c, n, p.vec_s);
    else
        v.zero();
}

template <typename T, int VEC, int WT>
__device__ __forceinline__ void load_weights(const ConvP& p, int c, int n, int W, float (&w)[Width<WT>::kMax][VEC],
                                             float (&bias)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
#pragma unroll
        for (int k = 0; k < Width<WT>::kMax; ++k)
            w[k][e] = (k < W && e < n) ? __ldg(p.a.weight + static_cast<long long>(c + e) * W + k) : 0.f;
        bias[e] = (p.a.bias && e < n) ? __ldg(p.a.bias + c + e) : 0.f;
    }
}

template <typename T, int VEC, int WT>
__global__ void __launch_bounds__(kThreads) conv_fwd_kernel(const ConvP p) {
    constexpr int KM = Width<WT>::kMax;
    const int W = Width<WT>::get(p.a.width);
    const int ci = (blockIdx.x % p.nchb) * p.cx + threadIdx.x % p.cx;
    const int rest = blockIdx.x / p.nchb;
    const int tile = (rest % p.ntb) * (kThreads / p.cx) + threadIdx.x / p.cx;
    const int b = rest / p.ntb;
    const long long t0 = static_cast<long long>(tile) * p.tt;
    const int c = ci * VEC;
    if (ci >= p.nch || (t0 >= p.a.length)) return;
    const int n = min(VEC, p.a.dim - c);
    const int t1 = static_cast<int>(min(t0 + p.tt, static_cast<long long>(p.a.length)));
    const int len = seq_len(p.a.lengths, b, p.a.length);
    float w[KM][VEC], bias[VEC];
    load_weights<T, VEC, WT>(p, c, n, W, w, bias);
    float xs[KM - 1 + kU][VEC];  // xs[W - 1 + u]: step t + u; before it, its past
#pragma unroll
    for (int k = 0; k < KM - 1; ++k)
        if (k < W - 1) {
            Vec<T, VEC> r;
            load_s<T, VEC>(p, b, c, n, static_cast<int>(t0) + k, W, len, r);
#pragma unroll
            for (int e = 0; e < VEC; ++e) xs[k][e] = r.get(e);
        }
    const T* xp = static_cast<const T*>(p.a.x) + b * p.a.x_batch + c;
    T* yp = static_cast<T*>(p.a.y) + static_cast<long long>(b) * p.a.length * p.a.dim + c;
    for (int t = static_cast<int>(t0); t < t1; t += kU) {
        Vec<T, VEC> raw[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            if (t + u < min(t1, len))
                raw[u].load_n(xp + (t + u) * p.a.x_time, n, p.vec_x);
            else
                raw[u].zero();
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            float v[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float cur = raw[u].get(e);
                v[e] = bias[e];
                if constexpr (WT != 0) {
                    xs[W - 1 + u][e] = cur;
#pragma unroll
                    for (int k = 0; k < KM; ++k) v[e] = fmaf(w[k][e], xs[k + u][e], v[e]);
                } else {  // runtime width: xs holds the past, moved up at every step
#pragma unroll
                    for (int k = 0; k < KM; ++k)
                        if (k < W) {
                            const float s = k == W - 1 ? cur : xs[k][e];
                            v[e] = fmaf(w[k][e], s, v[e]);
                        }
#pragma unroll
                    for (int k = 0; k < KM - 1; ++k)
                        if (k < W - 1) xs[k][e] = k == W - 2 ? cur : xs[k + 1][e];
                }
            }
            if (t + u < t1) {
                Vec<T, VEC> o;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float y = p.a.silu ? v[e] * sigmoidf(v[e]) : v[e];
                    o.set(e, t + u < len ? y : 0.f);
                }
                o.store_n(yp + static_cast<long long>(t + u) * p.a.dim, n, p.vec_y);
            }
        }
        if constexpr (WT != 0) {
#pragma unroll
            for (int k = 0; k < KM - 1; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) xs[k][e] = xs[k + kU][e];
        }
    }
    if (p.a.state_out && tile == 0) {
        for (int k = 0; k < W - 1; ++k) {
            Vec<T, VEC> r;
            load_s<T, VEC>(p, b, c, n, len + k, W, len, r);
            r.store_n(static_cast<T*>(p.a.state_out) + b * p.a.state_out_batch + static_cast<long long>(k) * p.a.dim + c, n, p.vec_so);
        }
    }
}

template <typename T, int VEC, int WT>
__global__ void __launch_bounds__(kThreads) conv_bwd_kernel(const ConvP p) {
    constexpr int KM = Width<WT>::kMax;
    const int W = Width<WT>::get(p.a.width);
    const int tx = threadIdx.x % p.cx;
    const int ci = (blockIdx.x % p.nchb) * p.cx + tx;
    const int rest = blockIdx.x / p.nchb;
    const int tile = (rest % p.ntb) * (kThreads / p.cx) + threadIdx.x / p.cx;
    const int b = rest / p.ntb;
    const long long t0l = static_cast<long long>(tile) * p.tt;
    const int c = ci * VEC;
    const bool live = ci < p.nch && t0l < p.a.length;
    float dw[KM][VEC], db[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        db[e] = 0.f;
#pragma unroll
        for (int k = 0; k < KM; ++k) dw[k][e] = 0.f;
    }
    if (live) {
        const int n = min(VEC, p.a.dim - c);
        const int t0 = static_cast<int>(t0l);
        const int t1 = min(t0 + p.tt, p.a.length);
        const int len = seq_len(p.a.lengths, b, p.a.length);
        float w[KM][VEC], bias[VEC];
        load_weights<T, VEC, WT>(p, c, n, W, w, bias);
        // The last W - 1 steps: of s oldest first, of gv newest first.
        float xs[KM][VEC], gs[KM][VEC];
#pragma unroll
        for (int k = 0; k < KM; ++k) {
            if (k < W - 1) {
                Vec<T, VEC> r;
                load_s<T, VEC>(p, b, c, n, t0 + k, W, len, r);
#pragma unroll
                for (int e = 0; e < VEC; ++e) xs[k][e] = r.get(e);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) gs[k][e] = 0.f;
        }
        const T* xp = static_cast<const T*>(p.a.x) + b * p.a.x_batch + c;
        const T* gp = static_cast<const T*>(p.a.dy) + b * p.a.dy_batch + c;
        T* dxp = static_cast<T*>(p.a.dx) + static_cast<long long>(b) * p.a.length * p.a.dim + c;
        // Step j brings gv[j] and with it dL/ds[j], which is the gradient of
        // x[j - (W - 1)]; the W - 1 steps behind the tile complete its last ones.
        const int j_end = t1 + W - 1;
        for (int j0 = t0; j0 < j_end; j0 += kU) {
            Vec<T, VEC> rx[kU], rg[kU];
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int nr = j0 + u < min(j_end, len) ? n : 0;
                rx[u].load_n(xp + (j0 + u) * p.a.x_time, nr, p.vec_x);
                rg[u].load_n(gp + (j0 + u) * p.a.dy_time, nr, p.vec_dy);
            }
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int j = j0 + u, t = j - (W - 1);
                const bool own = j < t1;
                float ds[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float cur = rx[u].get(e);
                    float g = rg[u].get(e);
                    if (p.a.silu) {
                        float v = bias[e];
#pragma unroll
                        for (int k = 0; k < KM; ++k)
                            if (k < W) v = fmaf(w[k][e], k == W - 1 ? cur : xs[k][e], v);
                        g *= dsilu(v);
                    }
                    if (j >= len) g = 0.f;
                    if (own) db[e] += g;
                    ds[e] = 0.f;
#pragma unroll
                    for (int k = 0; k < KM; ++k)
                        if (k < W) {
                            if (own) dw[k][e] = fmaf(g, k == W - 1 ? cur : xs[k][e], dw[k][e]);
                            ds[e] = fmaf(w[k][e], k == 0 ? g : gs[k > 0 ? k - 1 : 0][e], ds[e]);
                        }
#pragma unroll
                    for (int k = 0; k < KM - 1; ++k)
                        if (k < W - 1) xs[k][e] = k == W - 2 ? cur : xs[k + 1][e];
#pragma unroll
                    for (int k = KM - 1; k > 0; --k) gs[k][e] = gs[k - 1][e];
                    gs[0][e] = g;
                }
                if (p.a.dx && t >= t0 && t < t1) {
                    if (p.a.dstate_out && t < len && j >= len) {
                        Vec<T, VEC> r;
                        r.load_n(static_cast<const T*>(p.a.dstate_out) + (static_cast<long long>(b) * (W - 1) + (j - len)) * p.a.dim + c, n,
                                 p.vec_dso);
#pragma unroll
                        for (int e = 0; e < VEC; ++e) ds[e] += r.get(e);
                    }
                    Vec<T, VEC> o;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) o.set(e, t < len ? ds[e] : 0.f);
                    o.store_n(dxp + static_cast<long long>(t) * p.a.dim, n, p.vec_dx);
                }
            }
        }
    }
    if (p.part == nullptr) return;
    // The block's tiles, then one partial row of (W + 1) x dim per block.
    __shared__ float acc[kThreads * VEC];
    float* out = p.part + static_cast<size_t>(rest) * (W + 1) * p.a.dim;
    for (int k = 0; k <= W; ++k) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            float v = db[e];
#pragma unroll
            for (int q = 0; q < KM; ++q)
                if (q == k && k < W) v = dw[q][e];
            acc[threadIdx.x * VEC + e] = v;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < p.cx * VEC; i += kThreads) {
            float s = 0.f;
            for (int r = 0; r < kThreads / p.cx; ++r) s += acc[r * p.cx * VEC + i];
            const int col = (blockIdx.x % p.nchb) * p.cx * VEC + i;
            if (col < p.a.dim) out[static_cast<size_t>(k) * p.a.dim + col] = s;
        }
    }
}

__global__ void __launch_bounds__(1024) conv_reduce_kernel(const float* part, int nblk, int dim, int W, float* dw, float* db) {
    __shared__ float acc[32][33];
    pdl_wait();
    const long long cols = static_cast<long long>(W + 1) * dim;
    const long long c = blockIdx.x * 32ll + threadIdx.x;
    float s = 0.f;
    if (c < cols)
#pragma unroll 4
        for (int i = threadIdx.y; i < nblk; i += 32) s += part[i * cols + c];
    acc[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    s = warp_sum(acc[threadIdx.x][threadIdx.y]);
    const long long o = blockIdx.x * 32ll + threadIdx.y;
    if (threadIdx.x == 0 && o < cols) {
        const int k = static_cast<int>(o / dim), f = static_cast<int>(o % dim);
        if (k < W) {
            if (dw) dw[static_cast<long long>(f) * W + k] = s;
        } else if (db) {
            db[f] = s;
        }
    }
}

// Gradient of the W - 1 inputs before the series, which the first W - 1 values
// of gv alone determine: one thread per feature and series.
template <typename T>
__global__ void __launch_bounds__(kThreads) conv_dstate_kernel(const ConvP p) {
    const long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= static_cast<long long>(p.a.batch) * p.a.dim) return;
    const int b = static_cast<int>(i / p.a.dim), c = static_cast<int>(i % p.a.dim), W = p.a.width;
    const int len = seq_len(p.a.lengths, b, p.a.length);
    const T* xp = static_cast<const T*>(p.a.x) + b * p.a.x_batch + c;
    const T* gp = static_cast<const T*>(p.a.dy) + b * p.a.dy_batch + c;
    const T* sp = static_cast<const T*>(p.a.state_in) + b * p.a.state_in_batch + c;
    const T* op = static_cast<const T*>(p.a.dstate_out) + static_cast<long long>(b) * (W - 1) * p.a.dim + c;
    T* dp = static_cast<T*>(p.a.dstate_in) + static_cast<long long>(b) * (W - 1) * p.a.dim + c;
    const float* wp = p.a.weight + static_cast<long long>(c) * W;
    for (int j = 0; j < W - 1; ++j) {
        float ds = 0.f;
        for (int k = 0; k <= j; ++k) {  // w[k] gv[j - k]
            const int t = j - k;
            if (t >= len) continue;
            float g = to_f(gp[t * p.a.dy_time]);
            if (p.a.silu) {
                float v = p.a.bias ? p.a.bias[c] : 0.f;
                for (int q = 0; q < W; ++q) {
                    const int at = t + q - (W - 1);
                    float s = 0.f;
                    if (at >= 0)
                        s = to_f(xp[at * p.a.x_time]);
                    else if (p.a.state_in)
                        s = to_f(sp[static_cast<long long>(t + q) * p.a.dim]);
                    v = fmaf(wp[q], s, v);
                }
                g *= dsilu(v);
            }
            ds = fmaf(wp[k], g, ds);
        }
        if (p.a.dstate_out && j >= len) ds += to_f(op[static_cast<long long>(j - len) * p.a.dim]);
        dp[static_cast<long long>(j) * p.a.dim] = from_f<T>(ds);
    }
}

// One new step of every series: one thread per feature and series.
template <typename T>
__global__ void __launch_bounds__(kThreads) conv_step_kernel(const ConvP p) {
    const long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= static_cast<long long>(p.a.batch) * p.a.dim) return;
    const int b = static_cast<int>(i / p.a.dim), c = static_cast<int>(i % p.a.dim), W = p.a.width;
    const T* si = static_cast<const T*>(p.a.state_in) + b * p.a.state_in_batch + c;
    T* so = static_cast<T*>(p.a.state_out) + b * p.a.state_out_batch + c;
    const T cur = static_cast<const T*>(p.a.x)[b * p.a.x_batch + c];
    T s[kConvMaxWidth];
    // All reads before the writes: the two states may be one tensor.
#pragma unroll
    for (int k = 0; k < kConvMaxWidth; ++k) s[k] = k < W - 1 ? si[static_cast<long long>(k) * p.a.dim] : cur;
    float v = p.a.bias ? __ldg(p.a.bias + c) : 0.f;
#pragma unroll
    for (int k = 0; k < kConvMaxWidth; ++k)
        if (k < W) v = fmaf(__ldg(p.a.weight + static_cast<long long>(c) * W + k), to_f(s[k]), v);
#pragma unroll
    for (int k = 0; k < kConvMaxWidth - 1; ++k)
        if (k < W - 1) so[static_cast<long long>(k) * p.a.dim] = s[k + 1];
    static_cast<T*>(p.a.y)[i] = from_f<T>(p.a.silu ? v * sigmoidf(v) : v);
}

template <typename T, int VEC>
void conv_flags(ConvP& p) {
    const sdtw_conv_args& a = p.a;
    const bool d = a.dim % VEC == 0;
    const long long ds = static_cast<long long>(a.dim);
    p.vec_x = d && vec_ok<T, VEC>(a.x, a.x_batch, a.x_time);
    p.vec_y = d && vec_ok<T, VEC>(a.y, ds, 0);
    p.vec_s = d && vec_ok<T, VEC>(a.state_in, a.state_in_batch, ds);
    p.vec_so = d && vec_ok<T, VEC>(a.state_out, a.state_out_batch, ds);
    p.vec_dy = d && vec_ok<T, VEC>(a.dy, a.dy_batch, a.dy_time);
    p.vec_dx = d && vec_ok<T, VEC>(a.dx, ds, 0);
    p.vec_dso = d && vec_ok<T, VEC>(a.dstate_out, ds, 0);
}

template <typename T, int VEC, bool BWD>
cudaError_t run_conv(const sdtw_conv_args& a, cudaStream_t st) {
    ConvP p{};
    p.a = a;
    conv_geometry(p, VEC);
    conv_flags<T, VEC>(p);
    if (BWD && (a.dweight || a.dbias)) p.part = static_cast<float*>(a.workspace);
    const long long blocks = static_cast<long long>(p.nchb) * p.ntb * a.batch;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    const unsigned g = static_cast<unsigned>(blocks);
    auto go = [&](auto width) {
        constexpr int WT = decltype(width)::value;
        if constexpr (BWD)
            conv_bwd_kernel<T, VEC, WT><<<g, kThreads, 0, st>>>(p);
        else
            conv_fwd_kernel<T, VEC, WT><<<g, kThreads, 0, st>>>(p);
    };
    if (a.width == 2) go(std::integral_constant<int, 2>{});
    else if (a.width == 3) go(std::integral_constant<int, 3>{});
    else if (a.width == 4) go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 0>{});
    cudaError_t e = cudaGetLastError();
    if constexpr (BWD)
        if (e == cudaSuccess && a.dstate_in && a.width > 1) {
            const long long n = (static_cast<long long>(a.batch) * a.dim + kThreads - 1) / kThreads;
            conv_dstate_kernel<T><<<static_cast<unsigned>(n), kThreads, 0, st>>>(p);
            e = cudaGetLastError();
        }
    if (e != cudaSuccess || !BWD || !p.part) return e;
    const long long cols = static_cast<long long>(a.width + 1) * a.dim;
    return launch_pdl(true, conv_reduce_kernel, dim3(static_cast<unsigned>((cols + 31) / 32)), dim3(32, 32), 0, st,
                      static_cast<const float*>(p.part), p.ntb * a.batch, a.dim, a.width, a.dweight, a.dbias);
}

}  // namespace

size_t conv_bwd_ws(int batch, int length, int dim, int width) {
    ConvP p{};
    p.a.batch = batch;
    p.a.length = length;
    p.a.dim = dim;
    conv_geometry(p, kBwdVec);
    return static_cast<size_t>(p.ntb) * batch * (width + 1) * static_cast<size_t>(dim) * sizeof(float);
}

cudaError_t launch_conv_fwd(const sdtw_conv_args& a, cudaStream_t st) {
    if (a.dtype == SDTW_F32) return run_conv<float, 4, false>(a, st);
    if (a.dtype == SDTW_F16) return run_conv<__half, 8, false>(a, st);
    return run_conv<__nv_bfloat16, 8, false>(a, st);
}
cudaError_t launch_conv_bwd(const sdtw_conv_args& a, cudaStream_t st) {
    if (a.dtype == SDTW_F32) return run_conv<float, kBwdVec, true>(a, st);
    if (a.dtype == SDTW_F16) return run_conv<__half, kBwdVec, true>(a, st);
    return run_conv<__nv_bfloat16, kBwdVec, true>(a, st);
}
cudaError_t launch_conv_step(const sdtw_conv_args& a, cudaStream_t st) {
    ConvP p{};
    p.a = a;
    const long long blocks = (static_cast<long long>(a.batch) * a.dim + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    const unsigned g = static_cast<unsigned>(blocks);
    if (a.dtype == SDTW_F32) conv_step_kernel<float><<<g, kThreads, 0, st>>>(p);
    else if (a.dtype == SDTW_F16) conv_step_kernel<__half><<<g, kThreads, 0, st>>>(p);
    else conv_step_kernel<__nv_bfloat16><<<g, kThreads, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace sdtw

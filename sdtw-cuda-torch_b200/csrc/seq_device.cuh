// seq_device.cuh -- device helpers of the sequence operators: element types,
// vector loads and stores with a guarded fallback, lane reductions, packed
// float32 pairs.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "sdtw_device.cuh"

namespace sdtw {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The 16-bit halves of a word as floats, and back.
template <typename T>
__device__ __forceinline__ float half_bits(uint32_t h);
template <>
__device__ __forceinline__ float half_bits<__half>(uint32_t h) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(h)));
}
template <>
__device__ __forceinline__ float half_bits<__nv_bfloat16>(uint32_t h) { return __uint_as_float(h << 16); }
__device__ __forceinline__ uint32_t bits_of(__half v) { return __half_as_ushort(v); }
__device__ __forceinline__ uint32_t bits_of(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }

// Two floats as 16-bit elements, the first in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pair_bits(float a, float b);
template <>
__device__ __forceinline__ uint32_t pair_bits<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    uint32_t r;
    memcpy(&r, &v, 4);
    return r;
}
template <>
__device__ __forceinline__ uint32_t pair_bits<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    uint32_t r;
    memcpy(&r, &v, 4);
    return r;
}

// V elements in 32-bit words, moved in pieces of at most 16 bytes.  16-bit
// elements are loaded as unsigned short: the headers' __ldg of __half and
// __nv_bfloat16 is an asm statement without `volatile`, which the compiler may
// move in front of the condition that guards it (seen as an illegal address
// when the guarded pointer was null).
template <typename T, int V>
struct Vec {
    static constexpr bool k32 = sizeof(T) == 4;
    static constexpr int kWords = k32 ? V : (V + 1) / 2;
    static constexpr int kBytes = V * static_cast<int>(sizeof(T));
    static constexpr int kPiece = kBytes < 16 ? kBytes : 16;  // bytes of one access
    uint32_t w[kWords];

    __device__ __forceinline__ float get(int e) const {
        if constexpr (k32)
            return __uint_as_float(w[e]);
        else
            return half_bits<T>(e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu);
    }
    // Rounds V floats.  Pairs at a time: a pair's conversion is one instruction
    // of the ALU, a single one's takes the unit of the exponentials.
    __device__ __forceinline__ void put(const float (&v)[V]) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (k32)
                w[i] = __float_as_uint(v[i]);
            else if constexpr (V == 1)
                w[i] = bits_of(from_f<T>(v[0]));
            else
                w[i] = pair_bits<T>(v[2 * i], v[2 * i + 1]);
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kPiece == 16) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) {
                const uint4 q = __ldg(reinterpret_cast<const uint4*>(p) + i);
                w[4 * i] = q.x;
                w[4 * i + 1] = q.y;
                w[4 * i + 2] = q.z;
                w[4 * i + 3] = q.w;
            }
        } else if constexpr (kPiece == 8) {
            const uint2 q = __ldg(reinterpret_cast<const uint2*>(p));
            w[0] = q.x;
            w[1] = q.y;
        } else if constexpr (kPiece == 4) {
            w[0] = __ldg(reinterpret_cast<const unsigned int*>(p));
        } else {
            w[0] = __ldg(reinterpret_cast<const unsigned short*>(p));
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (kPiece == 16) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i)
                reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        } else if constexpr (kPiece == 8) {
            *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        } else if constexpr (kPiece == 4) {
            *reinterpret_cast<unsigned int*>(p) = w[0];
        } else {
            *reinterpret_cast<unsigned short*>(p) = static_cast<unsigned short>(w[0]);
        }
    }
    // From shared memory, aligned for whole pieces.
    __device__ __forceinline__ void load_shared(const T* p) {
        if constexpr (kPiece == 16) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) {
                const uint4 q = reinterpret_cast<const uint4*>(p)[i];
                w[4 * i] = q.x;
                w[4 * i + 1] = q.y;
                w[4 * i + 2] = q.z;
                w[4 * i + 3] = q.w;
            }
        } else if constexpr (kPiece == 8) {
            const uint2 q = *reinterpret_cast<const uint2*>(p);
            w[0] = q.x;
            w[1] = q.y;
        } else if constexpr (kPiece == 4) {
            w[0] = *reinterpret_cast<const unsigned int*>(p);
        } else {
            w[0] = *reinterpret_cast<const unsigned short*>(p);
        }
    }
    // n of the V elements exist at p (the others read as 0); `vec`: p is
    // aligned for whole pieces and n is 0 or V.
    __device__ __forceinline__ void load_n(const T* p, int n, bool vec) {
        zero();
        if (vec) {
            if (n > 0) load(p);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < n) {
                    if constexpr (k32)
                        w[i] = __float_as_uint(__ldg(reinterpret_cast<const float*>(p) + i));
                    else
                        w[i / 2] |= static_cast<uint32_t>(__ldg(reinterpret_cast<const unsigned short*>(p) + i)) << (i & 1 ? 16 : 0);
                }
        }
    }
    __device__ __forceinline__ void store_n(T* p, int n, bool vec) const {
        if (vec) {
            if (n > 0) store(p);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < n) {
                    if constexpr (k32)
                        reinterpret_cast<float*>(p)[i] = __uint_as_float(w[i]);
                    else
                        reinterpret_cast<unsigned short*>(p)[i] = static_cast<unsigned short>(i & 1 ? w[i / 2] >> 16 : w[i / 2]);
                }
        }
    }
};

// Whether groups of V elements at p + (multiples of the strides and of V) can
// be moved in Vec's pieces.
template <typename T, int V>
inline bool vec_ok(const void* p, long long s0, long long s1, long long s2 = 0) {
    const uintptr_t piece = Vec<T, V>::kPiece;
    return reinterpret_cast<uintptr_t>(p) % piece == 0 && (s0 * static_cast<long long>(sizeof(T))) % static_cast<long long>(piece) == 0 &&
           (s1 * static_cast<long long>(sizeof(T))) % static_cast<long long>(piece) == 0 &&
           (s2 * static_cast<long long>(sizeof(T))) % static_cast<long long>(piece) == 0;
}

// Logistic function: 1 / (1 + exp(-v)).  exp(-v) overflows to infinity below
// v = -88.7, where the quotient is 0 as it should be.
__device__ __forceinline__ float sigmoidf(float v) { return rcpf(1.f + ex2f(-1.4426950408889634f * v)); }
// Derivative of v sigmoid(v).
__device__ __forceinline__ float dsilu(float v) {
    const float sg = sigmoidf(v);
    return sg * fmaf(v, 1.f - sg, 1.f);
}

// softplus(v) = log(1 + exp(v)) = max(v, 0) + log1p(e) with e = exp(-|v|), and
// its derivative, the logistic function, from the same e.
//   e      2^t with t = -|v| log2(e) rounded, times 1 + (what t lost) ln 2: the
//          rounding of t alone would cost |v| 2^-24 of every step size
//   log1p  2 atanh(s), s = e / (2 + e) in (0, 1/3], with atanh(s) = s P(s^2) and
//          P of degree 5 fitted at Chebyshev nodes (1e-10); no small difference
//          of near-equal numbers, so tiny step sizes keep their relative accuracy
__device__ __forceinline__ float softplusf(float v, float* deriv = nullptr) {
    float n;  // -|v|, not below -126 (where e is 0 anyway), so that an infinite v gives no inf - inf; NaN stays
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(n) : "f"(-fabsf(v)), "f"(-126.f));
    const float t = n * 1.44269502f;
    const float lost = fmaf(n, 1.92596303e-8f, fmaf(n, 1.44269502f, -t));
    float e = ex2f(t);
    e = fmaf(e, lost * 0.693147181f, e);
    const float s = e * rcpf(2.f + e), z = s * s;
    float q = fmaf(z, 0.122047015f, 0.106971338f);
    q = fmaf(z, q, 0.143103123f);
    q = fmaf(z, q, 0.199993476f);
    q = fmaf(z, q, 0.333333403f);
    q = fmaf(z, q, 1.f);
    if (deriv) *deriv = (v >= 0.f ? 1.f : e) * rcpf(1.f + e);
    return fmaf(2.f * s, q, fmaxf(v, 0.f));
}

// Packed float32 pairs: halves the instructions of multiplies and adds.
struct f2 {
    unsigned long long v;
};
__device__ __forceinline__ f2 pk(float a, float b) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void upk(f2 p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ f2 ex22(f2 a) {
    float x, y;
    upk(a, x, y);
    return pk(ex2f(x), ex2f(y));
}
__device__ __forceinline__ float sum2(f2 a) {
    float x, y;
    upk(a, x, y);
    return x + y;
}

// Sums K values over the lanes that differ in bits LO .. LO * LANES / 2 of the
// lane number.  While several values are left, each exchange halves them: a
// lane keeps one half and sends the other.  Afterwards v[0 .. kept) are this
// lane's sums of the values lane_slot(lane) + i.
template <int K, int LO, int LANES>
struct LaneSum {
    static constexpr int kept = K > LANES ? K / LANES : 1;
    __device__ static __forceinline__ void run(float (&v)[K], int lane) {
        int n = K;
#pragma unroll
        for (int m = LO; m < LO * LANES; m *= 2) {
            if (n > 1) {
                n /= 2;
                const bool up = lane & m;
#pragma unroll
                for (int i = 0; i < K / 2; ++i)
                    if (i < n) {
                        const float keep = up ? v[i + n] : v[i];
                        const float send = up ? v[i] : v[i + n];
                        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, m);
                    }
            } else {
                v[0] += __shfl_xor_sync(0xffffffffu, v[0], m);
            }
        }
    }
    // First value that this lane ends up with; lanes that differ only in bits
    // beyond the halvings hold the same.
    __device__ static __forceinline__ int slot(int lane) {
        int n = K, s = 0;
#pragma unroll
        for (int m = LO; m < LO * LANES; m *= 2)
            if (n > 1) {
                n /= 2;
                if (lane & m) s += n;
            }
        return s;
    }
    // One of the lanes that hold the same sums.
    __device__ static __forceinline__ bool owner(int lane) {
        int n = K;
        bool own = true;
#pragma unroll
        for (int m = LO; m < LO * LANES; m *= 2) {
            if (n > 1)
                n /= 2;
            else if (lane & m)
                own = false;
        }
        return own;
    }
};

// One halving exchange over lane bit m of values whose pairs (2k, 2k + 1) are
// stored swapped in the lanes with that bit set: every lane keeps the even
// registers and sends the odd ones, without selects.
template <int K>
__device__ __forceinline__ void pair_exchange(const float (&v)[K], float (&out)[K / 2], int m) {
#pragma unroll
    for (int k = 0; k < K / 2; ++k) out[k] = v[2 * k] + __shfl_xor_sync(0xffffffffu, v[2 * k + 1], m);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

// Sequence length of batch entry b, clamped to [0, n].
__device__ __forceinline__ int seq_len(const long long* lengths, int b, int n) {
    if (lengths == nullptr) return n;
    const long long l = lengths[b];
    return l < 0 ? 0 : (l > n ? n : static_cast<int>(l));
}

}  // namespace sdtw

// Activations of the feed-forward operators (gated_linear, linear_act) and
// the 8-bit checkpoint format, shared by the elementwise kernels (ffn.cu) and
// the products' epilogues.
//
// Each activation is a(z) = z * g(z) with a gate g in [0, 1], so its slope is
// g + z g': silu g = sigmoid(z); gelu g = Phi(z), the normal CDF; gelu_tanh
// g = sigmoid(2 u), u = sqrt(2/pi) (z + 0.044715 z^3), since
// (1 + tanh u) / 2 = sigmoid(2 u); relu g = [z > 0].
//
// 16-bit results use ex2.approx / rcp.approx (relative error about 2^-21) and
// the Phi of ew_common.cuh (absolute error 3e-7); tanh.approx is not used,
// its 2^-11 is the rounding step of f16.  fp32 results use the accurate
// library functions.
#pragma once

#include "ew_common.cuh"

namespace tpb {
namespace {

template <bool Fast>
__device__ __forceinline__ float sigmoid_of(float z) {
    if constexpr (Fast) return rcp_approx(1.0f + __expf(-z));
    else return 1.0f / (1.0f + expf(-z));
}

template <bool Fast>
__device__ __forceinline__ float phi_of(float z) {
    if constexpr (Fast) return phi_narrow(z);
    else return normcdff(z);
}

constexpr float kTanhBeta = 0.79788456080286535588f;  // sqrt(2 / pi)
constexpr float kTanhKappa = 0.044715f;

template <int ACT, bool Fast>
__device__ __forceinline__ float act_value(float z) {
    if constexpr (ACT == TPB_ACT_RELU) return (z > 0.0f || z != z) ? z : 0.0f;
    else if constexpr (ACT == TPB_ACT_GELU) return z * phi_of<Fast>(z);
    else if constexpr (ACT == TPB_ACT_GELU_TANH) {
        return z * sigmoid_of<Fast>(2.0f * kTanhBeta * fmaf(kTanhKappa * z * z, z, z));
    } else if constexpr (ACT == TPB_ACT_SILU) return z * sigmoid_of<Fast>(z);
    else return z;
}

// The activation and its slope from one evaluation of the gate.
template <int ACT, bool Fast>
__device__ __forceinline__ void act_slope(float z, float& a, float& d) {
    if constexpr (ACT == TPB_ACT_RELU) {
        a = (z > 0.0f || z != z) ? z : 0.0f;
        d = z <= 0.0f ? 0.0f : 1.0f;
    } else if constexpr (ACT == TPB_ACT_GELU) {
        const float g = phi_of<Fast>(z);
        const float e = Fast ? __expf(-0.5f * z * z) : expf(-0.5f * z * z);
        a = z * g;
        d = fmaf(z * 0.39894228040143267794f, e, g);  // phi(z) = exp(-z^2 / 2) / sqrt(2 pi)
    } else if constexpr (ACT == TPB_ACT_GELU_TANH) {
        const float z2 = z * z;
        const float g = sigmoid_of<Fast>(2.0f * kTanhBeta * fmaf(kTanhKappa * z2, z, z));
        a = z * g;
        d = fmaf(a * (1.0f - g), 2.0f * kTanhBeta * fmaf(3.0f * kTanhKappa, z2, 1.0f), g);
    } else if constexpr (ACT == TPB_ACT_SILU) {
        const float g = sigmoid_of<Fast>(z);
        a = z * g;
        d = fmaf(a, 1.0f - g, g);
    } else {
        a = z;
        d = 1.0f;
    }
}

// z[j] <- act(z[j]); the switch is uniform over the grid and sits outside the
// unrolled loop.
template <bool Fast, int V>
__device__ __forceinline__ void act_values(int act, float (&z)[V]) {
    switch (act) {
#define TPB_ACT_CASE(A)                                            \
    case A:                                                        \
        _Pragma("unroll") for (int j = 0; j < V; ++j) z[j] = act_value<A, Fast>(z[j]); \
        break;
        TPB_ACT_CASE(TPB_ACT_RELU)
        TPB_ACT_CASE(TPB_ACT_GELU)
        TPB_ACT_CASE(TPB_ACT_GELU_TANH)
        TPB_ACT_CASE(TPB_ACT_SILU)
#undef TPB_ACT_CASE
        default: break;
    }
}

template <bool Fast, int V>
__device__ __forceinline__ void act_slopes(int act, const float (&z)[V], float (&a)[V], float (&d)[V]) {
    switch (act) {
#define TPB_ACT_CASE(A)                                            \
    case A:                                                        \
        _Pragma("unroll") for (int j = 0; j < V; ++j) act_slope<A, Fast>(z[j], a[j], d[j]); \
        break;
        TPB_ACT_CASE(TPB_ACT_RELU)
        TPB_ACT_CASE(TPB_ACT_GELU)
        TPB_ACT_CASE(TPB_ACT_GELU_TANH)
        TPB_ACT_CASE(TPB_ACT_SILU)
#undef TPB_ACT_CASE
        default: {
#pragma unroll
            for (int j = 0; j < V; ++j) act_slope<TPB_ACT_NONE, Fast>(z[j], a[j], d[j]);
        }
    }
}

// ------------------------------------------------------- 8-bit checkpoints --
//
// A block of kCkptBlock consecutive elements of a row is held as int8 values
// q and one power of two 2^e: q = round-to-nearest-even(x 2^-e), the least e
// with max|x| <= 127 * 2^e.  Multiplying by a power of two is exact, so the
// only rounding is the one to 8 bits: |x - q 2^e| <= 2^(e-1).  e is stored as
// e + 127 in a byte (1 .. 249); 255 marks a block that holds an infinity or a
// NaN, which reads back as NaN.  A block whose largest magnitude lies in the
// top half step of the storage type's last binade rounds down to 63 * 2^e
// there (64 * 2^e would overflow the type).
constexpr int kCkptBlock = 32;
constexpr int kCkptNonFinite = 255;
constexpr int kCkptMinExp = 1;  // e = -126: 2^-e and 2^e are normal floats

// The stored exponent of a block from its largest magnitude, and the largest
// |q| the block may hold.  kEmax: exponent of the storage type's last binade.
template <typename T> struct LastBinade { static constexpr int value = 127; };
template <> struct LastBinade<__half> { static constexpr int value = 15; };

template <typename T>
__device__ __forceinline__ int ckpt_exponent(float amax, float& qmax) {
    const uint32_t u = __float_as_uint(amax);  // amax >= 0, or NaN
    const int be = int(u >> 23);               // biased exponent E + 127
    if (be == 255) {
        qmax = 0.0f;
        return kCkptNonFinite;
    }
    // amax = m 2^E, 1 <= m < 2: amax / 2^(E-6) = 64 m <= 127 iff m <= 1 + 63/64.
    const int coarse = (u & 0x7fffffu) > 0x7e0000u ? 1 : 0;
    qmax = (coarse != 0 && be == LastBinade<T>::value + 127) ? 63.0f : 127.0f;
    return max(be - 6 + coarse, kCkptMinExp);
}

// 2^-e and 2^e of a stored exponent (not kCkptNonFinite).
__device__ __forceinline__ float ckpt_inverse(int stored) { return __uint_as_float(uint32_t(254 - stored) << 23); }
__device__ __forceinline__ float ckpt_step(int stored) {
    return stored == kCkptNonFinite ? __int_as_float(0x7fffffff) : __uint_as_float(uint32_t(stored) << 23);
}
__device__ __forceinline__ int8_t ckpt_quantise(float x, float inverse, float qmax) {
    return static_cast<int8_t>(__float2int_rn(fminf(fmaxf(x * inverse, -qmax), qmax)));
}

}  // namespace
}  // namespace tpb

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
// the Phi of ew_common.cuh (absolute error 3e-7), as the elementwise gelu does;
// tanh.approx is not used, its 2^-11 is the rounding step of f16.  Phi's error
// stays within half a step of gelu's result down to z = -3.2 in f16 and -3.8 in
// bf16; further out the result may be off by |z| 3e-7, more than its own fine
// steps there (-4.6: 1.4e-6 of 9.7e-6).  fp32 results use the accurate library
// functions.
#pragma once

#include "ew_common.cuh"

namespace tpb {
namespace {

constexpr float kTanhBeta = 0.79788456080286535588f;  // sqrt(2 / pi)
constexpr float kTanhKappa = 0.044715f;

// ---- fp32 results: accurate functions, one element at a time --------------

__device__ __forceinline__ float sigmoid_of(float z) { return 1.0f / (1.0f + expf(-z)); }

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
    if constexpr (ACT == TPB_ACT_RELU) return (z > 0.0f || z != z) ? z : 0.0f;
    else if constexpr (ACT == TPB_ACT_GELU) return z * normcdff(z);
    else if constexpr (ACT == TPB_ACT_GELU_TANH) {
        return z * sigmoid_of(2.0f * kTanhBeta * fmaf(kTanhKappa * z * z, z, z));
    } else if constexpr (ACT == TPB_ACT_SILU) return z * sigmoid_of(z);
    else return z;
}

// The activation and its slope from one evaluation of the gate.
template <int ACT>
__device__ __forceinline__ void act_slope(float z, float& a, float& d) {
    if constexpr (ACT == TPB_ACT_RELU) {
        a = (z > 0.0f || z != z) ? z : 0.0f;
        d = z <= 0.0f ? 0.0f : 1.0f;
    } else if constexpr (ACT == TPB_ACT_GELU) {
        const float g = normcdff(z);
        a = z * g;
        d = fmaf(z * 0.39894228040143267794f, expf(-0.5f * z * z), g);  // phi(z) = exp(-z^2 / 2) / sqrt(2 pi)
    } else if constexpr (ACT == TPB_ACT_GELU_TANH) {
        const float z2 = z * z;
        const float g = sigmoid_of(2.0f * kTanhBeta * fmaf(kTanhKappa * z2, z, z));
        a = z * g;
        d = fmaf(a * (1.0f - g), 2.0f * kTanhBeta * fmaf(3.0f * kTanhKappa, z2, 1.0f), g);
    } else if constexpr (ACT == TPB_ACT_SILU) {
        const float g = sigmoid_of(z);
        a = z * g;
        d = fmaf(a, 1.0f - g, g);
    } else {
        a = z;
        d = 1.0f;
    }
}

// ---- 16-bit results: two lanes at a time ------------------------------------
//
// The packed two-lane instructions halve the arithmetic, which otherwise costs
// more than the memory traffic of these passes (gelu's slope: 222 us over
// 8192 x 16384 bf16 from 8 bits, against 103 us for the bytes).

// a <- a * b and a <- a + b.
template <int V>
__device__ __forceinline__ void mul_to(float (&a)[V], const float (&b)[V]) {
#pragma unroll
    for (int j = 0; j + 1 < V; j += 2) {
        const float2 r = __fmul2_rn(make_float2(a[j], a[j + 1]), make_float2(b[j], b[j + 1]));
        a[j] = r.x;
        a[j + 1] = r.y;
    }
    if constexpr (V % 2) a[V - 1] *= b[V - 1];
}
template <int V>
__device__ __forceinline__ void add_to(float (&a)[V], const float (&b)[V]) {
#pragma unroll
    for (int j = 0; j + 1 < V; j += 2) {
        const float2 r = __fadd2_rn(make_float2(a[j], a[j + 1]), make_float2(b[j], b[j + 1]));
        a[j] = r.x;
        a[j + 1] = r.y;
    }
    if constexpr (V % 2) a[V - 1] += b[V - 1];
}

// 1 / (1 + 2^t): exp2 overflowing to infinity gives 0.
__device__ __forceinline__ float2 gate_of_exp2(float2 t) {
    float2 e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
    e = __fadd2_rn(e, f2(1.0f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(e.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(e.y));
    return r;
}

constexpr float kLog2E = 1.44269504088896340736f;

template <int ACT>
__device__ __forceinline__ float2 gate2(float2 z, float2 z2) {
    if constexpr (ACT == TPB_ACT_GELU) {
        return phi_narrow2(z);
    } else if constexpr (ACT == TPB_ACT_GELU_TANH) {
        // sigmoid(2 u) = 1 / (1 + 2^(-2 log2(e) u)), u = beta (z + kappa z^3)
        const float2 c = __ffma2_rn(z2, f2(-2.0f * kLog2E * kTanhBeta * kTanhKappa), f2(-2.0f * kLog2E * kTanhBeta));
        return gate_of_exp2(__fmul2_rn(z, c));
    } else {
        return gate_of_exp2(__fmul2_rn(z, f2(-kLog2E)));
    }
}

template <int ACT>
__device__ __forceinline__ float2 act_value2(float2 z) {
    if constexpr (ACT == TPB_ACT_NONE || ACT == TPB_ACT_RELU) {
        return make_float2(act_value<ACT>(z.x), act_value<ACT>(z.y));
    } else {
        return __fmul2_rn(z, gate2<ACT>(z, __fmul2_rn(z, z)));
    }
}

template <int ACT>
__device__ __forceinline__ void act_slope2(float2 z, float2& a, float2& d) {
    if constexpr (ACT == TPB_ACT_NONE || ACT == TPB_ACT_RELU) {
        act_slope<ACT>(z.x, a.x, d.x);
        act_slope<ACT>(z.y, a.y, d.y);
    } else {
        const float2 z2 = __fmul2_rn(z, z);
        const float2 g = gate2<ACT>(z, z2);
        a = __fmul2_rn(z, g);
        if constexpr (ACT == TPB_ACT_GELU) {
            const float2 t = __fmul2_rn(z2, f2(-0.5f * kLog2E));
            float2 e;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
            d = __ffma2_rn(__fmul2_rn(z, f2(0.39894228040143267794f)), e, g);
        } else {
            const float2 h = __ffma2_rn(g, f2(-1.0f), f2(1.0f));  // 1 - g
            float2 slope = __fmul2_rn(a, h);
            if constexpr (ACT == TPB_ACT_GELU_TANH) {
                slope = __fmul2_rn(slope, __ffma2_rn(z2, f2(6.0f * kTanhBeta * kTanhKappa), f2(2.0f * kTanhBeta)));
            }
            d = __fadd2_rn(slope, g);
        }
    }
}

// z[j] <- act(z[j]), and act and its slope; the switch is uniform over the
// grid and sits outside the unrolled loops.
template <int ACT, bool Fast, int V>
__device__ __forceinline__ void act_values_of(float (&z)[V]) {
    if constexpr (Fast && V % 2 == 0) {
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            const float2 r = act_value2<ACT>(make_float2(z[j], z[j + 1]));
            z[j] = r.x;
            z[j + 1] = r.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] = act_value<ACT>(z[j]);
    }
}

template <int ACT, bool Fast, int V>
__device__ __forceinline__ void act_slopes_of(const float (&z)[V], float (&a)[V], float (&d)[V]) {
    if constexpr (Fast && V % 2 == 0) {
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            float2 va, vd;
            act_slope2<ACT>(make_float2(z[j], z[j + 1]), va, vd);
            a[j] = va.x;
            a[j + 1] = va.y;
            d[j] = vd.x;
            d[j + 1] = vd.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) act_slope<ACT>(z[j], a[j], d[j]);
    }
}

template <bool Fast, int V>
__device__ __forceinline__ void act_values(int act, float (&z)[V]) {
    switch (act) {
        case TPB_ACT_RELU: act_values_of<TPB_ACT_RELU, Fast, V>(z); break;
        case TPB_ACT_GELU: act_values_of<TPB_ACT_GELU, Fast, V>(z); break;
        case TPB_ACT_GELU_TANH: act_values_of<TPB_ACT_GELU_TANH, Fast, V>(z); break;
        case TPB_ACT_SILU: act_values_of<TPB_ACT_SILU, Fast, V>(z); break;
        default: break;
    }
}

template <bool Fast, int V>
__device__ __forceinline__ void act_slopes(int act, const float (&z)[V], float (&a)[V], float (&d)[V]) {
    switch (act) {
        case TPB_ACT_RELU: act_slopes_of<TPB_ACT_RELU, Fast, V>(z, a, d); break;
        case TPB_ACT_GELU: act_slopes_of<TPB_ACT_GELU, Fast, V>(z, a, d); break;
        case TPB_ACT_GELU_TANH: act_slopes_of<TPB_ACT_GELU_TANH, Fast, V>(z, a, d); break;
        case TPB_ACT_SILU: act_slopes_of<TPB_ACT_SILU, Fast, V>(z, a, d); break;
        default: act_slopes_of<TPB_ACT_NONE, Fast, V>(z, a, d);
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

// V values (1, 2, or a multiple of 4) of a block as int8.  Adding 1.5 * 2^23
// rounds to the nearest integer, ties to even, and leaves it in the low byte
// of the sum's bits: a full-rate addition instead of a conversion.  stored:
// the block's exponent; qmax below 127 clamps (see ckpt_exponent).
template <int V>
__device__ __forceinline__ Vec<int8_t, V> ckpt_quantise(const float (&x)[V], int stored, float qmax) {
    const float inverse = stored == kCkptNonFinite ? 0.0f : ckpt_inverse(stored);
    float q[V], scale[V], round[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        q[j] = x[j];
        scale[j] = inverse;
        round[j] = 12582912.0f;
    }
    mul_to<V>(q, scale);
    if (qmax < 127.0f) {  // a block in the type's last binade, or one that is not finite (NaN becomes 0)
#pragma unroll
        for (int j = 0; j < V; ++j) q[j] = fminf(fmaxf(q[j], -qmax), qmax);
    }
    add_to<V>(q, round);
    uint32_t bits[V];
#pragma unroll
    for (int j = 0; j < V; ++j) bits[j] = __float_as_uint(q[j]);
    Vec<int8_t, V> out;
    if constexpr (V % 4 == 0) {
        uint32_t* o = reinterpret_cast<uint32_t*>(&out);
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            o[j / 4] = __byte_perm(__byte_perm(bits[j], bits[j + 1], 0x0040), __byte_perm(bits[j + 2], bits[j + 3], 0x0040),
                                   0x5410);
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) out.v[j] = static_cast<int8_t>(bits[j] & 0xffu);
    }
    return out;
}

// The values a checkpoint's bytes stand for.  A byte b with its sign bit
// flipped is b + 128; under the exponent of 2^23 it reads 2^23 + 128 + b, from
// which the offset is subtracted exactly: no conversion instruction.
template <int V>
__device__ __forceinline__ void ckpt_values(const Vec<int8_t, V>& q, int stored, float (&x)[V]) {
    const float step = ckpt_step(stored);
    if constexpr (V % 4 == 0) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&q);
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            const uint32_t u = w[j / 4] ^ 0x80808080u;
#pragma unroll
            for (int b = 0; b < 4; b += 2) {
                const float2 v = make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540 + b)),
                                             __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7541 + b)));
                const float2 r = __fmul2_rn(__fadd2_rn(v, f2(-8388736.0f)), f2(step));
                x[j + b] = r.x;
                x[j + b + 1] = r.y;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = float(q.v[j]) * step;
    }
}

}  // namespace
}  // namespace tpb

// What the feed-forward kernels share: element types, vector loads and stores
// of any alignment, the activations with their slopes, and the epilogue of a
// product.  Private to libbvml_ffn.so.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "bvml_ffn.h"

namespace bvml_ffn {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

// Element types, as the C ABI numbers them.
constexpr int kF32 = BVML_FFN_F32, kF16 = BVML_FFN_F16, kBF16 = BVML_FFN_BF16,
              kE4M3 = BVML_FFN_E4M3;

// ---------------------------------------------------------------------------
// conversions: sums and statistics are fp32; every rounding to 16 bits goes
// to nearest even, once, where a result is stored
// ---------------------------------------------------------------------------
__device__ __forceinline__ float from16(uint16_t bits, int type) {
    return type == kBF16 ? __builtin_bit_cast(float, (uint32_t)bits << 16)
                         : (float)__builtin_bit_cast(_Float16, bits);
}
__device__ __forceinline__ uint16_t to16(float v, int type) {
    return type == kBF16 ? __builtin_bit_cast(uint16_t, (__bf16)v)
                         : __builtin_bit_cast(uint16_t, (_Float16)v);
}

// A ragged end's own copy of a pointer: without it the compiler shares single
// values between the two branches below and takes the whole vector apart.
template <typename T>
__device__ __forceinline__ T* apart(T* p) {
    asm("" : "+v"(p));
    return p;
}

// V consecutive values at element `at` of a 16- or 32-bit array, the first n
// of them inside it (the others read as 0).  Whole vectors are loads of up to
// 16 bytes at any alignment (the hardware takes unaligned global accesses);
// only a row's ragged end goes value by value.
template <int V>
__device__ __forceinline__ void load_row(const void* base, int type, long long at, int n,
                                         float (&v)[V]) {
    if (type == kF32) {
        const float* p = static_cast<const float*>(base) + at;
        if (n >= V) {
            __builtin_memcpy(v, p, 4 * V);
        } else {
            p = apart(p);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = i < n ? p[i] : 0.0f;
        }
        return;
    }
    const uint16_t* p = static_cast<const uint16_t*>(base) + at;
    uint16_t h[V];
    if (n >= V) {
        __builtin_memcpy(h, p, 2 * V);
    } else {
        p = apart(p);
#pragma unroll
        for (int i = 0; i < V; ++i) h[i] = i < n ? p[i] : (uint16_t)0;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = from16(h[i], type);
}

template <int V>
__device__ __forceinline__ void store_row(void* base, int type, long long at, int n,
                                          const float (&v)[V]) {
    if (type == kF32) {
        float* p = static_cast<float*>(base) + at;
        if (n >= V) {
            __builtin_memcpy(p, v, 4 * V);
        } else {
            p = apart(p);
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < n) p[i] = v[i];
        }
        return;
    }
    uint16_t h[V];
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = to16(v[i], type);
    uint16_t* p = static_cast<uint16_t*>(base) + at;
    if (n >= V) {
        __builtin_memcpy(p, h, 2 * V);
    } else {
        p = apart(p);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) p[i] = h[i];
    }
}

// ---------------------------------------------------------------------------
// activations, in fp32 on the hardware's 2^x and reciprocal (about 1 ulp each)
// ---------------------------------------------------------------------------
constexpr float kLog2e = 1.4426950408889634f;

// 1 / (1 + 2^t)
__device__ __forceinline__ float logistic2(float t) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(t));
}
__device__ __forceinline__ float sigmoid_fast(float x) { return logistic2(-kLog2e * x); }

// The normal distribution's Phi(x), with e = exp(-x^2 / 2): the tail beyond |x|
// is e p(t), t = 1 / (1 + 0.3025 |x|), with p a polynomial without a constant
// fitted to Phi(-|x|) / e over |x| <= 13.6 (where e ends) for the least largest
// relative error: 1.0e-7, 3.8e-7 with fp32's own roundings.  So the tail keeps its
// relative accuracy, which a bound on the absolute error would not give it.
__device__ __forceinline__ float normal_cdf(float x, float e) {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3025f, __builtin_fabsf(x), 1.0f));
    constexpr float kP[] = {0.12063242f, 0.12164301f,   0.10146175f, 0.12550873f,
                            -0.047244925f, 0.19775172f, -0.15621658f, 0.036463842f};
    float p = kP[7];
#pragma unroll
    for (int i = 6; i >= 0; --i) p = __builtin_fmaf(p, t, kP[i]);
    const float tail = p * t * e;
    return x < 0.0f ? tail : 1.0f - tail;
}
__device__ __forceinline__ float normal_bell(float x) {  // exp(-x^2 / 2)
    return __builtin_amdgcn_exp2f((-0.5f * kLog2e) * x * x);
}

// 0.5 (1 + tanh(a)) = 1 / (1 + exp(-2 a)), a = sqrt(2 / pi) (x + 0.044715 x^3)
constexpr float kTanhA = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kTanhB = 0.044715f;
__device__ __forceinline__ float tanh_gate(float x, float x2) {
    return logistic2(x * __builtin_fmaf(x2, -kLog2e * kTanhA * kTanhB, -kLog2e * kTanhA));
}

__device__ __forceinline__ float act1(int act, float x) {
    switch (act) {
        case BVML_FFN_RELU: return x < 0.0f ? 0.0f : x;
        case BVML_FFN_GELU: return x * normal_cdf(x, normal_bell(x));
        case BVML_FFN_GELU_TANH: return x * tanh_gate(x, x * x);
        case BVML_FFN_SILU: return x * sigmoid_fast(x);
        default: return x;
    }
}

// The activation and its derivative.
__device__ __forceinline__ void act_slope1(int act, float x, float& value, float& slope) {
    switch (act) {
        case BVML_FFN_RELU:
            value = x < 0.0f ? 0.0f : x;
            slope = x > 0.0f ? 1.0f : 0.0f;
            return;
        case BVML_FFN_GELU: {
            const float e = normal_bell(x);
            const float c = normal_cdf(x, e);
            value = x * c;
            slope = __builtin_fmaf(x * e, 0.3989422804014327f, c);
            return;
        }
        case BVML_FFN_GELU_TANH: {
            // (s is 0 or 1 long before x^2 could pass the largest number, and
            // 0 times that would be no number: the square stays below)
            const float x2 = __builtin_fminf(x * x, 1e30f), s = tanh_gate(x, x2);
            value = x * s;
            slope = __builtin_fmaf(value * (1.0f - s),
                                   __builtin_fmaf(x2, 3.0f * kTanhA * kTanhB, kTanhA), s);
            return;
        }
        case BVML_FFN_SILU: {
            const float s = sigmoid_fast(x);
            value = x * s;
            slope = __builtin_fmaf(value, 1.0f - s, s);
            return;
        }
        default:
            value = x;
            slope = 1.0f;
    }
}

// `act` is the same for the whole launch: one scalar branch per vector.
#define BVML_FFN_ACTS(CASE) \
    CASE(BVML_FFN_RELU) CASE(BVML_FFN_GELU) CASE(BVML_FFN_GELU_TANH) CASE(BVML_FFN_SILU)

template <int V>
__device__ __forceinline__ void activate(int act, float (&v)[V]) {
    switch (act) {
#define BVML_FFN_CASE(A)                                                    \
    case A:                                                                 \
        _Pragma("unroll") for (int i = 0; i < V; ++i) v[i] = act1(A, v[i]); \
        break;
        BVML_FFN_ACTS(BVML_FFN_CASE)
#undef BVML_FFN_CASE
        default: break;
    }
}

template <int V>
__device__ __forceinline__ void act_slope(int act, const float (&x)[V], float (&value)[V],
                                          float (&slope)[V]) {
    switch (act) {
#define BVML_FFN_CASE(A)                                                                       \
    case A:                                                                                    \
        _Pragma("unroll") for (int i = 0; i < V; ++i) act_slope1(A, x[i], value[i], slope[i]); \
        break;
        BVML_FFN_ACTS(BVML_FFN_CASE)
#undef BVML_FFN_CASE
        default:
#pragma unroll
            for (int i = 0; i < V; ++i) act_slope1(BVML_FFN_NONE, x[i], value[i], slope[i]);
    }
}

// ---------------------------------------------------------------------------
// a product's epilogue
// ---------------------------------------------------------------------------
struct Epilogue {
    const void* bias;       // (R) of bias_type, or null
    const float* x_scale;   // (M) with w_scale (R), or null
    const float* w_scale;
    const void* residual;   // (M, N) of out_type, or null
    void* y;                // (M, N) of out_type
    void* z;                // (M, R) of z_type: the pre-activations, or null
    float* part;            // (splits, M, R) partial sums, or null
    long long ldr, ldy, ldz;
    int M, N;               // N: y's columns; R = N, or 2N for the gated form
    int bias_type, out_type, z_type, act;
};

// What a column adds, kept by the lane that finishes it.
template <int V>
struct Column {
    float bias[V], scale[V];
    // columns col .. col + V, the first c of them inside
    __device__ __forceinline__ void load(const Epilogue& e, int col, int c) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            bias[i] = 0.0f;
            scale[i] = 1.0f;
        }
        if (c <= 0) return;
        if (e.bias) load_row<V>(e.bias, e.bias_type, col, c, bias);
        if (e.w_scale) load_row<V>(e.w_scale, kF32, col, c, scale);
    }
    // kScaled false: 16-bit operands, which have no scales
    template <bool kScaled>
    __device__ __forceinline__ void apply(float row_scale, float (&v)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i)
            v[i] = kScaled ? __builtin_fmaf(v[i], row_scale * scale[i], bias[i]) : v[i] + bias[i];
    }
};

// V neighbouring sums of row m from column n on, c of them inside; r: the
// residual's values there (if any).  T: the 16-bit type, known to the kernel
// where its operands are of it.
template <int V>
__device__ __forceinline__ void finish(const Epilogue& e, const Column<V>& k, int type16, int m,
                                       int n, int c, float (&v)[V], const float (&r)[V]) {
    k.template apply<true>(e.x_scale ? e.x_scale[m] : 1.0f, v);
    if (e.z) store_row<V>(e.z, type16, (long long)m * e.ldz + n, c, v);
    activate<V>(e.act, v);
    if (e.residual) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] += r[i];
    }
    store_row<V>(e.y, e.out_type == kF32 ? kF32 : type16, (long long)m * e.ldy + n, c, v);
}

// act(gate) * up.
template <int V>
__device__ __forceinline__ void finish_gated(const Epilogue& e, const Column<V>& kg,
                                             const Column<V>& ku, int type16, int m, int n, int c,
                                             float (&g)[V], float (&u)[V]) {
    const float s = e.x_scale ? e.x_scale[m] : 1.0f;
    kg.template apply<true>(s, g);
    ku.template apply<true>(s, u);
    if (e.z) {
        store_row<V>(e.z, type16, (long long)m * e.ldz + n, c, g);
        store_row<V>(e.z, type16, (long long)m * e.ldz + e.N + n, c, u);
    }
    activate<V>(e.act, g);
#pragma unroll
    for (int i = 0; i < V; ++i) g[i] *= u[i];
    store_row<V>(e.y, e.out_type == kF32 ? kF32 : type16, (long long)m * e.ldy + n, c, g);
}

// One vector by itself, for the kernels that finish few: what it adds, asked
// for before the sums are there, then the rest.
template <int V, bool kGated>
struct Single {
    Column<V> k, ku;
    float r[V];
    __device__ __forceinline__ void load(const Epilogue& e, int type16, int m, int n) {
        const int c = e.N - n;
        if (m >= e.M || c <= 0) return;
        k.load(e, n, c);
        if constexpr (kGated) ku.load(e, e.N + n, c);
        if (!kGated && e.residual)
            load_row<V>(e.residual, e.out_type == kF32 ? kF32 : type16,
                        (long long)m * e.ldr + n, c, r);
    }
    // v: the sums (gated: the gate's), u: the other half's
    __device__ __forceinline__ void finish(const Epilogue& e, int type16, int m, int n,
                                           float (&v)[V], float (&u)[V]) const {
        const int c = e.N - n;
        if (m >= e.M || c <= 0) return;
        if constexpr (kGated)
            finish_gated<V>(e, k, ku, type16, m, n, c, v, u);
        else
            bvml_ffn::finish<V>(e, k, type16, m, n, c, v, r);
    }
};

// The 16-bit type of a call: its operands' or, from 8 bits, its output's.
__device__ __forceinline__ int type16_of(int in_type, const Epilogue& e) {
    return in_type == kE4M3 ? e.out_type : in_type;
}

}  // namespace bvml_ffn

// Shared by the kernels that say how likely tokens are: a row's running statistics, keys that order alternatives, activations.
#pragma once
#include "common.cuh"

namespace ib {
namespace score {

constexpr int MAX_TOP = 20;              // most alternatives of a row
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_fast(float x) {        // 2^-inf = 0, about 2 ulp
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What a product's sum z is as a logit. A masked one, -inf (also what stands for places outside the vocabulary), stays masked under a cap.
__device__ __forceinline__ float logit(float z, float scale, float cap) {
    const float l = z * scale;
    return cap > 0.0f && l != -INFINITY ? cap * tanhf(l / cap) : l;
}

// m = max l, s = sum exp(l - m), d = sum exp(l - m) (l - m) of the elements seen. Only the differences l - m are ever scaled or exponentiated,
// so that logprob keeps its digits where one token has nearly all of the probability.
struct Stats {
    float m, s, d;
    __device__ __forceinline__ void clear() { m = -INFINITY; s = 0.0f; d = 0.0f; }
    __device__ __forceinline__ void raise(float to) {        // to >= m, or m is NaN's neighbour: s says so already
        const float x = m - to, f = s != 0.0f ? exp2_fast(x * LOG2E) : 0.0f;
        d = f > 0.0f ? f * fmaf(x, s, d) : (f == 0.0f ? 0.0f : f);
        s *= f;
        m = to;
    }
    template <int N> __device__ __forceinline__ void add(const float (&l)[N]) {
        float top = l[0];
#pragma unroll
        for (int i = 1; i < N; i++) top = fmaxf(top, l[i]);
        if (top > m) raise(top);
        const float ref = m == -INFINITY ? 0.0f : m;
        float s0 = 0.0f, s1 = 0.0f, d0 = 0.0f, d1 = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float x = l[i] - ref, e = exp2_fast(x * LOG2E);
            // (an element of -inf: e = 0, and 0 * -1000 adds nothing; a NaN goes into s, which is enough)
            if (i & 1) { s1 += e; d1 = fmaf(e, fmaxf(x, -1000.0f), d1); } else { s0 += e; d0 = fmaf(e, fmaxf(x, -1000.0f), d0); }
        }
        s += s0 + s1;
        d += d0 + d1;
    }
    __device__ __forceinline__ void join(Stats o) {
        if (o.m > m) raise(o.m); else if (m > o.m) o.raise(m);
        s += o.s;
        d += o.d;
    }
    __device__ __forceinline__ float logprob(float l) const {
        return m == -INFINITY && s == 0.0f ? -INFINITY : (l - m) - logf(s);
    }
    __device__ __forceinline__ float entropy() const { return m == -INFINITY && s == 0.0f ? 0.0f : logf(s) - d / s; }
};

__device__ __forceinline__ Stats warp_join(Stats v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Stats w;
        w.m = __shfl_xor_sync(0xffffffffu, v.m, o);
        w.s = __shfl_xor_sync(0xffffffffu, v.s, o);
        w.d = __shfl_xor_sync(0xffffffffu, v.d, o);
        v.join(w);
    }
    return v;
}

__device__ __forceinline__ void finish(const Stats& st, int token, float at, int64_t vocab, float* logprob, float* entropy, int* status) {
    if (entropy) *entropy = st.entropy();
    if (!logprob) return;
    const bool none = token == -1, outside = !none && (token < 0 || token >= vocab);
    if (outside && status) atomicExch(status, 1);
    *logprob = none ? 0.0f : outside ? __int_as_float(0x7fc00000) : st.logprob(at);
}

// A key orders alternatives: a larger logit first, among equal ones a lower id (-0 is 0). Every key of an element is above 0.
__device__ __forceinline__ unsigned long long key(float z, uint32_t id) {
    const uint32_t bits = __float_as_uint(z + 0.0f), ord = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
    return (static_cast<unsigned long long>(ord) << 32) | (0xffffffffu - id);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
    const uint32_t ord = uint32_t(k >> 32);
    return __uint_as_float(ord & 0x80000000u ? ord & 0x7fffffffu : ~ord);
}
__device__ __forceinline__ uint32_t key_id(unsigned long long k) { return 0xffffffffu - uint32_t(k); }

// ------------------------------------------------------------------------------------------------ activations
constexpr int ACTIVATIONS = 6;
enum { NONE = 0, RELU = 1, RELU_SQUARED = 2, GELU_TANH = 3, GELU = 4, SILU = 5 };

// x sigmoid(y) without an IEEE division: for y below about -88 the exponential is infinite and the quotient 0.
__device__ __forceinline__ float times_sigmoid(float x, float y) { return __fdividef(x, 1.0f + exp2_fast(-LOG2E * y)); }

__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case RELU: return z > 0.0f ? z : (z != z ? z : 0.0f);
        case RELU_SQUARED: { const float r = z > 0.0f ? z : (z != z ? z : 0.0f); return r * r; }
        // 0.5 z (1 + tanh u) = z sigmoid(2 u), u = sqrt(2/pi) (z + 0.044715 z^3)
        case GELU_TANH: return times_sigmoid(z, 1.5957691216057308f * fmaf(0.044715f * z * z, z, z));
        case GELU: return 0.5f * z * erfcf(-0.70710678118654752f * z);
        case SILU: return times_sigmoid(z, z);
    }
    return z;
}

}  // namespace score
}  // namespace ib

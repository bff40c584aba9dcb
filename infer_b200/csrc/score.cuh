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

template <int N> __device__ __forceinline__ float largest_of(const float (&z)[N]) {
    float top = z[0];
#pragma unroll
    for (int i = 1; i < N; i++) top = fmaxf(top, z[i]);
    return top;
}

// The logit of a product's sum z under a cap, cap tanh(u) with u = z scale / cap: a value of z is the same logit wherever it is evaluated, in the sums, as the asked
// token or as an alternative, so that a token with nearly all the probability keeps its digits and is never likelier than 1. (No product here may be
// contracted into a sum that follows: __fmul_rn.)
// From |u| = 0.6 on tanh u = 1 - 2 / (1 + e^2u): beyond atanh(1/2) = 0.55 what is subtracted is below 1/2, so no digits cancel (5 x 2^-24 of the result).
// Below, an odd polynomial, a minimax fit of tanh(u) / u in u^2 made for this place, of the degree at which its error over [0, 0.6], 4.9e-9 with the
// constants as they are stored, is below its roundings (2 x 2^-24 with them).
constexpr float TANH_SPLIT = 0.6f;
__device__ __forceinline__ float tanh_below(float u) {
    const float q = u * u;
    float t = fmaf(q, -0.005852164700627327f, 0.02075362578034401f);
    t = fmaf(q, t, -0.05376870185136795f);
    t = fmaf(q, t, 0.13331688940525055f);
    t = fmaf(q, t, -0.3333328366279602f);
    t = fmaf(q, t, 1.0f);
    return __fmul_rn(u, t);
}
__device__ __forceinline__ float tanh_above(float u) {
    return copysignf(1.0f - __fdividef(2.0f, 1.0f + exp2_fast(__fmul_rn(fabsf(u), 2.0f * LOG2E))), u);
}
// (Both forms, then a choice: as two sides of a condition they became a branch for each element, 647 us at 512 rows x 1536 against 152,064 under a cap of 10; so 359.)
__device__ __forceinline__ float cap_tanh(float u, float cap) {
    const float below = tanh_below(u), above = tanh_above(u);
    return __fmul_rn(cap, fabsf(u) <= TANH_SPLIT ? below : above);
}
// A masked sum, -inf (also what stands for places outside the vocabulary), stays masked; a finite one never is, whatever its product with scale / cap. +inf: the cap.
__device__ __forceinline__ float cap_logit(float z, float scale, float cap) {
    const float l = cap_tanh(__fmul_rn(z, scale / cap), cap);
    return z == -INFINITY ? z : l;
}
// N of them (`counts`: whether the thread's results are needed). Where a thread's are all below the split, as a model's are, the second form is left out.
template <int N> __device__ __forceinline__ void cap_logits(float (&l)[N], const float (&z)[N], float scale, float cap, bool counts = true) {
    const float to_u = scale / cap;
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) { l[i] = __fmul_rn(z[i], to_u); most = fmaxf(most, z[i] == -INFINITY ? 0.0f : fabsf(l[i])); }
    if (most <= TANH_SPLIT || !counts) {
#pragma unroll
        for (int i = 0; i < N; i++) { const float t = __fmul_rn(cap, tanh_below(l[i])); l[i] = z[i] == -INFINITY ? z[i] : t; }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) { const float t = cap_tanh(l[i], cap); l[i] = z[i] == -INFINITY ? z[i] : t; }
    }
}

// m = max l, s = sum exp(l - m), d = sum exp(l - m) (l - m) of the elements seen. Only the differences l - m are ever exponentiated, so that
// logprob keeps its digits where one token has nearly all of the probability.
struct Stats {
    float m, s, d;
    __device__ __forceinline__ void clear() { m = -INFINITY; s = 0.0f; d = 0.0f; }
    __device__ __forceinline__ void raise(float to) {        // to >= m
        const float x = m - to, f = s != 0.0f ? exp2_fast(x * LOG2E) : 0.0f;
        d = f > 0.0f ? f * fmaf(x, s, d) : (f == 0.0f ? 0.0f : f);
        s *= f;
        m = to;
    }
    // Adds the logits z scale; `top`: the largest z (a NaN left out).
    template <int N> __device__ __forceinline__ void add(const float (&z)[N], float top, float scale = 1.0f) {
        if (top * scale > m) raise(top * scale);
        const float ref = m == -INFINITY ? 0.0f : m;
        float s0 = 0.0f, s1 = 0.0f, d0 = 0.0f, d1 = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float x = fmaf(z[i], scale, -ref), e = exp2_fast(x * LOG2E);
            // (an element of -inf: e = 0, and 0 * -1000 adds nothing; a NaN goes into s, which is enough)
            if (i & 1) { s1 += e; d1 = fmaf(e, fmaxf(x, -1000.0f), d1); } else { s0 += e; d0 = fmaf(e, fmaxf(x, -1000.0f), d0); }
        }
        s += s0 + s1;
        d += d0 + d1;
    }
    // of the logit z scale: its distance from m is formed as add() formed the others'. (A scale leaves it half a step above the largest one's, that of the rounded
    // m: no token is likelier than 1.)
    __device__ __forceinline__ float logprob(float z, float scale = 1.0f) const {
        const float l = fmaf(z, scale, -m) - logf(s);
        return m == -INFINITY && s == 0.0f ? -INFINITY : l > 0.0f ? 0.0f : l;
    }
    __device__ __forceinline__ float entropy() const { return m == -INFINITY && s == 0.0f ? 0.0f : logf(s) - d / s; }
};

// The statistics of a warp's lanes as one, in every lane: the common maximum first, so that each lane is rescaled once and without a branch
// (joined pair by pair, five rounds took 1,100 cycles).
__device__ __forceinline__ Stats warp_join(Stats v) {
    v.raise(warp_max(v.m));
    v.s = warp_sum(v.s);
    v.d = warp_sum(v.d);
    return v;
}

// (at: the token's sum z)
__device__ __forceinline__ float logprob_of(const Stats& st, float z, float scale, float cap) {
    return cap > 0.0f ? st.logprob(cap_logit(z, scale, cap)) : st.logprob(z, scale);
}
__device__ __forceinline__ void finish(const Stats& st, int token, float at, float scale, float cap, int64_t vocab, float* logprob, float* entropy, int* status) {
    if (entropy) *entropy = st.entropy();
    if (!logprob) return;
    const bool none = token == -1, outside = !none && (token < 0 || token >= vocab);
    if (outside && status) atomicExch(status, 1);
    *logprob = none ? 0.0f : outside ? __int_as_float(0x7fc00000) : logprob_of(st, at, scale, cap);
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

// x sigmoid(y ln 2) without an IEEE division: where 2^-y is infinite the quotient is 0.
__device__ __forceinline__ float times_sigmoid2(float x, float y) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + exp2_fast(-y)));
    return x * r;
}

// z Phi(z), Phi the normal distribution. With s = |z|: Phi(-s) = e^(-s^2 / 2) t P(t), t = 1 / (1 + 0.26 s), P a fit to erfcx (least largest relative
// error over 0 <= s <= 14.5 with the constants as they are stored: 8.2e-8); what s^2 and its product with log2(e) / 2 lose in rounding goes in by a factor. Off by 8 x 2^-24 of the
// result from z = -6 on and by 22 x 2^-24 at -12.6 (measured against 64 bits). With erfcf in its place 776 x 13580 x 264 took
// 53 us (37), in 32 bits 170 (109).
__device__ __forceinline__ float gelu(float z) {
    const float s = fminf(fabsf(z), 20.0f), h = s * s, y = h * -0.72134752f;
    float off = fmaf(h, -0.72134752f, -y);
    off = fmaf(fmaf(s, s, -h), -0.72134752f, off);
    float t;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(s, 0.26f, 1.0f)));
    float p = fmaf(t, 0.03023030050098896f, -0.15149444341659546f);
    p = fmaf(t, p, 0.24873320758342743f);
    p = fmaf(t, p, -0.1477893441915512f);
    p = fmaf(t, p, 0.1587587594985962f);
    p = fmaf(t, p, 0.05196481943130493f);
    p = fmaf(t, p, 0.10278867930173874f);
    p = fmaf(t, p, 0.10305097699165344f);
    p = fmaf(t, p, 0.10375702381134033f);
    float e = exp2_fast(y);
    e = fmaf(e, off * 0.6931472f, e);
    const float q = e * (t * p);
    return z * (z >= 0.0f ? 1.0f - q : q);
}

__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case RELU: return z > 0.0f ? z : (z != z ? z : 0.0f);
        case RELU_SQUARED: { const float r = z > 0.0f ? z : (z != z ? z : 0.0f); return r * r; }
        // 0.5 z (1 + tanh u) = z sigmoid(2 u), u = sqrt(2/pi) (z + 0.044715 z^3); the constants are 2 sqrt(2/pi) log2(e) and 0.044715 of it
        case GELU_TANH: return times_sigmoid2(z, z * fmaf(z * z, 0.10294324f, 2.3022082f));
        case GELU: return gelu(z);
        case SILU: return times_sigmoid2(z, LOG2E * z);
    }
    return z;
}
// N elements under one switch (a switch for each cost the epilogues more than the activations).
template <int N> __device__ __forceinline__ void activate_all(float (&z)[N], int act) {
#define IB_EACH(A) case A: { _Pragma("unroll") for (int i = 0; i < N; i++) z[i] = activate(z[i], A); break; }
    switch (act) { IB_EACH(RELU) IB_EACH(RELU_SQUARED) IB_EACH(GELU_TANH) IB_EACH(GELU) IB_EACH(SILU) }
#undef IB_EACH
}

}  // namespace score
}  // namespace ib

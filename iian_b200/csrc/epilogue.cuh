// What follows a matrix product in the kernel that forms it: out = residual + act(product + bias), in float32, one rounding at the end.
#pragma once
#include "common.cuh"

namespace iian {

enum { LACT_NONE = 0, LACT_SILU = 1, LACT_GELU_TANH = 2, LACT_GELU = 3, LACT_RELU = 4, LACT_RELU2 = 5, LACT_COUNT = 6 };

// What bounds an epilogue with an activation is the hardware's exponential and reciprocal (8 cycles each for a warp), so each form has as few
// of them as it can.  silu is y / (1 + e^-y), gelu_tanh y / (1 + e^-2u), which is 0.5 y (1 + tanh u) without the difference that loses
// the digits of its lower tail.  gelu y = max(y, 0) - |y| Q(|y|) with Q(t) = e^(-t^2 / 2) s P(s), s = 1 / (1 + 0.3 t): the tail keeps its digits,
// to 1e-6 of its value at y = -2, 3e-6 at -5.  P is the minimax polynomial of degree 7 in 1 - 2 s for 0 <= t <= 13.3 (1.2e-7 relative), where Q
// ends.  Results are float32 within a few 1e-7 of the value otherwise.
__device__ __forceinline__ float linear_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float linear_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int ACT> __device__ __forceinline__ float linear_act_of(float y) {
    if constexpr (ACT == LACT_SILU) return y * linear_rcp(1.0f + linear_exp2(-1.4426950408889634f * y));
    else if constexpr (ACT == LACT_GELU_TANH)              // 2 sqrt(2 / pi) log2 e and 0.044715 times that
        return y * linear_rcp(1.0f + linear_exp2(y * fmaf(y * y, -0.10294324f, -2.3022082f)));
    else if constexpr (ACT == LACT_GELU) {
        const float t = fabsf(y), s = linear_rcp(fmaf(0.3f, t, 1.0f)), q = fmaf(-2.0f, s, 1.0f);
        float p = fmaf(q, -0.00028153285f, -0.00050916435f);
        p = fmaf(q, p, 0.0024370512f);
        p = fmaf(q, p, 0.0017998982f);
        p = fmaf(q, p, -0.027763564f);
        p = fmaf(q, p, 0.08655123f);
        p = fmaf(q, p, -0.16457935f);
        p = fmaf(q, p, 0.22197059f);
        const float e = linear_exp2(t * t * -0.72134752044448170f);           // e^(-t^2 / 2)
        return fmaf(-(fminf(t, 64.0f) * e), s * p, y < 0.0f ? 0.0f : y);      // (an infinity times the 0 there would be no number)
    } else if constexpr (ACT == LACT_RELU) return y < 0.0f ? 0.0f : y;        // (what is no number stays none)
    else if constexpr (ACT == LACT_RELU2) return y < 0.0f ? 0.0f : y * y;
    else return y;
}

// One decision for all of COUNT values: between them the compiler interleaves, where each had its own branch they came one after the other
// (2,048 x 12,288 x 4,096 with gelu 364 us).
template <int COUNT> __device__ __forceinline__ void linear_act_values(float * y, int act) {
    auto all = [&](auto one) {
#pragma unroll
        for (int i = 0; i < COUNT; i++) y[i] = one(y[i]);
    };
    switch (act) {
        case LACT_SILU: all([](float v) { return linear_act_of<LACT_SILU>(v); }); break;
        case LACT_GELU_TANH: all([](float v) { return linear_act_of<LACT_GELU_TANH>(v); }); break;
        case LACT_GELU: all([](float v) { return linear_act_of<LACT_GELU>(v); }); break;
        case LACT_RELU: all([](float v) { return linear_act_of<LACT_RELU>(v); }); break;
        case LACT_RELU2: all([](float v) { return linear_act_of<LACT_RELU2>(v); }); break;
        default: break;
    }
}

// bias [M] or null; residual [N, M], float32 or bfloat16 (res_bf16), rows ldr apart, or null: may be `out` itself, every entry is read by the
// thread that writes it, before it does; out rows ldo apart.
struct LinearEpilogue {
    const float * bias;
    const void * res;
    void * out;
    long long ldr, ldo;
    int act, res_bf16, out_bf16;
    int res_vec, out_vec, bias_vec;       // whether 4 neighbouring columns from a multiple of 4 on are one aligned access

    __device__ __forceinline__ float residual1(size_t at) const {
        return res_bf16 ? __bfloat162float(((const __nv_bfloat16 *) res)[at]) : ((const float *) res)[at];
    }
    __device__ __forceinline__ void put1(float y, size_t at) const {
        if (out_bf16) ((__nv_bfloat16 *) out)[at] = __float2bfloat16_rn(y);
        else ((float *) out)[at] = y;
    }
    __device__ __forceinline__ void store(float y, size_t row, int col) const {
        if (bias != nullptr) y += bias[col];
        linear_act_values<1>(&y, act);
        if (res != nullptr) y += residual1(row * (size_t) ldr + col);
        put1(y, row * (size_t) ldo + col);
    }
    // 4 columns from col (a multiple of 4) on, `live` of them inside the matrix: the bias, the residual, and the results
    __device__ __forceinline__ float4 bias4(int col, int live) const {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (bias == nullptr || live <= 0) return v;
        if (live >= 4 && bias_vec) return __ldg(reinterpret_cast<const float4 *>(bias + col));
        v.x = bias[col];
        if (live > 1) v.y = bias[col + 1];
        if (live > 2) v.z = bias[col + 2];
        if (live > 3) v.w = bias[col + 3];
        return v;
    }
    __device__ __forceinline__ float4 residual4(size_t row, int col, int live) const {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (res == nullptr || live <= 0) return v;
        const size_t at = row * (size_t) ldr + col;
        if (live >= 4 && res_vec) {
            if (!res_bf16) return *reinterpret_cast<const float4 *>((const float *) res + at);
            const uint2 raw = *reinterpret_cast<const uint2 *>((const __nv_bfloat16 *) res + at);
            const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&raw.x)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&raw.y));
            return make_float4(a.x, a.y, b.x, b.y);
        }
        v.x = residual1(at);
        if (live > 1) v.y = residual1(at + 1);
        if (live > 2) v.z = residual1(at + 2);
        if (live > 3) v.w = residual1(at + 3);
        return v;
    }
    __device__ __forceinline__ void put4(const float * y, size_t row, int col, int live) const {
        if (live <= 0) return;
        const size_t at = row * (size_t) ldo + col;
        if (live >= 4 && out_vec) {
            if (out_bf16) {
                __nv_bfloat162 p[2] = {__floats2bfloat162_rn(y[0], y[1]), __floats2bfloat162_rn(y[2], y[3])};
                *reinterpret_cast<uint2 *>((__nv_bfloat16 *) out + at) = *reinterpret_cast<uint2 *>(p);
            } else {
                *reinterpret_cast<float4 *>((float *) out + at) = make_float4(y[0], y[1], y[2], y[3]);
            }
            return;
        }
        put1(y[0], at);
        if (live > 1) put1(y[1], at + 1);
        if (live > 2) put1(y[2], at + 2);
        if (live > 3) put1(y[3], at + 3);
    }
};

// The arguments of an entry point as the kernels take them; false: a kind that there is none of.
static inline bool linear_epilogue(LinearEpilogue & e, const float * bias, const void * res, int res_dtype, long long ldr, void * out, int out_dtype,
                                   long long ldo, int act) {
    if (act < 0 || act >= LACT_COUNT || (res_dtype != IIAN_F32 && res_dtype != IIAN_BF16) || (out_dtype != IIAN_F32 && out_dtype != IIAN_BF16)) return false;
    e.bias = bias; e.res = res; e.out = out; e.ldr = ldr; e.ldo = ldo; e.act = act;
    e.res_bf16 = res_dtype == IIAN_BF16;
    e.out_bf16 = out_dtype == IIAN_BF16;
    e.bias_vec = ((uintptr_t) bias & 15) == 0;
    e.res_vec = (uintptr_t) res % (e.res_bf16 ? 8 : 16) == 0 && ldr % 4 == 0;
    e.out_vec = (uintptr_t) out % (e.out_bf16 ? 8 : 16) == 0 && ldo % 4 == 0;
    return true;
}

}  // namespace iian

// What follows a matrix product in the kernel that forms it: out = residual + act(product + bias), in float32, one rounding at the end.
#pragma once
#include "common.cuh"

namespace iian {

enum { LACT_NONE = 0, LACT_SILU = 1, LACT_GELU_TANH = 2, LACT_GELU = 3, LACT_RELU = 4, LACT_RELU2 = 5, LACT_COUNT = 6 };

__device__ __forceinline__ float linear_act_value(float y, int act) {
    switch (act) {
        case LACT_SILU: return y / (1.0f + expf(-y));
        case LACT_GELU_TANH: return 0.5f * y * (1.0f + tanhf(0.7978845608028654f * (y + 0.044715f * y * y * y)));
        case LACT_GELU: return 0.5f * y * (1.0f + erff(0.7071067811865476f * y));
        case LACT_RELU: return y < 0.0f ? 0.0f : y;          // (what is no number stays none)
        case LACT_RELU2: return y < 0.0f ? 0.0f : y * y;
        default: return y;
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
    int res_vec, out_vec, bias_vec;       // whether 8 neighbouring columns from a multiple of 8 on lie on 16 bytes

    __device__ __forceinline__ float one(float y, size_t row, int col) const {
        if (bias != nullptr) y += bias[col];
        y = linear_act_value(y, act);
        if (res != nullptr) {
            const size_t at = row * (size_t) ldr + col;
            y += res_bf16 ? __bfloat162float(((const __nv_bfloat16 *) res)[at]) : ((const float *) res)[at];
        }
        return y;
    }
    __device__ __forceinline__ void store(float y, size_t row, int col) const {
        y = one(y, row, col);
        const size_t at = row * (size_t) ldo + col;
        if (out_bf16) ((__nv_bfloat16 *) out)[at] = __float2bfloat16_rn(y);
        else ((float *) out)[at] = y;
    }
    // 8 columns from col on, `live` of them inside the matrix
    __device__ __forceinline__ void store8(float * y, size_t row, int col, int live) const {
        if (live < 8) {
#pragma unroll
            for (int i = 0; i < 7; i++)
                if (i < live) store(y[i], row, col + i);
            return;
        }
        if (bias != nullptr) {
            if (bias_vec) {
                const float4 a = __ldg(reinterpret_cast<const float4 *>(bias + col)), b = __ldg(reinterpret_cast<const float4 *>(bias + col + 4));
                y[0] += a.x; y[1] += a.y; y[2] += a.z; y[3] += a.w; y[4] += b.x; y[5] += b.y; y[6] += b.z; y[7] += b.w;
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] += bias[col + i];
            }
        }
        if (act != LACT_NONE) {
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = linear_act_value(y[i], act);
        }
        if (res != nullptr) {
            const size_t at = row * (size_t) ldr + col;
            if (res_bf16) {
                const __nv_bfloat16 * r = (const __nv_bfloat16 *) res + at;
                float f[8];
                if (res_vec) unpack8(*reinterpret_cast<const uint4 *>(r), f);
                else {
#pragma unroll
                    for (int i = 0; i < 8; i++) f[i] = __bfloat162float(r[i]);
                }
#pragma unroll
                for (int i = 0; i < 8; i++) y[i] += f[i];
            } else {
                const float * r = (const float *) res + at;
                if (res_vec) {
                    const float4 a = *reinterpret_cast<const float4 *>(r), b = *reinterpret_cast<const float4 *>(r + 4);
                    y[0] += a.x; y[1] += a.y; y[2] += a.z; y[3] += a.w; y[4] += b.x; y[5] += b.y; y[6] += b.z; y[7] += b.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) y[i] += r[i];
                }
            }
        }
        const size_t at = row * (size_t) ldo + col;
        if (out_bf16) {
            __nv_bfloat16 * o = (__nv_bfloat16 *) out + at;
            __nv_bfloat162 p[4];
#pragma unroll
            for (int i = 0; i < 4; i++) p[i] = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
            if (out_vec) *reinterpret_cast<uint4 *>(o) = *reinterpret_cast<uint4 *>(p);
            else {
#pragma unroll
                for (int i = 0; i < 4; i++) { o[2 * i] = p[i].x; o[2 * i + 1] = p[i].y; }
            }
        } else {
            float * o = (float *) out + at;
            if (out_vec) {
                *reinterpret_cast<float4 *>(o) = make_float4(y[0], y[1], y[2], y[3]);
                *reinterpret_cast<float4 *>(o + 4) = make_float4(y[4], y[5], y[6], y[7]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) o[i] = y[i];
            }
        }
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
    e.res_vec = ((uintptr_t) res & 15) == 0 && ldr * (e.res_bf16 ? 2 : 4) % 16 == 0;
    e.out_vec = ((uintptr_t) out & 15) == 0 && ldo * (e.out_bf16 ? 2 : 4) % 16 == 0;
    return true;
}

}  // namespace iian

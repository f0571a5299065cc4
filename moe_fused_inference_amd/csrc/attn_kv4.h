// attn_kv4.h -- where attention over the MXFP4 cache leaves a row: fp32, bf16 or
// fp16, and / or the MXFP4 rows of its bf16 rounding (o_proj's activations).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mx_device.h"
#include "mxfp4_hip.h"
#include "quant_rows.h"

namespace mxa {

struct Out {
    void* o;        // or null
    int dtype;      // MXFP4_DT_*
    uint8_t* oq;    // or null, with os
    uint8_t* os;
};

// Columns c0 .. c0 + N - 1 (N = 8 or 4) of row `row` of (rows, D).  The lanes of a
// 32-block are neighbours (four of 8 columns, eight of 4) and all call it.
template <int N>
__device__ __forceinline__ void store(const Out& t, int64_t row, int D, int c0, const float (&o)[N]) {
    const int64_t at = row * D + c0;
    if (t.o) {
        if (t.dtype == MXFP4_DT_F32) {
            float* p = static_cast<float*>(t.o) + at;
#pragma unroll
            for (int c = 0; c < N; c += 4) *reinterpret_cast<float4*>(p + c) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
        } else {
            uint32_t w[N / 2];
#pragma unroll
            for (int c = 0; c < N; c += 2) {
                if (t.dtype == MXFP4_DT_BF16) {
                    w[c / 2] = mx::f32x2_to_bf16x2(o[c], o[c + 1]);
                } else {
                    w[c / 2] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)o[c]) |
                               (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)o[c + 1]) << 16;
                }
            }
            uint16_t* p = static_cast<uint16_t*>(t.o) + at;
            if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
            else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        }
    }
    if (t.oq) {
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, am = 0.0f;
#pragma unroll
        for (int c = 0; c < N; ++c) {
            v[c] = mx::bf16_to_f32(mx::f32_to_bf16_rne(o[c]));
            am = fmaxf(am, __builtin_fabsf(v[c]));
        }
        am = fmaxf(am, mx::dpp<mx::kDppQuadXor1>(am));
        am = fmaxf(am, mx::dpp<mx::kDppQuadXor2>(am));
        if constexpr (N == 4) am = fmaxf(am, mx::dpp<mx::kDppRowHalfMirror>(am));
        const uint32_t code = mx::e8m0_code(am);
        const uint32_t packed = mx::e2m1_pack8_short(v, mx::e8m0_inv_scale(code));
        uint8_t* q = t.oq + at / 2;
        if constexpr (N == 8) *reinterpret_cast<uint32_t*>(q) = packed;
        else *reinterpret_cast<uint16_t*>(q) = (uint16_t)packed;
        if (c0 % 32 == 0) t.os[at / 32] = (uint8_t)code;
    }
}

}  // namespace mxa

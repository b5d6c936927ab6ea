// gfx950 kernel of the block join: what a transformer block's output goes through before the next block reads it.
//
//   z  = p0 + p1 + p2 + p3 (BF16 planes, in order, FP32)
//   z  = z * rsqrt(mean z^2 + eps) * post_w          (where the block has a norm after it)
//   h' = h + scale * gate * z
//   n  = h' * rsqrt(mean h'^2 + eps) * pre_w         -> BF16 and / or wire rows (E4M3, a UE8M0 byte per 32)
//
// HBM-bound: a value costs 2 bytes per plane and 4 of h in, 4 of h' and 2 (BF16) and / or 1.03 (wire) out, against about
// 30 vector instructions. As separate calls (rank sum, residual add, norm, quantizer) z, h' and n travel to memory and back.
// One workgroup holds a row in registers between the two sums, so each value is read once and written once.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "q0_codec.h"

namespace m26g {

struct JoinArgs {
    const uint16_t* plane[4];
    const float *h, *gate, *pre_w, *post_w;
    float* h_out;
    uint16_t* norm;
    uint8_t *payload, *scales;
    long rows, plane_pitch, h_pitch, norm_pitch, gate_pitch;
    size_t payload_pitch, scales_pitch;
    int cols, planes, gate_cols;
    float scale, eps;
};

template <int CTRL, int ROWS>
__device__ __forceinline__ float add_from(float v) {  // v plus the lane's counterpart; lanes of rows outside ROWS add nothing
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, false));
}
// Sum over the wave, the same in every lane: within rows of sixteen by DPP, then rows 0 and 2 handed on, then the lower half.
__device__ __forceinline__ float wave_sum(float v) {
    v = add_from<0xB1, 0xf>(v);   // quad_perm [1,0,3,2]
    v = add_from<0x4E, 0xf>(v);   // quad_perm [2,3,0,1]
    v = add_from<0x141, 0xf>(v);  // row_half_mirror
    v = add_from<0x140, 0xf>(v);  // row_mirror
    v = add_from<0x142, 0xa>(v);  // row_bcast15 into rows 1 and 3
    v = add_from<0x143, 0xc>(v);  // row_bcast31 into rows 2 and 3
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

__device__ __forceinline__ uint32_t q0_byte_of_block(uint32_t most, float amax_of_numbers) {
    // `most`: largest magnitude pattern of the block. Numbers only: the exponent field rebased, with the carry of the
    // 0.875 threshold (quantize_hidden_kernel has the derivation); otherwise the rule on the largest number.
    if (most >= 0x7f800000u) return q0_scale_byte(amax_of_numbers);
    const uint32_t field = (most + 0x1fffffu) >> 23;
    return field > 8u ? field - 8u : 0u;
}
__device__ __forceinline__ float q0_inverse(uint32_t s) { return __uint_as_float(s == 254u ? 0x00400000u : (254u - s) << 23); }

// A workgroup per row at a time. VEC: a thread holds NG groups of eight neighbouring values, T groups apart (16-byte
// accesses); otherwise 8 * NG single values, T apart.
template <int T, int NG, bool VEC>
__global__ void __launch_bounds__(T) block_join_kernel(const JoinArgs a) {
    constexpr int WAVES = T / 64, N = 8 * NG;
    __shared__ float parts[2][WAVES];  // the two sums take turns, so a row's second barrier also guards its first sum's slots
    const int tid = threadIdx.x, wave = tid >> 6;
    int turn = 0;
    auto row_sum = [&](float v) {
        v = wave_sum(v);
        if ((tid & 63) == 0) parts[turn][wave] = v;
        __syncthreads();
        float s = parts[turn][0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s += parts[turn][w];
        turn ^= 1;
        return s;
    };
    // value i of this thread is column column(i); in_row(i) for whole groups of eight when VEC
    auto column = [&](int i) { return VEC ? (tid + T * (i >> 3)) * 8 + (i & 7) : tid + T * i; };
    auto floats = [&](const float* p, float (&v)[N]) {  // one row of floats
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                const int c = column(8 * j);
                float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
                if (c < a.cols) { lo = *reinterpret_cast<const float4*>(p + c); hi = *reinterpret_cast<const float4*>(p + c + 4); }
                v[8 * j] = lo.x; v[8 * j + 1] = lo.y; v[8 * j + 2] = lo.z; v[8 * j + 3] = lo.w;
                v[8 * j + 4] = hi.x; v[8 * j + 5] = hi.y; v[8 * j + 6] = hi.z; v[8 * j + 7] = hi.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = column(i) < a.cols ? p[column(i)] : 0.0f;
        }
    };
    auto halves = [&](const uint16_t* p, float (&v)[N]) {  // one row of BF16 values
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                const int c = column(8 * j);
                uint4 w = make_uint4(0, 0, 0, 0);
                if (c < a.cols) w = *reinterpret_cast<const uint4*>(p + c);
                const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) { v[8 * j + 2 * i] = __uint_as_float(d[i] << 16); v[8 * j + 2 * i + 1] = __uint_as_float(d[i] & 0xffff0000u); }
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = column(i) < a.cols ? __uint_as_float(uint32_t(p[column(i)]) << 16) : 0.0f;
        }
    };
    auto squares = [&](const float (&v)[N]) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) s = __builtin_fmaf(v[i], v[i], s);
        return s;
    };
    const float inv_cols = 1.0f / float(a.cols);
    for (long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        float z[N], h[N], t[N];
        halves(a.plane[0] + r * a.plane_pitch, z);
        floats(a.h + r * a.h_pitch, h);
        for (int p = 1; p < a.planes; ++p) {
            halves(a.plane[p] + r * a.plane_pitch, t);
#pragma unroll
            for (int i = 0; i < N; ++i) z[i] += t[i];
        }
        if (a.post_w) {
            floats(a.post_w, t);
            const float k = 1.0f / sqrtf(row_sum(squares(z)) * inv_cols + a.eps);
#pragma unroll
            for (int i = 0; i < N; ++i) z[i] = z[i] * k * t[i];
        }
        if (a.gate_cols > 1) {
            floats(a.gate + r * a.gate_pitch, t);
#pragma unroll
            for (int i = 0; i < N; ++i) h[i] += a.scale * (t[i] * z[i]);
        } else {
            const float g = a.gate_cols == 1 ? a.scale * a.gate[r * a.gate_pitch] : a.scale;
#pragma unroll
            for (int i = 0; i < N; ++i) h[i] += g * z[i];
        }
        if (a.h_out) {
            float* o = a.h_out + r * a.h_pitch;
            if constexpr (VEC) {
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    const int c = column(8 * j);
                    if (c >= a.cols) continue;
                    *reinterpret_cast<float4*>(o + c) = make_float4(h[8 * j], h[8 * j + 1], h[8 * j + 2], h[8 * j + 3]);
                    *reinterpret_cast<float4*>(o + c + 4) = make_float4(h[8 * j + 4], h[8 * j + 5], h[8 * j + 6], h[8 * j + 7]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (column(i) < a.cols) o[column(i)] = h[i];
            }
        }
        if (!a.norm && !a.payload) continue;  // the same for every thread
        floats(a.pre_w, t);
        const float k = 1.0f / sqrtf(row_sum(squares(h)) * inv_cols + a.eps);
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] = h[i] * k * t[i];
        if (a.norm) {
            uint16_t* o = a.norm + r * a.norm_pitch;
            if constexpr (VEC) {
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    const int c = column(8 * j);
                    if (c >= a.cols) continue;
                    const float* v = h + 8 * j;
                    *reinterpret_cast<uint4*>(o + c) = make_uint4(bf16_rne_nan(v[0]) | bf16_rne_nan(v[1]) << 16, bf16_rne_nan(v[2]) | bf16_rne_nan(v[3]) << 16,
                                                                  bf16_rne_nan(v[4]) | bf16_rne_nan(v[5]) << 16, bf16_rne_nan(v[6]) | bf16_rne_nan(v[7]) << 16);
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (column(i) < a.cols) o[column(i)] = uint16_t(bf16_rne_nan(h[i]));
            }
        }
        if (!a.payload) continue;
        // Wire rows. A block of 32 values is four neighbouring lanes when VEC, half a wave otherwise; cols is a multiple
        // of 32 here, so a block is in the row as a whole or not at all.
        auto numbers = [](float f) { return f != f ? 0.0f : fabsf(f); };
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                const float* v = h + 8 * j;
                const int c = column(8 * j);
                uint32_t most = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) { const uint32_t m = __float_as_uint(v[i]) & 0x7fffffffu; most = m > most ? m : most; }
                most = max_bits_over_four(most);
                float amax = 0.0f;
                if (most >= 0x7f800000u) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, numbers(v[i]));
                    amax = __uint_as_float(max_bits_over_four(__float_as_uint(amax)));
                }
                if (c >= a.cols) continue;
                const uint32_t s = q0_byte_of_block(most, amax);
                const float inv = q0_inverse(s);
                *reinterpret_cast<uint2*>(a.payload + r * a.payload_pitch + c) =
                    make_uint2(e4m3_half_up4(make_float4(v[0], v[1], v[2], v[3]), inv), e4m3_half_up4(make_float4(v[4], v[5], v[6], v[7]), inv));
                if ((tid & 3) == 0) a.scales[r * a.scales_pitch + c / 32] = uint8_t(s);
            }
        } else {
            for (int i = 0; i < N; ++i) {
                uint32_t most = __float_as_uint(h[i]) & 0x7fffffffu;
                float amax = numbers(h[i]);
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const uint32_t m = __shfl_xor(most, d);
                    most = m > most ? m : most;
                    amax = fmaxf(amax, __shfl_xor(amax, d));
                }
                if (column(i) >= a.cols) continue;
                const uint32_t s = q0_byte_of_block(most, amax);
                a.payload[r * a.payload_pitch + column(i)] = uint8_t(e4m3_half_up(h[i], q0_inverse(s)));
                if ((tid & 31) == 0) a.scales[r * a.scales_pitch + column(i) / 32] = uint8_t(s);
            }
        }
    }
}

}  // namespace m26g

// gfx950 kernel of the block join: what a transformer block's output goes through before the next block reads it.
//
//   z  = p0 + p1 + p2 + p3 (BF16 planes, in order, FP32)
//   z  = z * rsqrt(mean z^2 + eps) * post_w          (where the block has a norm after it)
//   h' = h + scale * gate * z
//   n  = h' * rsqrt(mean h'^2 + eps) * pre_w         -> BF16 and / or wire rows (E4M3, a UE8M0 byte per 32)
//
// HBM-bound: a value costs 2 bytes per plane and 4 of h in, 4 of h' and 2 (BF16) and / or 1.03 (wire) out, against about
// 30 vector instructions. As separate calls (rank sum, residual add, norm, quantizer) z, h' and n travel to memory and back.
// One workgroup holds a row in registers between the two sums, so each value is read once and written once: 8192 rows x 4096, one
// plane, norms on both sides, both outputs, 437 MB in 87 us (5.0 TB/s, what a copy reaches); 128 rows, four planes 4.4 us, of
// which a launch is 2 and the bytes 2.
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

// Sixteen bytes at any alignment of the element: the memory path takes them as they come, an odd row costs it a line more.
typedef float v4f __attribute__((ext_vector_type(4)));
typedef v4f v4f_any __attribute__((aligned(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef v4u v4u_any __attribute__((aligned(2)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef v2u v2u_any __attribute__((aligned(1)));

// A workgroup of T threads per row at a time; a thread holds NG groups of eight neighbouring values, T groups apart. With RAGGED the
// row's last group is the last eight values, of which the first ones belong to the group before it: they count as zero and
// are not written. (Loads value by value under a condition wait for one another: 1021 rows x 2047, two planes 11.0 us
// against 9.2.) Rows of
// under eight values are loaded value by value.
template <int T, int NG, bool RAGGED>
__global__ void __launch_bounds__(T) block_join_kernel(const JoinArgs a) {
    constexpr int WAVES = T / 64, N = 8 * NG;
    constexpr int LIVE = T == 1024 && NG == 2 && RAGGED ? 1 : 4;  // planes on their way together, as the 128 registers of a lane allow
    __shared__ float parts[2][WAVES];  // the sums take turns: who writes a slot again has passed the barrier behind its last readers
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
    // Of group j: whether it has values in the row, the column of its first one, and how many of them are not its own.
    auto there = [&](int j) { return (tid + T * j) * 8 < a.cols; };
    auto short_by = [&](int j) { return RAGGED && there(j) && (tid + T * j) * 8 + 8 > a.cols ? (tid + T * j) * 8 + 8 - a.cols : 0; };
    auto column = [&](int j) { return (tid + T * j) * 8 - (RAGGED && a.cols >= 8 ? short_by(j) : 0); };
    auto owned = [&](int j, int i) { return !RAGGED || (a.cols >= 8 ? i >= short_by(j) : i < a.cols); };
    const bool tiny = RAGGED && a.cols < 8;
    auto floats = [&](const float* p, float (&v)[N]) {  // one row of floats
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            v4f lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
            if (there(j)) {
                if (!tiny) {
                    lo = *reinterpret_cast<const v4f_any*>(p + column(j));
                    hi = *reinterpret_cast<const v4f_any*>(p + column(j) + 4);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (i < a.cols) lo[i] = p[i];
                        if (4 + i < a.cols) hi[i] = p[4 + i];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[8 * j + i] = lo[i]; v[8 * j + 4 + i] = hi[i]; }
        }
    };
    auto halves = [&](const uint16_t* p, v4u (&v)[NG]) {  // one row of BF16 values, as they lie
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            v[j] = v4u{0, 0, 0, 0};
            if (!there(j)) continue;
            if (!tiny) {
                v[j] = *reinterpret_cast<const v4u_any*>(p + column(j));
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < a.cols) v[j][i / 2] |= uint32_t(p[i]) << (16 * (i & 1));
            }
        }
    };
    auto own = [&](float (&v)[N]) {
        if constexpr (RAGGED)
#pragma unroll
            for (int j = 0; j < NG; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[8 * j + i] = owned(j, i) ? v[8 * j + i] : 0.0f;
    };
    auto add = [&](float (&z)[N], const v4u (&v)[NG]) {
#pragma unroll
        for (int j = 0; j < NG; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                z[8 * j + 2 * i] += __uint_as_float(v[j][i] << 16);
                z[8 * j + 2 * i + 1] += __uint_as_float(v[j][i] & 0xffff0000u);
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
        v4u plane[LIVE][NG];
        halves(a.plane[0] + r * a.plane_pitch, plane[0]);
#pragma unroll
        for (int p = 1; p < LIVE; ++p)
            if (p < a.planes) halves(a.plane[p] + r * a.plane_pitch, plane[p]);
        floats(a.h + r * a.h_pitch, h);
        if (a.post_w) floats(a.post_w, t);
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = 0.0f;
        add(z, plane[0]);
#pragma unroll
        for (int p = 1; p < LIVE; ++p)
            if (p < a.planes) add(z, plane[p]);
#pragma unroll
        for (int p = LIVE; p < 4; ++p)
            if (p < a.planes) {
                halves(a.plane[p] + r * a.plane_pitch, plane[0]);
                add(z, plane[0]);
            }
        own(z);
        if (a.post_w) {
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
        own(h);  // behind the gate: an infinite one makes NaN of a zero
        if (a.h_out) {
            float* o = a.h_out + r * a.h_pitch;
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                const int c = column(j);
                if (!there(j)) continue;
                if (!RAGGED || short_by(j) == 0) {
                    *reinterpret_cast<v4f_any*>(o + c) = v4f{h[8 * j], h[8 * j + 1], h[8 * j + 2], h[8 * j + 3]};
                    *reinterpret_cast<v4f_any*>(o + c + 4) = v4f{h[8 * j + 4], h[8 * j + 5], h[8 * j + 6], h[8 * j + 7]};
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (owned(j, i)) o[c + i] = h[8 * j + i];
                }
            }
        }
        if (!a.norm && !a.payload) continue;  // the same for every thread
        floats(a.pre_w, t);
        const float k = 1.0f / sqrtf(row_sum(squares(h)) * inv_cols + a.eps);
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] = h[i] * k * t[i];
        if (a.norm) {
            uint16_t* o = a.norm + r * a.norm_pitch;
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                const int c = column(j);
                if (!there(j)) continue;
                if (!RAGGED || short_by(j) == 0) {
                    v4u w;
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = bf16_rne_nan(h[8 * j + 2 * i]) | bf16_rne_nan(h[8 * j + 2 * i + 1]) << 16;
                    *reinterpret_cast<v4u_any*>(o + c) = w;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (owned(j, i)) o[c + i] = uint16_t(bf16_rne_nan(h[8 * j + i]));
                }
            }
        }
        if (!a.payload) continue;
        // Wire rows: a block of 32 values is four neighbouring lanes; cols is a multiple of 32 here, so a block is in the row as
        // a whole or not at all.
        auto numbers = [](float f) { return f != f ? 0.0f : fabsf(f); };
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const float* v = h + 8 * j;
            const int c = column(j);
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
            if (!there(j)) continue;
            const uint32_t s = q0_byte_of_block(most, amax);
            const float inv = q0_inverse(s);
            *reinterpret_cast<v2u_any*>(a.payload + r * a.payload_pitch + c) =
                v2u{e4m3_half_up4(make_float4(v[0], v[1], v[2], v[3]), inv), e4m3_half_up4(make_float4(v[4], v[5], v[6], v[7]), inv)};
            if ((tid & 3) == 0) a.scales[r * a.scales_pitch + c / 32] = uint8_t(s);
        }
    }
}

}  // namespace m26g

// gfx950 kernels of the products with MXFP4 weights for few rows:
//
//   y[r][j] = sum over k of x[r][k] * e2m1(code[j][k]) * 2^(scale[j][k / 32] - 127),    x in BF16 or in wire rows
//
// A weight is 4.25 bits and meets each row once, so up to about 64 rows the weights' way from HBM is the bound. The weights
// are widened to BF16 in registers (v_cvt_scalef32_pk_bf16_fp4: two values and the group's scale in one instruction,
// exact for scale bytes 2..252) and multiplied on v_mfma_f32_16x16x32_bf16, whose products of BF16 values are exact and
// whose sums are FP32. One 16-column tile's 128 k take 1 KB of codes, 16 conversions and, per 16 rows, 4 MFMAs of 16 cycles
// on one of a compute unit's four SIMDs; at 6.5 TB/s such a kilobyte arrives every 96 cycles per compute unit.
//
// Operand order. v_mfma_f32_16x16x32_bf16: lane l holds row (l % 16) of either operand, eight k values of quarter
// (l / 16); the result's lane l holds D[4 * (l / 16) + i][l % 16]. Which k a quarter stands for is free as long as both
// operands agree: lane l takes group 4 * step + l / 16 of a 128-wide k-step, the 16 code bytes of one group of one weight row
// as the checkpoint has them, and feeds its 32 values to four MFMAs, eight at a time.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "q0_codec.h"

namespace m26g {

typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f32 __attribute__((ext_vector_type(4)));

// Prepared weights. payload [tile = ceil(n / 16)][step = ceil(k / 128)][lane = 64][16 B]; scales [tile][quad =
// ceil(steps / 4)][lane = 64][4 B], byte b of a dword for step 4 * quad + b. Rows past n and groups past k hold zero
// codes under scale 1.
struct W4Layout {
    long n, k;
    int tiles, steps, quads;
};

__global__ void __launch_bounds__(256) w4_prepare_kernel(const uint8_t* __restrict__ payload, const uint8_t* __restrict__ scales, W4Layout w,
                                                         uint8_t* __restrict__ out, uint8_t* __restrict__ out_scales, uint32_t* __restrict__ fault) {
    const long cells = long(w.tiles) * w.quads * 4 * 64;  // one lane of one step, the last quad's missing steps included
    for (long i = long(blockIdx.x) * 256 + threadIdx.x; i < cells; i += long(gridDim.x) * 256) {
        const int lane = int(i & 63);
        const long step = (i >> 6) % (w.quads * 4), tile = (i >> 6) / (w.quads * 4);
        const long row = tile * 16 + (lane & 15), group = step * 4 + (lane >> 4), groups = w.k / 32;
        uint4 codes = make_uint4(0, 0, 0, 0);
        uint32_t s = 127;
        if (row < w.n && group < groups) {
            codes = *reinterpret_cast<const uint4*>(payload + row * (w.k / 2) + group * 16);
            if ((codes.x | codes.y | codes.z | codes.w) & 0x77777777u) {
                s = scales[row * groups + group];
                if (s < 2 || s > 252) { atomicOr(fault, 1u); s = 127; }
            }
        }
        if (step < w.steps) *reinterpret_cast<uint4*>(out + ((tile * w.steps + step) * 64 + lane) * 16) = codes;
        out_scales[((tile * w.quads + step / 4) * 64 + lane) * 4 + step % 4] = uint8_t(s);
    }
}

struct W4Args {
    W4Layout w;
    const uint8_t* payload;
    const uint32_t* scales;
    const uint16_t* x;       // BF16 rows, or
    const uint8_t* x_codes;  // wire rows
    const uint8_t* x_scales;
    long x_pitch;            // elements, or bytes of the codes
    long x_scales_pitch;
    int rows;
    void* y;
    int y_bf16;
    long y_pitch;
};

// Eight weights (one dword of codes, low nibble first) as BF16.
__device__ __forceinline__ v8bf w4_widen(uint32_t codes, float scale) {
    union { v2bf pair[4]; v8bf all; } u;
    u.pair[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
    u.pair[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
    u.pair[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
    u.pair[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
    return u.all;
}

// The 32 values of one group of one row of x, as four MFMA operands.
struct W4Group {
    v8bf part[4];
};
template <bool FP8>
__device__ __forceinline__ W4Group w4_load_x(const W4Args& a, long row, long group, bool there) {
    W4Group g;
    if (!there) {  // past k: the weights are zero there, x has to be a number
        for (int i = 0; i < 4; ++i) g.part[i] = v8bf{};
        return g;
    }
    if constexpr (FP8) {
        const uint8_t* p = a.x_codes + row * a.x_pitch + group * 32;
        const uint32_t s = a.x_scales[row * a.x_scales_pitch + group];
        // scale byte 0 marks a block of zeros; 255 is not a number, and a NaN scale makes every product one
        const float scale = __uint_as_float(s == 255u ? 0x7fc00000u : (s ? s : 1u) << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint2 c = *reinterpret_cast<const uint2*>(p + 8 * i);
            union { v2bf pair[4]; v8bf all; } u;
            u.pair[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, scale, false);
            u.pair[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, scale, true);
            u.pair[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, scale, false);
            u.pair[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, scale, true);
            if (s == 255u)
                for (int j = 0; j < 8; ++j) u.all[j] = __bf16(__builtin_nanf(""));
            g.part[i] = u.all;
        }
    } else {
        const uint16_t* p = a.x + row * a.x_pitch + group * 32;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            union { uint4 bits; v8bf all; } u;
            u.bits = *reinterpret_cast<const uint4*>(p + 8 * i);
            g.part[i] = u.all;
        }
    }
    return g;
}

typedef uint32_t v4u32 __attribute__((ext_vector_type(4)));

// A run of memory with its end: loads past it return zero and move nothing, so a wave may ask for steps or tiles that are
// not there without a branch (a load under a condition makes the compiler wait for everything in flight).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t w4_run_of(const void* base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00027000);
}
constexpr int kStreamed = 2;  // non-temporal: a weight is used once

// Rows resident: x stays in registers. A workgroup's waves are `groups` column groups of `slices` k-slices, S steps each;
// a wave converts its slice of 16 * TT rows to matrix operands once and then walks over tiles, DEPTH of them in flight, with
// nothing but weights left to load. The slices' sums meet in LDS, in order, two buffers taking turns so that one
// barrier per tile does.
template <int TT, int S, int DEPTH, bool FP8>
__global__ void __launch_bounds__(512) w4_resident_kernel(const W4Args a, int slices, int groups, int turns) {
    __shared__ float sums[2][8][TT][256];
    const int lane = threadIdx.x & 63, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slice = wave % slices, group = wave / slices;
    const int row0 = blockIdx.y * 16 * TT, k_groups = int(a.w.k / 32);
    const long tile0 = long(blockIdx.x) * groups + group, tile_stride = long(gridDim.x) * groups;
    const uint32_t step_bytes = uint32_t(a.w.steps) * 1024, scale_bytes = uint32_t(a.w.quads) * 256;
    struct Tile {
        v4u32 codes[S];
        uint32_t scales[S];
    };
    auto load = [&](long tile, Tile& t) {
        const bool there = tile < a.w.tiles;
        const long at = there ? tile : 0;
        const __amdgpu_buffer_rsrc_t codes = w4_run_of(a.payload + at * step_bytes, there ? step_bytes : 0);
        const __amdgpu_buffer_rsrc_t scales = w4_run_of(reinterpret_cast<const uint8_t*>(a.scales) + at * scale_bytes, there ? scale_bytes : 0);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int step = slice * S + s;
            t.codes[s] = __builtin_amdgcn_raw_buffer_load_b128(codes, lane * 16, step * 1024, kStreamed);
            // one byte per step and lane; four neighbouring steps share a dword
            t.scales[s] = __builtin_amdgcn_raw_buffer_load_b8(scales, lane * 4, (step >> 2) * 256 + (step & 3), 0);
        }
    };
    Tile ahead[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(tile0 + d * tile_stride, ahead[d]);
    W4Group x[S][TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        const int r = row0 + 16 * t + (lane & 15);  // rows past the last repeat it: their columns of the result are not stored
        const long row = r < a.rows ? r : a.rows - 1;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int g = (slice * S + s) * 4 + q;
            x[s][t] = w4_load_x<FP8>(a, row, g, g < k_groups);
        }
    }
    for (int turn = 0; turn < turns; turn += DEPTH) {  // the same for every wave
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (turn + d >= turns) break;
            const long tile = tile0 + (turn + d) * tile_stride;
            v4f32 acc[TT];
#pragma unroll
            for (int t = 0; t < TT; ++t) acc[t] = v4f32{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const float scale = __uint_as_float(ahead[d].scales[s] << 23);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const v8bf wide = w4_widen(ahead[d].codes[s][i], scale);
#pragma unroll
                    for (int t = 0; t < TT; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wide, x[s][t].part[i], acc[t], 0, 0, 0);
                }
            }
            load(tile + DEPTH * tile_stride, ahead[d]);
            float (*mine)[TT][256] = sums[(turn + d) & 1];
#pragma unroll
            for (int t = 0; t < TT; ++t) *reinterpret_cast<v4f32*>(&mine[wave][t][(lane & 15) * 16 + 4 * q]) = acc[t];
            __syncthreads();
            for (int i = threadIdx.x; i < groups * TT * 256; i += blockDim.x) {
                const int g = i / (TT * 256), t = i / 256 % TT, cell = i % 256;
                float s = mine[g * slices][t][cell];
                for (int w = 1; w < slices; ++w) s += mine[g * slices + w][t][cell];
                const long r = row0 + 16 * t + cell / 16;
                const long c = (long(blockIdx.x) * groups + g + (turn + d) * tile_stride) * 16 + cell % 16;
                if (r >= a.rows || c >= a.w.n) continue;
                if (a.y_bf16) static_cast<uint16_t*>(a.y)[r * a.y_pitch + c] = uint16_t(bf16_rne_nan(s));
                else static_cast<float*>(a.y)[r * a.y_pitch + c] = s;
            }
        }
    }
}

// A workgroup of eight waves takes one tile of sixteen columns and 16 * TT rows; the waves take the tile's quads of k-steps
// in turn and their sums meet in LDS, in wave order.
template <int TT, bool FP8>
__global__ void __launch_bounds__(512) w4_matvec_kernel(const W4Args a) {
    constexpr int WAVES = 8;
    __shared__ float sums[WAVES][TT][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
    const long tile = blockIdx.x, row0 = long(blockIdx.y) * 16 * TT, groups = a.w.k / 32;
    v4f32 acc[TT];
    long row[TT];  // rows past the last repeat it: their columns of the result are not stored
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        acc[t] = v4f32{0.f, 0.f, 0.f, 0.f};
        const long r = row0 + 16 * t + (lane & 15);
        row[t] = r < a.rows ? r : a.rows - 1;
    }
    const uint4* payload = reinterpret_cast<const uint4*>(a.payload) + tile * a.w.steps * 64 + lane;
    const uint32_t* scales = a.scales + tile * a.w.quads * 64 + lane;
    for (int quad = wave; quad < a.w.quads; quad += WAVES) {
        const uint32_t sc = scales[quad * 64];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int step = quad * 4 + b;
            if (step >= a.w.steps) break;  // the same for the whole workgroup
            const uint4 codes = payload[step * 64];
            const long group = long(step) * 4 + q;
            W4Group x[TT];
#pragma unroll
            for (int t = 0; t < TT; ++t) x[t] = w4_load_x<FP8>(a, row[t], group, group < groups);
            const float scale = __uint_as_float(((sc >> (8 * b)) & 0xffu) << 23);
            const uint32_t dword[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const v8bf wide = w4_widen(dword[i], scale);
#pragma unroll
                for (int t = 0; t < TT; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wide, x[t].part[i], acc[t], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < TT; ++t)  // [row][column of the tile]
        *reinterpret_cast<v4f32*>(&sums[wave][t][(lane & 15) * 16 + 4 * q]) = acc[t];
    __syncthreads();
    for (int i = threadIdx.x; i < TT * 256; i += 512) {
        const long r = row0 + i / 16, c = tile * 16 + i % 16;
        float s = sums[0][i / 256][i % 256];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s += sums[w][i / 256][i % 256];
        if (r >= a.rows || c >= a.w.n) continue;
        if (a.y_bf16) static_cast<uint16_t*>(a.y)[r * a.y_pitch + c] = uint16_t(bf16_rne_nan(s));
        else static_cast<float*>(a.y)[r * a.y_pitch + c] = s;
    }
}

}  // namespace m26g

// gfx950 kernels of the products with MXFP4 weights for few rows:
//
//   y[r][j] = sum over k of x[r][k] * e2m1(code[j][k]) * 2^(scale[j][k / 32] - 127),    x in BF16 or in wire rows
//
// A weight is 4.25 bits and meets each row once, so up to about 64 rows the weights' way from HBM is the bound. The weights
// are widened to BF16 in registers (v_cvt_scalef32_pk_bf16_fp4: two values and the group's scale in one instruction,
// exact for scale bytes 2..252) and multiplied on v_mfma_f32_16x16x32_bf16, whose products of BF16 values are exact and
// whose sums are FP32. One 16-column tile's 128 k take 1 KB of codes, 16 conversions and, per 16 rows, 4 MFMAs of 16 cycles
// on one of a compute unit's four SIMDs; at 6.5 TB/s such a kilobyte arrives every 96 cycles per compute unit. 16 rows,
// 131072 x 4096: 48 us, 6.1 TB/s; 64 rows, 16384 x 4096: 16.5 us, of which fetching x takes 2.7, joining the slices' sums 2.6.
//
// Operand order. v_mfma_f32_16x16x32_bf16: lane l holds row (l % 16) of either operand, eight k values of quarter
// (l / 16); the result's lane l holds D[4 * (l / 16) + i][l % 16]. A 128-wide k-step is four MFMAs, one per group of 32, and a
// quarter is eight neighbouring values: the four lanes of a row of x read 64 neighbouring bytes with each load.
// (With a quarter holding a whole group the checkpoint's 16 bytes of a group stay together, but a load of x touches 64 separate
// pieces of 16 bytes: 16 rows x 4096 took 3.4 us to fetch instead of 1.)
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "q0_codec.h"
#include "wave_fence.h"

namespace m26g {

typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f32 __attribute__((ext_vector_type(4)));

// Prepared weights. payload [tile = ceil(n / 16)][step = ceil(k / 128)][lane = 64][4 dwords]: dword i of lane l is dword
// l / 16 of group 4 * step + i of row 16 * tile + l % 16 (eight codes, low nibble first). scales [tile][quad = ceil(steps / 4)]
// [column = 16][step % 4][4 B], byte i for group i of the step. Rows past n and groups past k hold zero codes under scale 1.
struct W4Layout {
    long n, k;
    int tiles, steps, quads;
};

__global__ void __launch_bounds__(256) w4_prepare_kernel(const uint8_t* __restrict__ payload, const uint8_t* __restrict__ scales, W4Layout w,
                                                         uint8_t* __restrict__ out, uint8_t* __restrict__ out_scales, uint32_t* __restrict__ fault) {
    const long cells = long(w.tiles) * w.quads * 4 * 64;  // one lane of one step, the last quad's missing steps included
    for (long cell = long(blockIdx.x) * 256 + threadIdx.x; cell < cells; cell += long(gridDim.x) * 256) {
        const int lane = int(cell & 63), q = lane >> 4;
        const long step = (cell >> 6) % (w.quads * 4), tile = (cell >> 6) / (w.quads * 4);
        const long row = tile * 16 + (lane & 15), groups = w.k / 32;
        const long group = step * 4 + q;  // this lane reads group q of its row's step and takes care of its scale
        uint4 all = make_uint4(0, 0, 0, 0);
        uint32_t s = 127;
        if (row < w.n && group < groups) {
            all = *reinterpret_cast<const uint4*>(payload + row * (w.k / 2) + group * 16);
            if ((all.x | all.y | all.z | all.w) & 0x77777777u) {
                s = scales[row * groups + group];
                if (s < 2 || s > 252) { atomicOr(fault, 1u); s = 127; }
            }
        }
        // dword i of this lane is dword q of the lane that read group i: the four lanes of a row exchange in four rounds
        uint32_t dword[4];
        for (int d = 0; d < 4; ++d) {
            const int other = q ^ d;
            const uint32_t got = __shfl_xor(other == 0 ? all.x : other == 1 ? all.y : other == 2 ? all.z : all.w, 16 * d);
            for (int i = 0; i < 4; ++i)
                if (i == other) dword[i] = got;
        }
        if (step < w.steps) *reinterpret_cast<uint4*>(out + ((tile * w.steps + step) * 64 + lane) * 16) = make_uint4(dword[0], dword[1], dword[2], dword[3]);
        out_scales[(((tile * w.quads + step / 4) * 16 + (lane & 15)) * 4 + step % 4) * 4 + q] = uint8_t(s);
    }
}

struct W4Args {
    W4Layout w;
    const uint8_t* payload;
    const uint32_t* scales;
    const uint16_t* x;       // BF16 rows, or
    const uint8_t* x_codes;  // wire rows
    const uint8_t* x_scales;
    bool fp8;
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

typedef uint32_t u32_any __attribute__((aligned(1)));
typedef uint32_t v2u32 __attribute__((ext_vector_type(2)));
typedef uint32_t v4u32 __attribute__((ext_vector_type(4)));

// A run of memory with its end: loads past it return zero and move nothing, so a wave may ask for steps or tiles that are
// not there without a branch (a load under a condition makes the compiler wait for everything in flight).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t w4_run_of(const void* base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00027000);
}
constexpr uint32_t kRunMost = 0x7fffffff;  // a run whose end only kOutside passes
constexpr int kOutside = int(0x80000000u);
constexpr int kStreamed = 2;  // non-temporal: a weight is used once

// A lane's share of STEPS k-steps of TT * 16 rows of x, as MFMA operands. The operand order asks for 64 bytes of each of
// sixteen rows at a time, which a compute unit's memory path serves at 16 bytes a cycle; four rows of 256 bytes come at
// 40 to 52. So a wave loads whole steps of rows, 256 bytes (128 of wire rows) each, and turns them round in a corner of LDS
// of its own, with a fence between the lanes' writes and the other lanes' reads and one behind the reads, ahead of the next step's
// writes. All loads are issued before the first is looked at; what is past k or past the last row is asked for outside the
// buffer, which moves nothing and gives zero. (Past k the weights are zero and x has to be a number.)
constexpr int kTurnRow = 256 + 16, kTurnBytes = 16 * kTurnRow;  // a row's step in LDS, padded so that the rows of a column start in different banks
template <int STEPS, int TT>
struct W4Rows {
    v8bf part[STEPS][TT][4];

    __device__ __forceinline__ void load(const W4Args& a, long row0, int rows, int step0, uint8_t* corner) {
        const int lane = threadIdx.x & 63, q = lane >> 4, c = lane & 15;
        if (a.fp8) {
            const __amdgpu_buffer_rsrc_t codes = w4_run_of(a.x_codes + row0 * a.x_pitch, kRunMost);
            const int groups = int(a.w.k / 32);
            v2u32 raw[STEPS][TT][4];
            // A step's four bytes of a row at once, at any alignment: byte by byte they took longer than the codes (16 rows, 256 x
            // 4096: 7.0 us against 4.6).
            uint32_t scale[STEPS][TT];
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
#pragma unroll
                for (int t = 0; t < TT; ++t) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row = 16 * t + 4 * i + q;
                        const bool there = row < rows && (step0 + s) * 128 + c * 8 < a.w.k;
                        raw[s][t][i] = __builtin_amdgcn_raw_buffer_load_b64(codes, there ? row * int(a.x_pitch) + c * 8 : kOutside, (step0 + s) * 128, 0);
                    }
                    // Rows that are not there take the last one's. At the row's end the last four bytes, moved down; past k the codes are zero.
                    const int row = 16 * t + c < rows ? 16 * t + c : rows - 1, group = (step0 + s) * 4;
                    const uint8_t* bytes = a.x_scales + (row0 + row) * a.x_scales_pitch;
                    if (groups >= 4) {
                        const int at = group + 4 <= groups ? group : groups - 4, past = group - at < 4 ? group - at : 0;
                        scale[s][t] = *reinterpret_cast<const u32_any*>(bytes + at) >> (8 * past);
                    } else {
                        scale[s][t] = bytes[0] | (groups > 1 ? bytes[1] << 8 : 0) | (groups > 2 ? bytes[2] << 16 : 0);
                    }
                }
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
#pragma unroll
                for (int t = 0; t < TT; ++t) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) *reinterpret_cast<v2u32*>(corner + (4 * i + q) * kTurnRow + c * 8) = raw[s][t][i];
                    wave_fence();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const v2u32 code = *reinterpret_cast<const v2u32*>(corner + c * kTurnRow + i * 32 + q * 8);
                        const uint32_t byte = scale[s][t] >> (8 * i) & 0xffu;
                        // The conversion reads the exponent field alone: byte 0 is 2^-127, which blocks of the smallest values carry. Codes are
                        // exact up to byte 246; under bytes 0..2 they are rounded to multiples of 2^-133, BF16's smallest step.
                        const float f = __uint_as_float(byte << 23);
                        union { v2bf pair[4]; v8bf all; uint32_t dword[4]; } u;
                        u.pair[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code.x, f, false);
                        u.pair[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code.x, f, true);
                        u.pair[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code.y, f, false);
                        u.pair[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code.y, f, true);
#pragma unroll
                        for (int j = 0; j < 4; ++j) u.dword[j] = byte == 255u ? 0x7fc07fc0u : u.dword[j];  // 255 is not a number
                        part[s][t][i] = u.all;
                    }
                    wave_fence();
                }
        } else {
            const __amdgpu_buffer_rsrc_t x = w4_run_of(a.x + row0 * a.x_pitch, kRunMost);
            v4u32 raw[STEPS][TT][4];
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
#pragma unroll
                for (int t = 0; t < TT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row = 16 * t + 4 * i + q;
                        const bool there = row < rows && (step0 + s) * 128 + c * 8 < a.w.k;
                        raw[s][t][i] = __builtin_amdgcn_raw_buffer_load_b128(x, there ? row * int(a.x_pitch) * 2 + c * 16 : kOutside, (step0 + s) * 256, 0);
                    }
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
#pragma unroll
                for (int t = 0; t < TT; ++t) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) *reinterpret_cast<v4u32*>(corner + (4 * i + q) * kTurnRow + c * 16) = raw[s][t][i];
                    wave_fence();
#pragma unroll
                    for (int i = 0; i < 4; ++i) part[s][t][i] = *reinterpret_cast<const v8bf*>(corner + c * kTurnRow + i * 64 + q * 16);
                    wave_fence();
                }
        }
    }
};

// The scale of group i of a step out of the step's dword.
__device__ __forceinline__ float w4_scale(uint32_t dword, int i) { return __uint_as_float((dword >> (8 * i) & 0xffu) << 23); }

// Rows resident: x stays in registers. A workgroup's waves are `groups` column groups of `slices` k-slices, S steps each;
// a wave converts its slice of 16 * TT rows to matrix operands once and then walks over the tiles, the next one on its way,
// with nothing but weights left to load. The slices' sums meet in LDS, in order, two buffers taking turns so that one
// barrier per turn does. A workgroup's tiles are neighbours, so that what it writes of a row grows into whole 256-byte
// pieces in its L2 (16 rows x 131072 columns from 131072 x 4096: 50 us; with a workgroup's tiles a grid apart, 64 bytes
// of a row from each XCD in turn, 55). Tiles past the last load and store nothing. blockIdx.y is a run of `share` rows.
//
// Where the registers do not hold x's whole width (LONG, one column group of W slices), it goes in phases of W * S steps: a
// phase loads its part of x, walks over all tiles, and the sums so far wait in LDS. Streaming x with the weights instead moves
// it once a tile (16 rows, 32768 x 16384: 93 us against 49, 6.0 TB/s).
constexpr int kTurnsKept = 32;
template <int TT, int S, int W, bool LONG, typename OUT>
__global__ void __launch_bounds__(64 * W, W / 4) w4_resident_kernel(const W4Args a, int slices, int groups, int turns, int phases, int share) {
    // Each wave's corner while x is turned round, the slices' sums afterwards.
    constexpr int kSums = 2 * W * TT * 256 * 4;
    __shared__ __attribute__((aligned(16))) uint8_t shared[kSums > W * kTurnBytes ? kSums : W * kTurnBytes];
    __shared__ float kept[LONG ? kTurnsKept : 1][TT * 256];  // each cell by one thread
    float (*sums)[W][TT][256] = reinterpret_cast<float (*)[W][TT][256]>(shared);
    // a workgroup is (64 lanes, slices, groups)
    const int lane = threadIdx.x, q = lane >> 4;
    const int slice = __builtin_amdgcn_readfirstlane(threadIdx.y), group = __builtin_amdgcn_readfirstlane(threadIdx.z), wave = group * slices + slice;
    const int row0 = blockIdx.y * share, rows = a.rows - row0 < share ? a.rows - row0 : share, threads = groups * slices * 64;
    auto tile_of = [&](int turn) { return turn < turns ? (int(blockIdx.x) * turns + turn) * groups : a.w.tiles; };  // of column group 0
    if (tile_of(0) >= a.w.tiles) return;  // the grid is rounded up
    const uint32_t step_bytes = uint32_t(a.w.steps) * 1024, scale_bytes = uint32_t(a.w.quads) * 256;
    struct Tile {
        v4u32 codes[S];
        uint32_t scales[S];
    };
    auto load = [&](int tile, int phase, Tile& t) {
        const int step0 = phase * (W * S) + slice * S;
        const bool there = tile < a.w.tiles;
        const long at = there ? tile : 0;
        const __amdgpu_buffer_rsrc_t codes = w4_run_of(a.payload + at * step_bytes, there ? step_bytes : 0);
        const __amdgpu_buffer_rsrc_t scales = w4_run_of(reinterpret_cast<const uint8_t*>(a.scales) + at * scale_bytes, there ? scale_bytes : 0);
#pragma unroll
        for (int s = 0; s < S; ++s) t.codes[s] = __builtin_amdgcn_raw_buffer_load_b128(codes, lane * 16, (step0 + s) * 1024, kStreamed);
        // a dword per step and column; four steps of a quad lie together
        if constexpr (S % 4 == 0) {
#pragma unroll
            for (int s = 0; s < S; s += 4) {
                const v4u32 v = __builtin_amdgcn_raw_buffer_load_b128(scales, (lane & 15) * 16, (step0 + s) * 64, kStreamed);
#pragma unroll
                for (int j = 0; j < 4; ++j) t.scales[s + j] = v[j];
            }
        } else {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const int step = step0 + s;
                t.scales[s] = __builtin_amdgcn_raw_buffer_load_b32(scales, (lane & 15) * 16, (step >> 2) * 256 + (step & 3) * 4, kStreamed);
            }
        }
    };
    Tile ahead;
    load(tile_of(0) + group, 0, ahead);
    for (int phase = 0; phase < (LONG ? phases : 1); ++phase) {
        if (phase) __syncthreads();  // the last turn's sums are read
        W4Rows<S, TT> x;
        x.load(a, row0, rows, phase * (W * S) + slice * S, shared + wave * kTurnBytes);
        __syncthreads();
        for (int turn = 0; turn < turns; ++turn) {  // the same for every wave
            const int tile = tile_of(turn);
            v4f32 acc[TT];
#pragma unroll
            for (int t = 0; t < TT; ++t) acc[t] = v4f32{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const v8bf wide = w4_widen(ahead.codes[s][i], w4_scale(ahead.scales[s], i));
#pragma unroll
                    for (int t = 0; t < TT; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wide, x.part[s][t][i], acc[t], 0, 0, 0);
                }
            // under the sums and stores of this one
            if (LONG && turn + 1 == turns && phase + 1 < phases) load(tile_of(0) + group, phase + 1, ahead);
            else load(tile_of(turn + 1) + group, phase, ahead);
            float (*mine)[TT][256] = sums[turn & 1];
#pragma unroll
            for (int t = 0; t < TT; ++t) *reinterpret_cast<v4f32*>(&mine[wave][t][(lane & 15) * 16 + 4 * q]) = acc[t];
            __syncthreads();
            const __amdgpu_buffer_rsrc_t y = w4_run_of(static_cast<OUT*>(a.y) + row0 * a.y_pitch + long(tile) * 16, kRunMost);
            const long left = a.w.n - long(tile) * 16;
            for (int i = wave * 64 + lane; i < groups * TT * 256; i += threads) {
                const int g = i / (TT * 256), t = i / 256 % TT, cell = i % 256, r = 16 * t + cell / 16, c = 16 * g + cell % 16;
                float s = 0.0f;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float part = mine[g * slices + (w < slices ? w : 0)][t][cell];
                    s += w < slices ? part : 0.0f;
                }
                if (LONG) {
                    if (phase) s += kept[turn][i];
                    kept[turn][i] = s;
                    if (phase + 1 < phases) continue;
                }
                const int at = (r * int(a.y_pitch) + c) * int(sizeof(OUT));
                if (r < rows && c < left) {
                    if constexpr (sizeof(OUT) == 2) __builtin_amdgcn_raw_buffer_store_b16(uint16_t(bf16_rne_nan(s)), y, at, 0, 0);
                    else __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(s), y, at, 0, 0);
                }
            }
        }
    }
}

// Rows streamed: a workgroup takes one tile of sixteen columns and `share` <= 16 rows; its waves take the tile's k-steps in
// turn, weights and rows alike, AHEAD of them on their way at once, and their sums meet in LDS, in wave order.
template <int WAVES, int AHEAD>
__global__ void __launch_bounds__(64 * WAVES) w4_streamed_kernel(const W4Args a, int share) {
    __shared__ float sums[WAVES][256];
    __shared__ __attribute__((aligned(16))) uint8_t corners[WAVES][kTurnBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4;
    const long tile = blockIdx.x, row0 = long(blockIdx.y) * share;
    if (tile >= a.w.tiles) return;  // the grid is rounded up
    const int rows = a.rows - row0 < share ? int(a.rows - row0) : share;
    const uint4* payload = reinterpret_cast<const uint4*>(a.payload) + tile * a.w.steps * 64 + lane;
    const uint32_t* scales = a.scales + tile * a.w.quads * 64 + (lane & 15) * 4;
    v4f32 acc = {0.f, 0.f, 0.f, 0.f};
    for (int first = wave * AHEAD; first < a.w.steps; first += WAVES * AHEAD) {
        uint4 codes[AHEAD];
        uint32_t scale[AHEAD];
#pragma unroll
        for (int s = 0; s < AHEAD; ++s) {
            const int step = first + s < a.w.steps ? first + s : a.w.steps - 1;
            codes[s] = payload[step * 64];
            scale[s] = scales[(step >> 2) * 64 + (step & 3)];
        }
        W4Rows<AHEAD, 1> x;  // zeros past k
        x.load(a, row0, rows, first, corners[wave]);
#pragma unroll
        for (int s = 0; s < AHEAD; ++s) {
            const uint32_t dword[4] = {codes[s].x, codes[s].y, codes[s].z, codes[s].w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w4_widen(dword[i], w4_scale(scale[s], i)), x.part[s][0][i], acc, 0, 0, 0);
        }
    }
    *reinterpret_cast<v4f32*>(&sums[wave][(lane & 15) * 16 + 4 * q]) = acc;  // [row][column of the tile]
    __syncthreads();
    const int i = threadIdx.x, r = i / 16;
    const long c = tile * 16 + i % 16;
    if (i >= 256 || r >= rows || c >= a.w.n) return;
    float s = sums[0][i];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s += sums[w][i];
    if (a.y_bf16) static_cast<uint16_t*>(a.y)[(row0 + r) * a.y_pitch + c] = uint16_t(bf16_rne_nan(s));
    else static_cast<float*>(a.y)[(row0 + r) * a.y_pitch + c] = s;
}

}  // namespace m26g

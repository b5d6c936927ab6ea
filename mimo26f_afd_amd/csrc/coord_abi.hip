// C ABI of the coordinator-side operators (include/m26c_coord.h): argument checks and launches.
#include "../../include/m26c_coord.h"
#include <cmath>
#include <new>
#include <stdio.h>
#include "join_kernels.h"
#include "logprob_kernels.h"
#include "w4_kernels.h"

namespace {

using namespace m26g;

int launched() { return int(hipGetLastError()); }
uintptr_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }
bool on(const void* p, uintptr_t boundary) { return address(p) % boundary == 0; }

// ---- block join
template <int T, int NG>
void launch_join(const JoinArgs& a, hipStream_t st) {
    const unsigned grid = unsigned(a.rows < 65536 ? a.rows : 65536);
    if (a.cols % 8) block_join_kernel<T, NG, true><<<grid, T, 0, st>>>(a);
    else block_join_kernel<T, NG, false><<<grid, T, 0, st>>>(a);
}

// ---- log probabilities
// How a call is cut, by rows and vocabulary alone (us a pass inside a captured graph on inputs in turn, as everywhere in this file; where a
// rule turns, both forms were timed at sizes on either side of it; walking / short parts):
//  * up to two waves' registers hold a row: a workgroup per row, short parts (16384 x 1000 BF16, top 5: 39 / 26)
//  * up to eight, as long as the chip holds all rows at once (512 x 8000, top 5: 11.8 / 9.6; 2048 x 8000 18.1 / 30.2 the other way)
//  * few rows: over several workgroups in short parts of two chunks, of four where 128 parts would not reach (1 row x 131072
//    FP32, top 20: 13.9 / 9.8; 128 x 50003 BF16, top 5: 17.4 / 14.9; 600 x 20000, top 5: 17.5 / 20.9 the other way)
//  * otherwise waves walk: over parts, about 4096 waves over all rows and two chunks each at least, or over whole rows where
//    that leaves a row fewer than eight parts (300 x 131072: 44 against 50).
struct LogprobCut {
    int parts;   // over several workgroups, 0: a workgroup takes whole rows
    int chunks;  // of a short part, 0: waves walk
};
LogprobCut cut_of(int rows, int vocab) {
    const int waves = (vocab + 2 * kChunk - 1) / (2 * kChunk);
    if (waves <= 2 || (waves <= 8 && long(waves) * rows <= 4096)) return {0, 2};
    const int chunks = vocab <= 2 * kChunk * kPartsMost ? 2 : 4;
    const long parts4 = (long(vocab) + chunks * kChunk * kPartWaves - 1) / (chunks * kChunk * kPartWaves), short_parts = parts4 * kPartWaves;
    if (short_parts <= kPartsMost && short_parts * rows <= 8192) return {int(short_parts), chunks};
    int parts = vocab / kChunk / 2;
    parts = parts < 4096 / rows ? parts : 4096 / rows;
    parts = parts < kPartsMost ? parts : kPartsMost;
    parts = parts / kPartWaves * kPartWaves;
    return {parts < 8 ? 0 : parts, 0};
}
size_t stats_bytes(int rows, int parts) { return size_t(rows) * parts * sizeof(float4); }

template <bool BF16, int WAVES>
int launch_rows(const LogprobArgs& a, hipStream_t st) {
    const int wide = a.rows < 4096 ? a.rows : 4096;  // workgroups walk over the rows from there on
    logprob_row_kernel<BF16, WAVES><<<unsigned(wide), 64 * WAVES, 0, st>>>(a);
    return launched();
}

template <bool BF16, int WAVES>
int launch_short_rows(const LogprobArgs& a, hipStream_t st) {
    const int wide = a.rows < 16384 ? a.rows : 16384;
    logprob_short_row_kernel<BF16, WAVES, 2><<<unsigned(wide), 64 * WAVES, 0, st>>>(a);
    return launched();
}

template <bool BF16>
int launch_logprobs(const LogprobArgs& a, int short_chunks, hipStream_t st) {
    if (a.parts) {
        const unsigned grid = unsigned(a.rows) * unsigned(a.parts / kPartWaves);
        if (short_chunks == 2) logprob_short_part_kernel<BF16, 2><<<grid, 64 * kPartWaves, 0, st>>>(a);
        else if (short_chunks == 4) logprob_short_part_kernel<BF16, 4><<<grid, 64 * kPartWaves, 0, st>>>(a);
        else logprob_part_kernel<BF16><<<grid, 64 * kPartWaves, 0, st>>>(a);
        if (int rc = launched()) return rc;
        logprob_join_kernel<BF16><<<unsigned(a.rows), kJoinThreads, 0, st>>>(a);
        return launched();
    }
    if (short_chunks) {
        const int waves = (a.vocab + 2 * kChunk - 1) / (2 * kChunk);
        if (waves == 1) return launch_short_rows<BF16, 1>(a, st);
        if (waves == 2) return launch_short_rows<BF16, 2>(a, st);
        if (waves <= 4) return launch_short_rows<BF16, 4>(a, st);
        return launch_short_rows<BF16, 8>(a, st);
    }
    // Waves to a row: as few as fill the chip, since each finds its own largest values first (2000 x 20000, top 30: two waves 52
    // us, four 60, eight 97; 1024 x 50003, top 20: four 43, two 52, eight 49; 600 x 100000, top 5: eight 37, four 40).
    if (a.rows >= 1536) return launch_rows<BF16, 2>(a, st);
    if (a.rows >= 768 || a.vocab < 16 * kChunk) return launch_rows<BF16, 4>(a, st);
    return launch_rows<BF16, 8>(a, st);
}

}  // namespace

// ---- MXFP4 weights
struct m26c_w4 {
    W4Layout lay;
    uint8_t* payload;
    uint32_t* scales;
    int device;
};

namespace {

constexpr long kPitchMost = 1L << 24;  // a kernel addresses up to 32 rows of x or y with 31 bits

int fail(char* err, size_t errlen, int rc, const char* what) {
    if (err && errlen) snprintf(err, errlen, "%s", what);
    return rc;
}

void release(m26c_w4* w) {
    if (!w) return;
    if (w->payload) (void)hipFree(w->payload);
    if (w->scales) (void)hipFree(w->scales);
    delete w;
}

// Workgroups go round over the eight XCDs. With a multiple of eight of them in a row of the grid, the runs of rows that read the
// same weights share an L2 (32000 x 8192, 64 rows in four runs: 56 us; with 63 workgroups in a row of the grid 93).
unsigned over_xcds(int wide, int runs) { return unsigned(runs > 1 ? (wide + 7) / 8 * 8 : wide); }

template <int TT, int S, int W, bool LONG = false>
int launch_resident(const W4Args& a, int workgroups, int share, hipStream_t st) {
    const int phases = LONG ? (a.w.steps + W * S - 1) / (W * S) : 1, slices = LONG ? W : (a.w.steps + S - 1) / S, groups = W / slices;
    const int tiles = (a.w.tiles + groups - 1) / groups;
    int turns = (tiles + workgroups - 1) / workgroups;
    if (LONG && turns > kTurnsKept) turns = kTurnsKept;
    const int wide = (tiles + turns - 1) / turns, runs = (a.rows + share - 1) / share;
    const dim3 grid(over_xcds(wide, runs), unsigned(runs)), block(64, unsigned(slices), unsigned(groups));
    if (a.y_bf16) w4_resident_kernel<TT, S, W, LONG, uint16_t><<<grid, block, 0, st>>>(a, slices, groups, turns, phases, share);
    else w4_resident_kernel<TT, S, W, LONG, float><<<grid, block, 0, st>>>(a, slices, groups, turns, phases, share);
    return launched();
}

// The form of a product, by sizes alone (us a pass):
//  * few tiles and rows: a workgroup per tile, rows streamed with the weights, as long as there is one per compute unit at most (256
//    tiles x 32 steps, 1 row 3.9 against 4.9 with resident rows; 157 x 128 9.8 against 12.9) or up to four with little to do each
//    (813 x 8, 16 rows 4.5 against 5.3; 626 x 17, 5 wire rows 6.5 against 7.8; 313 x 64 11.0 against 9.5 and 563 x 32 of
//    wire rows 10.9 against 8.9 the other way; against phases longer, 468 x 68 10.9 against 21.4, 750 x 68 16.2 against 19.7, 750 x
//    128 37 against 25 the other way). Eight waves, a step at a time: sixteen lose where tiles meet on a compute
//    unit (626 x 17 of wire rows 9.4 against 7.0), and so do two steps on their way (6.8 against 6.3), which gain on long k
//    (125 x 128, 16 rows 9.8 against 11.4; 256 x 64, 1 row 6.3 against 7.1).
//  * otherwise resident rows, as many workgroups over all row runs as fit on the compute units at once, so that each loads its
//    rows once. Sixteen waves hold sixteen rows up to 64 steps (8192 tiles x 32 steps: 48.3 us with sixteen waves of two steps, 50.1
//    with eight of four) and 32 rows up to 32 (1024 x 32, 64 rows: 17.8 against 22.3 with 16 a run). Up to 24 steps a workgroup of
//    sixteen rows has twelve waves at most, and two of them fit (3750 x 18: 17.4 against 20.4 with one; of 32 rows the registers
//    do not allow it, 64 rows 45 against 39); up to sixteen steps two of eight waves (8192 x 16, 16 rows 27.6 against 37, 64 rows
//    68 against 76), up to eight steps four (8192 x 8: 17.4 against 21.5 with two). Past 64 steps in phases, again 32 rows a
//    run (1875 x 80, 64 rows: 88 against 110), but from 33 to 64 sixteen, which need none (2000 x 64, 64 rows: 56 against 68).
int launch_w4(const W4Args& a, hipStream_t st) {
    const int steps = a.w.steps, runs16 = (a.rows + 15) / 16;
    const long cells = long(a.w.tiles) * runs16;
    if (cells <= 256 || (cells <= 1024 && cells * steps <= (steps > 64 ? 72000 : 17000))) {
        const int share = (a.rows + runs16 - 1) / runs16;
        const dim3 grid(over_xcds(a.w.tiles, runs16), unsigned(runs16));
        if (steps >= 64) w4_streamed_kernel<8, 2><<<grid, 512, 0, st>>>(a, share);
        else w4_streamed_kernel<8, 1><<<grid, 512, 0, st>>>(a, share);
        return launched();
    }
    const int runs = a.rows > 16 && (steps <= 32 || steps > 64) ? (a.rows + 31) / 32 : runs16, share = (a.rows + runs - 1) / runs;
    const int workgroups = runs < 256 ? 256 / runs : 1;
    if (share > 16) {
        if (steps <= 8) return launch_resident<2, 1, 8>(a, 4 * workgroups, share, st);
        if (steps <= 16) return launch_resident<2, 2, 8>(a, 2 * workgroups, share, st);
        if (steps <= 32) return launch_resident<2, 2, 16>(a, workgroups, share, st);
        return launch_resident<2, 2, 16, true>(a, workgroups, share, st);
    }
    if (steps <= 8) return launch_resident<1, 1, 8>(a, 4 * workgroups, share, st);
    if (steps <= 16) return launch_resident<1, 2, 8>(a, 2 * workgroups, share, st);
    if (steps <= 32) return launch_resident<1, 2, 16>(a, steps <= 24 ? 2 * workgroups : workgroups, share, st);
    if (steps <= 48) return launch_resident<1, 3, 16>(a, workgroups, share, st);
    if (steps <= 64) return launch_resident<1, 4, 16>(a, workgroups, share, st);
    const int threes = (steps + 47) / 48 * 3, fours = (steps + 63) / 64 * 4;  // steps a wave goes through
    if (threes < fours) return launch_resident<1, 3, 16, true>(a, workgroups, share, st);
    return launch_resident<1, 4, 16, true>(a, workgroups, share, st);
}

int w4_run(const m26c_w4* w, W4Args a, bool fp8, void* stream) {
    if (!w || a.rows < 0) return 1;
    if (a.rows == 0) return 0;
    int device = -1;
    if (hipGetDevice(&device) != hipSuccess || device != w->device) return 1;
    if (!a.y || a.y_pitch < w->lay.n || a.y_pitch > kPitchMost || !on(a.y, a.y_bf16 ? 2 : 4)) return 1;
    a.w = w->lay;
    a.fp8 = fp8;
    a.payload = w->payload;
    a.scales = w->scales;
    constexpr int kLaunchRows = 1 << 19;  // row runs are the grid's second dimension
    for (int left = a.rows;;) {
        a.rows = left < kLaunchRows ? left : kLaunchRows;
        if (int rc = launch_w4(a, hipStream_t(stream))) return rc;
        if ((left -= a.rows) == 0) return 0;
        if (fp8) {
            a.x_codes += long(kLaunchRows) * a.x_pitch;
            a.x_scales += long(kLaunchRows) * a.x_scales_pitch;
        } else {
            a.x += long(kLaunchRows) * a.x_pitch;
        }
        a.y = static_cast<char*>(a.y) + long(kLaunchRows) * a.y_pitch * (a.y_bf16 ? 2 : 4);
    }
}

}  // namespace

extern "C" {

int m26c_block_join(const m26c_join* plan, long rows, const float* h, const uint16_t* p0, const uint16_t* p1, const uint16_t* p2,
                    const uint16_t* p3, const float* gate, float* h_out, uint16_t* norm, uint8_t* payload, uint8_t* scales,
                    void* stream) {
    if (!plan || rows < 0) return 1;
    const m26c_join& p = *plan;
    const uint16_t* planes[4] = {p0, p1, p2, p3};
    if (p.cols <= 0 || p.cols > 16384 || p.planes < 1 || p.planes > 4 || p.plane_pitch < p.cols || p.h_pitch < p.cols ||
        !(p.eps > 0.0f) || !std::isfinite(p.eps) || !std::isfinite(p.scale) || (p.gate_cols != 0 && p.gate_cols != 1 && p.gate_cols != p.cols) ||
        (p.gate_cols && (p.gate_pitch < 0 || (p.gate_pitch && p.gate_pitch < p.gate_cols))))
        return 1;
    if (rows == 0) return 0;
    const bool normed = norm || payload;
    if (!h || (!h_out && !normed) || (normed && !p.pre_weight) || (p.gate_cols && !gate) || !payload != !scales ||
        (norm && p.norm_pitch < p.cols))
        return 1;
    if (payload && (p.cols % 32 || p.payload_pitch < size_t(p.cols) || p.scales_pitch < size_t(p.cols / 32))) return 1;
    if (!on(h, 4) || !on(h_out, 4) || !on(norm, 2) || !on(p.pre_weight, 4) || !on(p.post_weight, 4) || (p.gate_cols && !on(gate, 4))) return 1;
    for (int i = 0; i < p.planes; ++i)
        if (!planes[i] || !on(planes[i], 2)) return 1;
    JoinArgs a{};
    for (int i = 0; i < p.planes; ++i) a.plane[i] = planes[i];
    a.h = h; a.gate = gate; a.pre_w = p.pre_weight; a.post_w = p.post_weight;
    a.h_out = h_out; a.norm = norm; a.payload = payload; a.scales = scales;
    a.rows = rows; a.plane_pitch = p.plane_pitch; a.h_pitch = p.h_pitch; a.norm_pitch = p.norm_pitch; a.gate_pitch = p.gate_pitch;
    a.payload_pitch = p.payload_pitch; a.scales_pitch = p.scales_pitch;
    a.cols = p.cols; a.planes = p.planes; a.gate_cols = p.gate_cols; a.scale = p.scale; a.eps = p.eps;
    hipStream_t st = hipStream_t(stream);
    if (rows < 512) {  // few rows: as many threads to a row as it has groups
        if (p.cols <= 2048) launch_join<256, 1>(a, st);
        else if (p.cols <= 4096) launch_join<512, 1>(a, st);
        else if (p.cols <= 8192) launch_join<1024, 1>(a, st);
        else launch_join<1024, 2>(a, st);
    } else {
        if (p.cols <= 2048) launch_join<256, 1>(a, st);
        else if (p.cols <= 4096) launch_join<256, 2>(a, st);
        else if (p.cols <= 8192) launch_join<512, 2>(a, st);
        else launch_join<1024, 2>(a, st);
    }
    return launched();
}

int m26c_w4_new(const uint8_t* payload, const uint8_t* scales, long n, long k, void* stream, m26c_w4** out, char* err, size_t errlen) {
    if (!out) return fail(err, errlen, 1, "w4 weights: no place for the handle");
    *out = nullptr;
    if (!payload || !scales || n <= 0 || k <= 0 || k % 32 || n > kPitchMost || k > kPitchMost) return fail(err, errlen, 1, "w4 weights: bad pointers or sizes");
    if (!on(payload, 16)) return fail(err, errlen, 1, "w4 weights: the payload has to be 16-byte aligned");
    hipStream_t st = hipStream_t(stream);
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(st, &capture) != hipSuccess) (void)hipGetLastError();  // no device, say: what follows reports it
    if (capture != hipStreamCaptureStatusNone) return fail(err, errlen, 1, "w4 weights: the stream is being captured");
    m26c_w4* w = new (std::nothrow) m26c_w4{};
    if (!w) return fail(err, errlen, 2, "w4 weights: out of host memory");
    w->lay = W4Layout{n, k, int((n + 15) / 16), int((k + 127) / 128), int((k + 511) / 512)};
    const size_t payload_bytes = size_t(w->lay.tiles) * w->lay.steps * 1024, scale_bytes = size_t(w->lay.tiles) * w->lay.quads * 256;
    uint32_t* fault = nullptr;
    if (hipGetDevice(&w->device) != hipSuccess || hipMalloc(&w->payload, payload_bytes) != hipSuccess ||
        hipMalloc(&w->scales, scale_bytes + 256) != hipSuccess) {
        (void)hipGetLastError();
        release(w);
        return fail(err, errlen, 2, "w4 weights: device allocation failed");
    }
    fault = w->scales + scale_bytes / 4;  // one word behind the scales
    uint32_t seen = 0;
    const long cells = long(w->lay.tiles) * w->lay.quads * 256;
    const long blocks = (cells + 255) / 256;
    hipError_t e = hipMemcpyAsync(fault, &seen, 4, hipMemcpyHostToDevice, st);
    if (e == hipSuccess) {
        w4_prepare_kernel<<<unsigned(blocks < 65536 ? blocks : 65536), 256, 0, st>>>(payload, scales, w->lay, w->payload, reinterpret_cast<uint8_t*>(w->scales), fault);
        e = hipGetLastError();
    }
    if (e == hipSuccess) e = hipMemcpyAsync(&seen, fault, 4, hipMemcpyDeviceToHost, st);
    if (e == hipSuccess) e = hipStreamSynchronize(st);
    if (e != hipSuccess || seen) {
        (void)hipGetLastError();  // reported here, not by the next launch
        release(w);
        return e != hipSuccess ? fail(err, errlen, 2, hipGetErrorString(e))
                               : fail(err, errlen, 3, "w4 weights: a scale byte outside 2..252 over a nonzero code");
    }
    *out = w;
    return 0;
}

void m26c_w4_free(m26c_w4* w) { release(w); }

int m26c_w4_matvec(const m26c_w4* w, const uint16_t* x, long x_pitch, int rows, void* y, int y_bf16, long y_pitch, void* stream) {
    if (rows > 0 && (!w || !x || !on(x, 16) || x_pitch < w->lay.k || x_pitch > kPitchMost || x_pitch % 8)) return 1;
    W4Args a{};
    a.x = x; a.x_pitch = x_pitch; a.rows = rows; a.y = y; a.y_bf16 = y_bf16 != 0; a.y_pitch = y_pitch;
    return w4_run(w, a, false, stream);
}

int m26c_w4_matvec_fp8(const m26c_w4* w, const uint8_t* payload, size_t payload_pitch, const uint8_t* scales, size_t scales_pitch,
                       int rows, void* y, int y_bf16, long y_pitch, void* stream) {
    if (rows > 0 && (!w || !payload || !scales || !on(payload, 8) || payload_pitch % 8 || payload_pitch < size_t(w->lay.k) ||
                     scales_pitch < size_t(w->lay.k / 32) || payload_pitch > size_t(kPitchMost) || scales_pitch > size_t(kPitchMost)))
        return 1;
    W4Args a{};
    a.x_codes = payload; a.x_scales = scales; a.x_pitch = long(payload_pitch); a.x_scales_pitch = long(scales_pitch);
    a.rows = rows; a.y = y; a.y_bf16 = y_bf16 != 0; a.y_pitch = y_pitch;
    return w4_run(w, a, true, stream);
}

constexpr int kVocabMost = 1 << 30;           // ids past a row's end, up to a chunk of every part, still fit
constexpr float kScaleMost = float(1 << 20);  // a temperature of a millionth: scale * log2 e and ordinary logits times it stay finite

size_t m26c_token_logprobs_workspace(int rows, int vocab, int top) {
    if (rows <= 0 || vocab <= 0 || vocab > kVocabMost || top < 0 || top > kTopMost) return 0;
    const int parts = cut_of(rows, vocab).parts;
    return stats_bytes(rows, parts) + size_t(rows) * parts * top * 8;
}

int m26c_token_logprobs(const void* logits, int bf16, long pitch, int rows, int vocab, float scale, const int* given, int n_given,
                        float* given_logprob, float* entropy, int top, int* top_ids, float* top_logprob, void* workspace,
                        size_t workspace_bytes, void* stream) {
    if (rows < 0 || vocab <= 0 || vocab > kVocabMost || n_given < 0 || n_given > kVocabMost || top < 0 || top > kTopMost || top > vocab ||
        !(scale > 0.0f && scale <= kScaleMost) || pitch < vocab)
        return 1;
    if (rows == 0) return 0;
    if (!logits || !on(logits, bf16 ? 2 : 4) || (n_given && (!given || !given_logprob || !on(given, 4) || !on(given_logprob, 4))) || !on(entropy, 4) ||
        (top && (!top_ids || !top_logprob || !on(top_ids, 4) || !on(top_logprob, 4))))
        return 1;
    LogprobArgs a{};
    const LogprobCut cut = cut_of(rows, vocab);
    a.parts = cut.parts;
    const size_t need = m26c_token_logprobs_workspace(rows, vocab, top);
    if (need && (!workspace || !on(workspace, 16) || workspace_bytes < need)) return 1;
    a.logits = logits; a.pitch = pitch; a.rows = rows; a.vocab = vocab; a.scale = scale;
    a.given = given; a.n_given = n_given; a.given_logprob = given_logprob; a.entropy = entropy;
    a.top = top; a.top_ids = top_ids; a.top_logprob = top_logprob;
    if (need) {
        a.stats = static_cast<float4*>(workspace);
        a.lists = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + stats_bytes(rows, a.parts));
    }
    return bf16 ? launch_logprobs<true>(a, cut.chunks, hipStream_t(stream)) : launch_logprobs<false>(a, cut.chunks, hipStream_t(stream));
}

}  // extern "C"

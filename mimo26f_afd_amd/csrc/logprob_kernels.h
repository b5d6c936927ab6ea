// gfx950 kernels of the token log probabilities. Per row of logits l, with t = scale * l and m = max t, in one pass:
//
//   Z = sum exp(t - m),  S = sum exp(t - m) (t - m)
//   log p(j) = t_j - m - ln Z,   entropy = ln Z - S / Z,   the largest logits in descending order, equal ones by the lower id
//
// The logits are read once, which is the bound: everything else is a few values per row. About ten vector instructions a
// value, one of them an exponential of four times the cost, are 1.5 times what the chip does in the time HBM needs for a FP32
// value and close to it for BF16, so the selection may add next to nothing to the common path.
//
// Selection. A wave walks its part of the row in ascending order, 512 values at a time, with a threshold that at least
// `top` values already set aside reach. A value above the threshold is set aside in the wave's list; an equal one need not
// be: `top` values of at least its size with lower ids are there. One comparison of each lane's maximum, which the softmax needs
// anyway, and a scalar branch are the whole cost where nothing qualifies. A list that has grown is cut back to the
// exact `top` and raises the threshold, so that a list sees about top * ln(length / 512) values beyond the first.
// List entries are 64-bit keys, the value's bits in integer order above the complemented id: a total order, so the result does not
// depend on who finds what when.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>
#include "q0_codec.h"

namespace m26g {

constexpr int kTopMost = 32;        // alternatives a call may ask for
constexpr int kListCut = 128;       // a list longer than this is cut back to `top`
constexpr int kListCap = 640;       // entries of a wave's list: kListCut and a whole chunk, whatever it holds
constexpr int kLogprobWaves = 4;    // per workgroup
constexpr int kChunk = 512;         // values a wave takes at once
constexpr int kSegmentsMost = 64;   // a lane of the joining wave each
constexpr uint64_t kNoKey = 0;      // below every key of a number above -infinity

struct LogprobArgs {
    const void* logits;
    long pitch;
    int rows, vocab, segments;  // a row is cut into `segments` runs of whole chunks
    float scale;
    const int* given;
    int n_given;
    float *given_logprob, *entropy;
    int top;
    int* top_ids;
    float* top_logprob;
    float4* stats;    // [rows][segments] max logit, Z, S in units of log2, unused
    uint64_t* lists;  // [rows][segments][top], descending
};

// Bits of a value in the order of the integers; -0 counts as 0.
__device__ __forceinline__ uint32_t order_bits(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t o) { return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint64_t list_key(float v, int id) { return uint64_t(order_bits(v)) << 32 | uint32_t(~id); }
__device__ __forceinline__ int key_id(uint64_t key) { return int(~uint32_t(key)); }
__device__ __forceinline__ float key_value(uint64_t key) { return order_value(uint32_t(key >> 32)); }
__device__ __forceinline__ int lanes_below(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi(uint32_t(mask >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(mask), 0));
}

// Running sums of one lane, relative to its own maximum.
struct SoftmaxSums {
    float m = -INFINITY, z = 0.0f, s = 0.0f;  // s in units of log2
    // The sums relative to the maximum `to` (>= m). c = scale * log2(e). Without a number so far z and s are 0, or NaN.
    __device__ __forceinline__ SoftmaxSums at(float to, float c) const {
        const float d = m == to || m == -INFINITY ? 0.0f : (m - to) * c, f = __builtin_amdgcn_exp2f(d);
        return SoftmaxSums{to, f * z, f * (s + (d == -INFINITY ? 0.0f : d * z))};
    }
    __device__ __forceinline__ void add(float v, float c, float from) {  // from: m, or 0 where m is -infinity
        const float d = (v - from) * c, e = __builtin_amdgcn_exp2f(d);
        z += e;
        s += e * fmaxf(d, -300.0f);  // a masked value adds 0, not 0 * infinity
    }
    __device__ __forceinline__ void join(const SoftmaxSums& o, float c) {
        const float to = fmaxf(m, o.m);
        const SoftmaxSums p = at(to, c), r = o.at(to, c);
        m = to;
        z = p.z + r.z;
        s = p.s + r.s;
    }
    __device__ __forceinline__ void join_lanes(float c) {  // over the wave, in a fixed order, the same in every lane
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            join(SoftmaxSums{__shfl_xor(m, d), __shfl_xor(z, d), __shfl_xor(s, d)}, c);
        }
    }
};

// One wave's list, in LDS.
struct TopList {
    uint64_t* entries;  // [kListCap]
    int count;          // uniform
    float threshold;    // uniform; -infinity until `top` values are known
};

// Cuts a list of `count` distinct keys down to its `top` largest, in no order, and returns the smallest of them. The value
// of the top-th largest is found bit by bit with counts over the wave, then, where equal values straddle the cut, the
// id in the same way.
template <int R>  // at most 64 * R entries
__device__ __forceinline__ uint64_t cut_list_of(uint64_t* entries, int count, int top) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // other lanes of this wave wrote the entries
    const int lane = threadIdx.x & 63;
    uint64_t key[R];
#pragma unroll
    for (int i = 0; i < R; ++i) key[i] = 64 * i + lane < count ? entries[64 * i + lane] : kNoKey;
    auto at_least = [&](uint64_t k) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) n += __popcll(__ballot(key[i] >= k));
        return n;
    };
    uint64_t cut = 0;  // the largest key that at least `top` entries reach
    for (int bit = 63; bit >= 32; --bit)
        if (at_least(cut | 1ull << bit) >= top) cut |= 1ull << bit;
    if (at_least(cut) > top)
        for (int bit = 31; bit >= 0; --bit)
            if (at_least(cut | 1ull << bit) >= top) cut |= 1ull << bit;
    int at = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const bool keep = key[i] >= cut && key[i] != kNoKey;
        const uint64_t mask = __ballot(keep);
        if (keep) entries[at + lanes_below(mask)] = key[i];
        at += __popcll(mask);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    return cut;
}
__device__ __forceinline__ uint64_t cut_list(uint64_t* entries, int count, int top) {
    return count <= 192 ? cut_list_of<3>(entries, count, top) : cut_list_of<kListCap / 64>(entries, count, top);
}

// The top-th largest of the lanes' values: at least `top` lanes reach it.
__device__ __forceinline__ float top_of_lanes(float v, int top) {
    const uint32_t mine = order_bits(v);
    uint32_t cut = 0;
    for (int bit = 31; bit >= 0; --bit)
        if (int(__popcll(__ballot(mine >= (cut | 1u << bit)))) >= top) cut |= 1u << bit;
    return order_value(cut);
}

// The slow path of a chunk: sets aside what may be among the `top` largest. Element j of the lane has id `id` + j.
__device__ __forceinline__ void set_aside(TopList& list, const float (&v)[8], int id, int top) {
    int n = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) n += __popcll(__ballot(v[j] > list.threshold));
    if (n <= 64) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool mine = v[j] > list.threshold;
            const uint64_t mask = __ballot(mine);
            if (mine) list.entries[list.count + lanes_below(mask)] = list_key(v[j], id + j);
            list.count += __popcll(mask);
        }
    } else {
        // Many at once, as in the first chunk: the top-th largest of the lanes' maxima is a bound that fewer than `top`
        // lanes exceed. Of the values equal to it the first `top` in order suffice.
        float most = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = v[j] > most ? v[j] : most;  // a NaN takes no part
        const float bound = top_of_lanes(most, top);
        const bool raised = bound > list.threshold;  // otherwise fewer than `top` lanes hold anything above the threshold
        const float over = raised ? bound : list.threshold;
        int equals = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) equals += raised && v[j] == over;
        int before = equals;  // equals in the lanes below
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int o = __shfl_up(before, d);
            if (int(threadIdx.x & 63) >= d) before += o;
        }
        before -= equals;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool same = raised && v[j] == over;
            const bool mine = v[j] > over || (same && before < top);
            before += same;
            const uint64_t mask = __ballot(mine);
            if (mine) list.entries[list.count + lanes_below(mask)] = list_key(v[j], id + j);
            list.count += __popcll(mask);
        }
        list.threshold = over;
    }
    if (list.count > kListCut) {
        list.threshold = key_value(cut_list(list.entries, list.count, top));
        list.count = top;
    }
}

// Orders `count` distinct keys by counting, for each, the larger ones: position p of the result goes to `put(p, key)` for p < top.
// All `threads` threads of the caller's group take part.
template <typename F>
__device__ __forceinline__ void rank_keys(const uint64_t* keys, int count, int top, int tid, int threads, F&& put) {
    for (int i = tid; i < count; i += threads) {
        const uint64_t k = keys[i];
        int larger = 0;
        for (int j = 0; j < count; ++j) larger += keys[j] > k;
        if (larger < top) put(larger, k);
    }
}

// What a row's sums and ordered keys give.
template <bool BF16>
__device__ __forceinline__ void write_row(const LogprobArgs& a, long row, SoftmaxSums sum, const uint64_t* keys, int count, int tid, int threads) {
    const bool empty = sum.m == -INFINITY && sum.z == 0.0f;
    const float ln_z = logf(sum.z);
    auto logprob = [&](float v) { return (v - sum.m) * a.scale - ln_z; };
    if (tid == 0 && a.entropy) a.entropy[row] = empty ? 0.0f : ln_z - 0.69314718055994531f * (sum.s / sum.z);
    for (int i = tid; i < a.n_given; i += threads) {
        const int id = a.given[row * a.n_given + i];
        float lp = __builtin_nanf("");
        if (id >= 0 && id < a.vocab) {
            const long at = row * a.pitch + id;
            const float v = BF16 ? __uint_as_float(uint32_t(static_cast<const uint16_t*>(a.logits)[at]) << 16) : static_cast<const float*>(a.logits)[at];
            lp = empty ? -INFINITY : logprob(v);
        }
        a.given_logprob[row * a.n_given + i] = lp;
    }
    rank_keys(keys, count, a.top, tid, threads, [&](int p, uint64_t k) {
        a.top_ids[row * a.top + p] = key_id(k);
        a.top_logprob[row * a.top + p] = logprob(key_value(k));
    });
    for (int p = count + tid; p < a.top; p += threads) {
        a.top_ids[row * a.top + p] = -1;
        a.top_logprob[row * a.top + p] = -INFINITY;
    }
}

// One workgroup per (row, segment). Rows start anywhere: up to 15 bytes ahead of the first 16-byte boundary and what is left
// behind the last whole group of eight values are taken as chunks of their own by the wave that is first or last.
template <bool BF16>
__global__ void __launch_bounds__(64 * kLogprobWaves) logprob_kernel(const LogprobArgs a) {
    __shared__ uint64_t lists[kLogprobWaves][kListCap];
    __shared__ float wave_m[kLogprobWaves], wave_z[kLogprobWaves], wave_s[kLogprobWaves];
    __shared__ int counts[kLogprobWaves];
    __shared__ uint64_t merged[kLogprobWaves * kTopMost];
    typedef typename std::conditional<BF16, uint16_t, float>::type T;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long row = blockIdx.x / a.segments;
    const int segment = int(blockIdx.x % a.segments);
    const T* base = static_cast<const T*>(a.logits) + row * a.pitch;
    const int off = int((16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15) / int(sizeof(T));
    const int head = off < a.vocab ? off : a.vocab, groups = (a.vocab - head) / 8, tail = a.vocab - head - 8 * groups;
    const int chunks = (groups + 63) / 64;
    // this wave's run of chunks
    const long parts = long(a.segments) * kLogprobWaves, part = long(segment) * kLogprobWaves + wave;
    const int from = int(chunks * part / parts), to = int(chunks * (part + 1) / parts);
    const float c = a.scale * 1.44269504088896341f;

    SoftmaxSums sum;
    TopList list{lists[wave], 0, -INFINITY};
    auto take = [&](const float (&v)[8], int id) {
        float most = v[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) most = fmaxf(most, v[j]);
        if (__any(most > sum.m))
            sum = sum.at(fmaxf(most, sum.m), c);
        const float m = sum.m == -INFINITY ? 0.0f : sum.m;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum.add(v[j], c, m);
        if (a.top && __any(most > list.threshold)) set_aside(list, v, id, a.top);
    };
    auto value = [&](int i) -> float {
        if constexpr (BF16) return __uint_as_float(uint32_t(base[i]) << 16);
        else return base[i];
    };
    auto single = [&](int first, int n) {  // n < 64 values, one to a lane
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = -INFINITY;
        if (lane < n) v[0] = value(first + lane);
        take(v, first + lane);
    };
    if (part == 0 && head) single(0, head);
    for (int chunk = from; chunk < to; ++chunk) {
        const int g = chunk * 64 + lane;
        float v[8];
        if (g < groups) {
            const T* p = base + head + 8 * long(g);
            if constexpr (BF16) {
                const uint4 w = *reinterpret_cast<const uint4*>(p);
                const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) { v[2 * j] = __uint_as_float(d[j] << 16); v[2 * j + 1] = __uint_as_float(d[j] & 0xffff0000u); }
            } else {
                const float4 lo = *reinterpret_cast<const float4*>(p), hi = *reinterpret_cast<const float4*>(p + 4);
                v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w; v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = -INFINITY;
        }
        take(v, head + 8 * g);
    }
    if (part == parts - 1 && tail) single(head + 8 * groups, tail);

    sum.join_lanes(c);
    if (a.top && list.count > a.top) {
        cut_list(list.entries, list.count, a.top);
        list.count = a.top;
    }
    if (lane == 0) {
        wave_m[wave] = sum.m;
        wave_z[wave] = sum.z;
        wave_s[wave] = sum.s;
        counts[wave] = list.count;
    }
    __syncthreads();
    sum = SoftmaxSums{wave_m[0], wave_z[0], wave_s[0]};
#pragma unroll
    for (int w = 1; w < kLogprobWaves; ++w) sum.join(SoftmaxSums{wave_m[w], wave_z[w], wave_s[w]}, c);
    int first = 0;
    for (int w = 0; w < wave; ++w) first += counts[w];
    for (int i = lane; i < counts[wave]; i += 64) merged[first + i] = lists[wave][i];
    int count = 0;
    for (int w = 0; w < kLogprobWaves; ++w) count += counts[w];
    __syncthreads();
    if (a.segments == 1) {
        write_row<BF16>(a, row, sum, merged, count, threadIdx.x, 64 * kLogprobWaves);
        return;
    }
    const long cell = row * a.segments + segment;
    if (threadIdx.x == 0) a.stats[cell] = make_float4(sum.m, sum.z, sum.s, 0.0f);
    uint64_t* mine = a.lists + cell * a.top;
    rank_keys(merged, count, a.top, threadIdx.x, 64 * kLogprobWaves, [&](int p, uint64_t k) { mine[p] = k; });
    for (int p = count + threadIdx.x; p < a.top; p += 64 * kLogprobWaves) mine[p] = kNoKey;
}

// Joins a row's segments. Their lists are ordered, so the largest of their last keys is a bound that `top` keys reach, and few others.
template <bool BF16>
__global__ void __launch_bounds__(256) logprob_join_kernel(const LogprobArgs a) {
    extern __shared__ uint64_t keys[];  // [segments * top]
    __shared__ unsigned long long bound;
    __shared__ int count;
    const long row = blockIdx.x;
    const float c = a.scale * 1.44269504088896341f;
    SoftmaxSums sum;  // a lane per segment, each wave for itself
    if (int(threadIdx.x & 63) < a.segments) {
        const float4 p = a.stats[row * a.segments + (threadIdx.x & 63)];
        sum = SoftmaxSums{p.x, p.y, p.z};
    }
    sum.join_lanes(c);
    if (threadIdx.x == 0) { bound = 0; count = 0; }
    __syncthreads();
    const uint64_t* lists = a.lists + row * a.segments * a.top;
    if (a.top)
        for (int s = threadIdx.x; s < a.segments; s += 256) atomicMax(&bound, (unsigned long long)lists[s * a.top + a.top - 1]);
    __syncthreads();
    for (int i = threadIdx.x; i < a.segments * a.top; i += 256) {
        const uint64_t k = lists[i];
        if (k != kNoKey && k >= bound) keys[atomicAdd(&count, 1)] = k;
    }
    __syncthreads();
    write_row<BF16>(a, row, sum, keys, count, threadIdx.x, 256);
}

}  // namespace m26g

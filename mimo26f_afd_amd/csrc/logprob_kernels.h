// gfx950 kernels of the token log probabilities. Per row of logits l, with t = scale * l and m = max t, in one pass:
//
//   Z = sum exp(t - m),  S = sum exp(t - m) (t - m)
//   log p(j) = t_j - m - ln Z,   entropy = ln Z - S / Z,   the largest logits in descending order, equal ones by the lower id
//
// The logits are read once, which is the bound: everything else is a few values per row. About nine vector instructions a
// value (one of them an exponential) are four fifths of what the chip does in the time HBM needs for a BF16 value, so the
// selection may add next to nothing to the common path.
//
// Selection. A wave keeps its part's largest values in order, one to a lane, and walks the part in ascending order, 512 values
// at a time, with the top-th of them as a threshold. A value above it is put in its place with one comparison and one shift
// over the lanes; an equal one need not be: `top` values of its size with lower ids are there. One comparison of each
// lane's maximum, which the softmax needs anyway, and a scalar branch are the whole cost where nothing qualifies, which after i
// chunks is all but top / i of them. The waves of a workgroup help each other: what each wave's (top / waves)-th value
// reaches is a bound that `top` values of the row reach. List entries are 64-bit keys, the value's bits in integer order above the
// complemented id: a total order, so the result does not depend on who finds what when.
//
// A row is cut into parts, a wave each, whose chunks lie side by side. The parts' lists meet in one workgroup: their keys in
// 128 groups, the top-th largest of the groups' maxima is a bound that `top` keys reach and few others, and what reaches it is
// ordered by counting.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>
#include "q0_codec.h"

namespace m26g {

constexpr int kTopMost = 32;       // alternatives a call may ask for
constexpr int kChunk = 512;        // values a wave takes at once
constexpr int kPartsMost = 128;    // of a row: two to a lane of the wave that joins them
constexpr uint64_t kNoKey = 0;     // below every key of a number above -infinity

struct LogprobArgs {
    const void* logits;
    long pitch;
    int rows, vocab, parts;  // a row is cut into `parts` runs of whole chunks
    float scale;
    const int* given;
    int n_given;
    float *given_logprob, *entropy;
    int top;
    int* top_ids;
    float* top_logprob;
    float4* stats;    // [rows][parts] max logit, Z, S in units of log2
    uint64_t* lists;  // [rows][parts][top]
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
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint64_t o = uint64_t(__shfl_xor(uint32_t(v >> 32), d)) << 32 | __shfl_xor(uint32_t(v), d);
        v = o > v ? o : v;
    }
    return v;
}

// Running sums of 2^(v c - r), c = scale * log2 e, and of that times its exponent, relative to r = m c rounded to FP32, m the
// largest value so far: the exponent is then one fused multiply-add, rounded once, and r, the same number everywhere, comes
// out again at the end. Values so large that m c may pass FP32's range (masks of the type's lowest value in a row of nothing
// else) are measured from m itself, (v - m) c.
struct SoftmaxSums {
    float m = -INFINITY, z = 0.0f, s = 0.0f;

    __device__ __forceinline__ static bool far(float m) { return fabsf(m) > 1e30f && m != -INFINITY; }
    __device__ __forceinline__ static float distance(float v, float m, float c) {
        return far(m) ? (v - m) * c : __builtin_fmaf(v, c, m == -INFINITY ? 0.0f : -(m * c));
    }
    // The sums relative to the maximum `to` (>= m). Without a number so far z and s are 0, or NaN.
    __device__ __forceinline__ SoftmaxSums at(float to, float c) const {
        const float d = m == to || m == -INFINITY ? 0.0f : far(m) || far(to) ? (m - to) * c : m * c - to * c, f = __builtin_amdgcn_exp2f(d);
        return SoftmaxSums{to, f * z, f * (s + (d == -INFINITY ? 0.0f : d * z))};
    }
    __device__ __forceinline__ void join(const SoftmaxSums& o, float c) {
        const float to = fmaxf(m, o.m);
        const SoftmaxSums p = at(to, c), r = o.at(to, c);
        m = to;
        z = p.z + r.z;
        s = p.s + r.s;
    }
    __device__ __forceinline__ void add(float d) {  // d: the value's distance
        const float e = __builtin_amdgcn_exp2f(d);
        z += e;
        s = __builtin_fmaf(e, fmaxf(d, -300.0f), s);  // a masked value adds 0, not 0 * infinity
    }
    __device__ __forceinline__ void join_lanes(float c) {  // over the wave, in a fixed order, the same in every lane
#pragma unroll
        for (int d = 1; d < 64; d *= 2) join(SoftmaxSums{__shfl_xor(m, d), __shfl_xor(z, d), __shfl_xor(s, d)}, c);
    }
};

// The largest 32-bit number that at least `top` of the wave's N numbers a lane reach, as far as its upper BITS bits go (lower
// ones 0); 0 if there are fewer. Two bits at a time, with counts over the wave.
template <int BITS, int N>
__device__ __forceinline__ uint32_t reached_by(const uint32_t (&v)[N], int top) {
    uint32_t cut = 0;
    for (int bit = 30; bit >= 32 - BITS; bit -= 2) {
        const uint32_t k1 = cut | 1u << bit, k2 = cut | 2u << bit, k3 = cut | 3u << bit;
        int n1 = 0, n2 = 0, n3 = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            n1 += int(__popcll(__ballot(v[i] >= k1)));
            n2 += int(__popcll(__ballot(v[i] >= k2)));
            n3 += int(__popcll(__ballot(v[i] >= k3)));
        }
        cut = n3 >= top ? k3 : n2 >= top ? k2 : n1 >= top ? k1 : cut;
    }
    return cut;
}

// A wave's largest keys in descending order, lane i the i-th; kNoKey where there are fewer.
template <int WAVES>
struct TopList {
    float* shared;  // LDS, one of each wave of the workgroup: its share-th largest value
    int top, share, wave;
    uint64_t key = kNoKey;
    uint64_t floor = kNoKey;       // uniform: a key has to be above this one to matter
    float threshold = -INFINITY;   // uniform: a value of a later chunk has to be above this one

    __device__ __forceinline__ uint64_t of_lane(uint64_t k, int lane) const {
        return uint64_t(__builtin_amdgcn_readlane(uint32_t(k >> 32), lane)) << 32 | uint32_t(__builtin_amdgcn_readlane(uint32_t(k), lane));
    }
    __device__ __forceinline__ void insert(uint64_t k) {  // k uniform and new
        const bool above = key > k;
        const uint64_t mask = __ballot(above);  // the first lanes
        const uint32_t hi = uint32_t(key >> 32), lo = uint32_t(key);
        const uint64_t moved = uint64_t(__builtin_amdgcn_update_dpp(0u, hi, 0x138, 0xf, 0xf, false)) << 32 |  // wave_shr:1
                               uint32_t(__builtin_amdgcn_update_dpp(0u, lo, 0x138, 0xf, 0xf, false));
        const int place = int(__popcll(mask));
        key = above ? key : int(threadIdx.x & 63) == place ? k : moved;
    }
    // The floor and the threshold from this list's top-th key and from what the waves have in common.
    __device__ __forceinline__ void settle() {
        const uint64_t last = of_lane(key, top - 1);
        floor = last > floor ? last : floor;
        if (last != kNoKey) threshold = fmaxf(threshold, key_value(last));
    }
    __device__ __forceinline__ void common() {
        if constexpr (WAVES > 1) {
            const int lane = threadIdx.x & 63;
            float v = __hip_atomic_load(&shared[lane % WAVES], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
#pragma unroll
            for (int d = 1; d < WAVES; d *= 2) v = fminf(v, __shfl_xor(v, d));
            const uint32_t bound = __builtin_amdgcn_readfirstlane(order_bits(v));
            // `top` values reach v, at any ids: equal ones still count
            if (uint64_t(bound) << 32 > floor && v > -INFINITY) {
                floor = (uint64_t(bound) << 32) - 1;
                // the next number below it; below zero's bits lie those of -0, which no value has
                threshold = fmaxf(threshold, order_value(bound - (bound == 0x80000000u ? 2 : 1)));
            }
        }
    }
    // The slow path of a chunk. Element j of the lane has id `id` + j.
    __device__ __forceinline__ void take(const float (&v)[8], int id) {
        common();
        if (of_lane(key, top - 1) == kNoKey) {
            // Not `top` values yet: the top-th largest of the lanes' maxima is a bound that `top` values of this chunk reach.
            float most = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) most = v[j] > most ? v[j] : most;  // a NaN takes no part
            const uint32_t mine[1] = {order_bits(most)};
            const uint32_t bound = reached_by<16>(mine, top);
            if (bound > order_bits(-INFINITY) && uint64_t(bound) << 32 > floor) floor = (uint64_t(bound) << 32) - 1;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint64_t k = list_key(v[j], id + j);
            const bool number = v[j] > -INFINITY;
            for (uint64_t mask = __ballot(number && k > floor); mask;) {
                const int lane = __ffsll(static_cast<unsigned long long>(mask)) - 1;
                insert(of_lane(k, lane));
                settle();
                mask &= mask - 1;
                mask &= __ballot(k > floor);
            }
        }
        if constexpr (WAVES > 1) {
            const uint64_t mine = of_lane(key, share - 1);
            if (mine != kNoKey && (threadIdx.x & 63) == 0) __hip_atomic_store(&shared[wave], key_value(mine), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
    }
};

// One wave's part of a row, every parts-th chunk of it: its sums, the same in every lane, and its list. Rows start anywhere: the
// first part also takes the up to seven values ahead of the first 16-byte boundary, the last part what is behind the last whole
// chunk.
template <bool BF16>
struct RowPart {
    typedef typename std::conditional<BF16, uint16_t, float>::type T;
    static constexpr int kLoads = BF16 ? 1 : 2;  // 16-byte loads of a lane's eight values
    typedef uint32_t v4 __attribute__((ext_vector_type(4)));
    struct Raw {
        v4 part[kLoads];
    };

    const T* base;
    int vocab, head, chunks, part, parts;

    __device__ __forceinline__ RowPart(const LogprobArgs& a, long row, int part_, int parts_) : part(part_), parts(parts_) {
        base = static_cast<const T*>(a.logits) + row * a.pitch;
        vocab = a.vocab;
        const int off = int((16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15) / int(sizeof(T));
        head = off < vocab ? off : vocab;
        chunks = (vocab - head) / kChunk;  // whole ones
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (BF16) return __uint_as_float(uint32_t(base[i]) << 16);
        else return base[i];
    }
    __device__ __forceinline__ Raw load(int chunk) const {  // chunk < chunks
        const v4* p = reinterpret_cast<const v4*>(base + head + long(chunk) * kChunk) + (threadIdx.x & 63) * kLoads;
        Raw r;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) r.part[i] = __builtin_nontemporal_load(p + i);
        return r;
    }
    __device__ __forceinline__ static void widen(const Raw& r, float (&v)[8]) {
        if constexpr (BF16) {
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[2 * j] = __uint_as_float(r.part[0][j] << 16); v[2 * j + 1] = __uint_as_float(r.part[0][j] & 0xffff0000u); }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r.part[j / 4][j % 4]);
        }
    }

    template <typename LIST>
    __device__ __forceinline__ void walk(const LogprobArgs& a, SoftmaxSums& sum, LIST& list) const {
        const int lane = threadIdx.x & 63;
        const float c = a.scale * 1.44269504088896341f;
        // The hardware's maximum passes a signalling NaN on, quieted, and loses what it was compared with. A part whose sum turns
        // out to be no number is therefore gone through once more for its list, with comparisons.
        for (bool careful = false;; careful = true) {
            bool far = false;  // uniform
            auto take = [&](const float (&v)[8], int id) {
                float most = v[0];
                if (careful) {
                    most = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 8; ++j) most = v[j] > most ? v[j] : most;
                } else {
#pragma unroll
                    for (int j = 1; j < 8; ++j) most = fmaxf(most, v[j]);
                    if (__any(most > sum.m)) {
                        sum = sum.at(fmaxf(most, sum.m), c);
                        far = __any(SoftmaxSums::far(sum.m));
                    }
                    if (far) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) sum.add(SoftmaxSums::distance(v[j], sum.m, c));
                    } else {
                        const float r = sum.m == -INFINITY ? 0.0f : -(sum.m * c);
#pragma unroll
                        for (int j = 0; j < 8; ++j) sum.add(__builtin_fmaf(v[j], c, r));
                    }
                }
                if (a.top && __any(most > list.threshold)) list.take(v, id);
            };
            // Chunk -1 stands for the values ahead of the boundary, chunk `chunks` for those behind the last whole one. Two chunks
            // are in flight ahead of the one that is worked on; past the end the last one is asked for again.
            const int done = head + chunks * kChunk, end = chunks + (done < vocab && part == parts - 1);
            Raw now{}, next{};
            if (part < chunks) {
                now = load(part);
                next = load(part + parts < chunks ? part + parts : part);
            }
            for (int chunk = part == 0 && head ? -1 : part < chunks ? part : chunks; chunk < end;) {
                float v[8];
                int id;
                if (unsigned(chunk) < unsigned(chunks)) {
                    const Raw ahead = load(chunk + 2 * parts < chunks ? chunk + 2 * parts : chunk);
                    widen(now, v);
                    id = head + chunk * kChunk + lane * 8;
                    now = next;
                    next = ahead;
                } else {
                    id = (chunk < 0 ? 0 : done) + lane * 8;
                    const int stop = chunk < 0 ? head : vocab;  // up to seven values, or under a chunk
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = id + j < stop ? value(id + j) : -INFINITY;
                }
                take(v, id);
                // the last part comes by `chunks` whatever its own stride
                chunk = chunk < 0 ? part : chunk < chunks && chunk + parts >= chunks && end > chunks ? chunks : chunk + parts;
            }
            if (careful || !a.top || !__any(sum.z != sum.z)) break;
            list.key = list.floor = kNoKey;
            list.threshold = -INFINITY;
        }
        sum.join_lanes(c);
    }
};

// What a workgroup of THREADS makes of a row's joined sums and the parts' keys: N a thread, kNoKey for none. Every thread of
// the workgroup comes here.
constexpr int kRoom = 256, kGroups = 128;
struct RowShared {
    uint64_t room[kRoom];
    uint32_t most[kGroups];
    int count, reached[64];
    float share[16];  // of the waves' lists
};
template <bool BF16, int THREADS, int N>
__device__ __forceinline__ void write_row(const LogprobArgs& a, long row, const SoftmaxSums& sum, const uint64_t (&key)[N], RowShared& sh) {
    const int tid = threadIdx.x, lane = tid & 63;
    const float c = a.scale * 1.44269504088896341f, log_z = log2f(sum.z);
    constexpr float kLn2 = 0.69314718055994531f;
    const bool empty = sum.m == -INFINITY && sum.z == 0.0f;
    // Z is relative to 2^r, r = m c rounded: what r is short of m c is exactly a fused product
    const float ln_z = kLn2 * (SoftmaxSums::far(sum.m) || sum.m == -INFINITY ? log_z : log_z - __builtin_fmaf(sum.m, c, -(sum.m * c)));
    auto logprob = [&](float v) { return (v - sum.m) * a.scale - ln_z; };
    if (tid == 0 && a.entropy) a.entropy[row] = empty ? 0.0f : kLn2 * (log_z - sum.s / sum.z);
    for (int i = tid; i < a.n_given; i += THREADS) {
        const int id = a.given[row * a.n_given + i];
        float lp = __builtin_nanf("");
        if (id >= 0 && id < a.vocab) {
            const long at = row * a.pitch + id;
            const float v = BF16 ? __uint_as_float(uint32_t(static_cast<const uint16_t*>(a.logits)[at]) << 16) : static_cast<const float*>(a.logits)[at];
            lp = empty ? -INFINITY : logprob(v);
        }
        a.given_logprob[row * a.n_given + i] = lp;
    }
    if (!a.top) return;
    // The bound: values alone, from the maxima of kGroups groups of threads (all of a wave's where there are fewer threads).
    constexpr int kLanes = THREADS > kGroups ? THREADS / kGroups : 1;  // of a group
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) most = uint32_t(key[i] >> 32) > most ? uint32_t(key[i] >> 32) : most;
#pragma unroll
    for (int d = 1; d < kLanes; d *= 2) {
        const uint32_t o = __shfl_xor(most, d);
        most = o > most ? o : most;
    }
    if (tid % kLanes == 0) sh.most[tid / kLanes] = most;
    if (THREADS < kGroups && tid < kGroups - THREADS) sh.most[THREADS + tid] = 0;
    if (tid < 64) sh.reached[tid] = 0;
    if (tid == 64 % THREADS) sh.count = 0;
    __syncthreads();
    const uint32_t two[2] = {sh.most[lane], sh.most[64 + lane]};
    uint64_t bound = uint64_t(reached_by<32>(two, a.top)) << 32;
    auto reach = [&](uint64_t k) {  // keys of this wave that reach k
        int n = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) n += int(__popcll(__ballot(key[i] != kNoKey && key[i] >= k)));
        return n;
    };
    const int here = reach(bound);
    int at = 0;
    if (here && lane == 0) at = atomicAdd(&sh.count, here);  // a key's place in the result does not depend on which wave is first
    at = __builtin_amdgcn_readfirstlane(at);
    __syncthreads();
    int count = sh.count;
    if (count > kRoom) {  // many equal values, or lists that each hold all but one of the largest: the exact cut, bit by bit
        bound = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const int n = reach(bound | 1ull << bit);
            if (n && lane == 0) atomicAdd(&sh.reached[bit], n);
            __syncthreads();
            if (sh.reached[bit] >= a.top) bound |= 1ull << bit;
        }
        if (tid == 0) sh.count = 0;
        __syncthreads();
        const int exact = reach(bound);
        if (exact && lane == 0) at = atomicAdd(&sh.count, exact);
        at = __builtin_amdgcn_readfirstlane(at);
        __syncthreads();
        count = sh.count;  // `top`, or all there are
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool kept = key[i] != kNoKey && key[i] >= bound;
        const uint64_t mask = __ballot(kept);
        if (kept) sh.room[at + lanes_below(mask)] = key[i];
        at += int(__popcll(mask));
    }
    __syncthreads();
    // a key's place is the number of larger ones
    for (int i = tid; i < count; i += THREADS) {
        const uint64_t k = sh.room[i];
        int larger = 0, j = 0;
        for (; j + 8 <= count; j += 8)
#pragma unroll
            for (int u = 0; u < 8; ++u) larger += sh.room[j + u] > k;
        for (; j < count; ++j) larger += sh.room[j] > k;
        if (larger < a.top) {
            a.top_ids[row * a.top + larger] = key_id(k);
            a.top_logprob[row * a.top + larger] = logprob(key_value(k));
        }
    }
    for (int p = count + tid; p < a.top; p += THREADS) {
        a.top_ids[row * a.top + p] = -1;
        a.top_logprob[row * a.top + p] = -INFINITY;
    }
}

template <int WAVES>
__device__ __forceinline__ TopList<WAVES> empty_list(float* shared, int top) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (WAVES > 1) {
        if (threadIdx.x < WAVES) shared[threadIdx.x] = -INFINITY;
        __syncthreads();
    }
    return TopList<WAVES>{shared, top, (top + WAVES - 1) / WAVES, wave};
}

// A workgroup per row, a part for each of its WAVES waves.
template <bool BF16, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) logprob_row_kernel(const LogprobArgs a) {
    __shared__ float4 sums[WAVES];
    __shared__ RowShared shared;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    SoftmaxSums sum;
    TopList<WAVES> list = empty_list<WAVES>(shared.share, a.top);
    RowPart<BF16>(a, blockIdx.x, wave, WAVES).walk(a, sum, list);
    if (lane == 0) sums[wave] = make_float4(sum.m, sum.z, sum.s, 0.0f);
    __syncthreads();
    const float c = a.scale * 1.44269504088896341f;
    sum = SoftmaxSums{};
    if (lane < WAVES) sum = SoftmaxSums{sums[lane].x, sums[lane].y, sums[lane].z};
    sum.join_lanes(c);
    const uint64_t key[1] = {lane < a.top ? list.key : kNoKey};
    write_row<BF16, 64 * WAVES>(a, blockIdx.x, sum, key, shared);
}

// A row over several workgroups: each wave leaves its part's sums and list in memory ...
constexpr int kPartWaves = 4;
template <bool BF16>
__global__ void __launch_bounds__(64 * kPartWaves) logprob_part_kernel(const LogprobArgs a) {
    __shared__ float shared[kPartWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long cell = long(blockIdx.x) * kPartWaves + wave;  // parts is a multiple of kPartWaves: a workgroup is of one row
    SoftmaxSums sum;
    TopList<kPartWaves> list = empty_list<kPartWaves>(shared, a.top);
    RowPart<BF16>(a, cell / a.parts, int(cell % a.parts), a.parts).walk(a, sum, list);
    if (lane == 0) a.stats[cell] = make_float4(sum.m, sum.z, sum.s, 0.0f);
    if (lane < a.top) a.lists[cell * a.top + lane] = list.key;
}

// ... and a workgroup per row joins them, everything it reads asked for at once.
template <bool BF16>
__global__ void __launch_bounds__(1024) logprob_join_kernel(const LogprobArgs a) {
    constexpr int N = kPartsMost * kTopMost / 1024;
    __shared__ RowShared shared;
    const int lane = threadIdx.x & 63;
    const long row = blockIdx.x;
    const float c = a.scale * 1.44269504088896341f;
    const float4* stats = a.stats + row * a.parts;
    const uint64_t* lists = a.lists + row * a.parts * a.top;
    float4 two[2];
    uint64_t key[N];
#pragma unroll
    for (int i = 0; i < 2; ++i) two[i] = lane + 64 * i < a.parts ? stats[lane + 64 * i] : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int at = int(threadIdx.x) + 1024 * i;
        key[i] = at < a.parts * a.top ? lists[at] : kNoKey;
    }
    SoftmaxSums sum{two[0].x, two[0].y, two[0].z};
    sum.join(SoftmaxSums{two[1].x, two[1].y, two[1].z}, c);
    sum.join_lanes(c);
    write_row<BF16, 1024>(a, row, sum, key, shared);
}

}  // namespace m26g

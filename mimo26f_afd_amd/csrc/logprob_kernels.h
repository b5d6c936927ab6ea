// gfx950 kernels of the token log probabilities. Per row of logits l, with t = scale * l and m = max t, in one pass:
//
//   Z = sum exp(t - m),  S = sum exp(t - m) (t - m)
//   log p(j) = t_j - m - ln Z,   entropy = ln Z - S / Z,   the largest logits in descending order, equal ones by the lower id
//
// The logits are read once, which is the bound of large calls: everything else is a few values per row. The vector instructions
// (10.9 a BF16 value counted, one of them an exponential) keep their pipe busy 78 % of the counted cycles of such a call,
// so the selection may add next to nothing to the common path: 2048 rows x 131072 BF16, top 5, 537 MB in 98 us (5.5
// TB/s, 82 % of a streaming read). Small calls are chains of dependent steps: 1 row x 131072 9.8 us, two launches 4 of them.
//
// Two forms. Many long rows are walked, as follows; few rows or short ones are held in registers (short_part below).
//
// Selection. A wave keeps its part's largest values in order, one to a lane, and walks the part in ascending order, 512 values
// at a time, with the top-th of them as a threshold. Values above it wait in LDS until there are as many as the list is to
// hold and are put in their places together; an equal one need not be: `top` values of its size with lower ids are there. One
// comparison of each lane's maximum, which the softmax needs anyway, and a scalar branch are the whole cost where nothing
// qualifies, which after i chunks is all but about top / i of them. The waves of a workgroup help each other: of the 64 values
// that they have on show, the largest of each, the top-th largest is a bound that `top` values of the row reach. List entries
// are 64-bit keys, the value's bits in integer order above the complemented id: a total order, so the result does not depend
// on who finds what when.
//
// A row is cut into parts, a wave each, whose chunks lie side by side. The parts' lists meet in one workgroup: their keys in
// 128 groups, the top-th largest of the groups' maxima is a bound that `top` keys reach and few others, and what reaches it is
// ordered by counting.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>
#include "join_kernels.h"
#include "wave_fence.h"

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
template <int CTRL, int ROWS>
__device__ __forceinline__ float max_from(float v) {
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), CTRL, ROWS, 0xf, false)));
}
__device__ __forceinline__ float wave_max(float v) {  // as wave_sum
    v = max_from<0xB1, 0xf>(v);
    v = max_from<0x4E, 0xf>(v);
    v = max_from<0x141, 0xf>(v);
    v = max_from<0x140, 0xf>(v);
    v = max_from<0x142, 0xa>(v);
    v = max_from<0x143, 0xc>(v);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Running sums of 2^(v c - r), c = scale * log2 e, and of that times its exponent, relative to r = m c rounded to FP32, m the
// largest value so far: the exponent is then one fused multiply-add, rounded once, and r, the same number everywhere, comes
// out again at the end. From 2^24 on that rounding is more than one, up to any size (masks of -1e9, or of the type's lowest
// value, in a row of nothing else): such values are `far`, and measured from m itself, (v - m) c.
struct SoftmaxSums {
    float m = -INFINITY, z = 0.0f, s = 0.0f;

    __device__ __forceinline__ static bool far(float m, float c) { return fabsf(m * c) > 16777216.0f && m != -INFINITY; }
    __device__ __forceinline__ static float distance(float v, float m, float c) {
        return far(m, c) ? (v - m) * c : __builtin_fmaf(v, c, m == -INFINITY ? 0.0f : -(m * c));
    }
    // The sums relative to the maximum `to` (>= m). Without a number so far z and s are 0, or NaN.
    __device__ __forceinline__ SoftmaxSums at(float to, float c) const {
        const bool here = far(m, c), there = far(to, c);
        const float between = here == there ? (here ? (m - to) * c : m * c - to * c)
                                            : here ? __builtin_fmaf(m, c, -(to * c)) : -__builtin_fmaf(to, c, -(m * c));
        return moved(to, m == to || m == -INFINITY ? 0.0f : between);
    }
    // The same where all sums are relative to a rounded r, whatever its size.
    __device__ __forceinline__ SoftmaxSums at_rounded(float to, float c) const {
        return moved(to, m == to || m == -INFINITY ? 0.0f : m * c - to * c);
    }
    // What is left far behind counts nothing, even if a rounded r had made it infinite; NaN stays.
    __device__ __forceinline__ SoftmaxSums moved(float to, float d) const {
        if (d < -256.0f) return SoftmaxSums{to, z != z ? z : 0.0f, z != z ? z : 0.0f};
        const float f = __builtin_amdgcn_exp2f(d);
        return SoftmaxSums{to, f * z, f * (s + d * z)};
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
    // Over the wave, the same in every lane: the largest m first, then each lane's sums relative to it, added up in a fixed order.
    __device__ __forceinline__ void join_lanes(float c) {
        *this = at(wave_max(m), c);
        z = wave_sum(z);
        s = wave_sum(s);
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

// The next number below v; below zero that is the smallest negative one.
__device__ __forceinline__ float just_below(float v) {
    const uint32_t o = order_bits(v);
    return order_value(o - (o == 0x80000000u ? 2 : 1));  // below zero's bits lie those of -0, which counts as zero
}

// A wave's largest keys in descending order, lane i the i-th; kNoKey where there are fewer. Lanes from `top` on mean nothing.
template <int WAVES>
struct TopList {
    uint32_t* shown;         // LDS: of each wave of the workgroup the order bits of its 64 / WAVES largest values, 0 for none
    uint64_t *batch, *turn;  // LDS, 64 each, this wave's
    int top, wave;
    uint64_t key = kNoKey;
    float threshold = -INFINITY;  // uniform: a value has to be above this one to matter
    int waiting = 0;              // uniform: keys in `batch`

    __device__ __forceinline__ static uint64_t of_lane(uint64_t k, int lane) {
        return uint64_t(__builtin_amdgcn_readlane(uint32_t(k >> 32), lane)) << 32 | uint32_t(__builtin_amdgcn_readlane(uint32_t(k), lane));
    }
    // Puts what waits in its place: a key's place is the number of larger ones.
    __device__ __forceinline__ void merge() {
        const int lane = threadIdx.x & 63;
        wave_fence();
        const uint64_t fresh = lane < waiting ? batch[lane] : kNoKey;
        int place = 0, moved = lane;
        for (int i = 0; i < waiting; ++i) {
            const uint64_t k = of_lane(fresh, i);
            const bool above = key > k;
            const int before = int(__popcll(__ballot(above)));  // places that the list's keys take ahead of this one
            moved += !above;
            place += (lane == i ? before : 0) + (k > fresh);
        }
        turn[lane] = kNoKey;
        wave_fence();
        if (key != kNoKey && moved < 64) turn[moved] = key;
        if (fresh != kNoKey && place < 64) turn[place] = fresh;
        wave_fence();
        key = turn[lane];
        wave_fence();
        waiting = 0;
    }
    __device__ __forceinline__ int enough() const { return top < 8 ? 8 : top; }
    // What the values on show vouch for: `top` values of the row reach it, at any ids, so equal ones still count.
    __device__ __forceinline__ void common() {
        const uint32_t v[1] = {__hip_atomic_load(&shown[threadIdx.x & 63], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)};
        const uint32_t bound = reached_by<16>(v, top);
        if (bound > order_bits(-INFINITY)) threshold = fmaxf(threshold, just_below(order_value(bound)));
    }
    // The slow path of a chunk. Element j of the lane has id `id` + j. What is above the threshold waits, and is put in its place
    // when as much waits as the list is to hold: a place costs 50 cycles then, in a list of its own 300.
    __device__ __forceinline__ void take(const float (&v)[8], int id) {
        if (threshold == -INFINITY) {
            // Nothing known yet: what `top` of the lanes' maxima reach, as many values of this chunk do. As many as are put in
            // their places at once: the few values ahead of a boundary would give a bound that lets half the next chunk pass
            // (600 x 50003 BF16, top 1: 49 us against 26).
            float largest = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) largest = v[j] > largest ? v[j] : largest;  // a NaN takes no part
            const uint32_t mine[1] = {order_bits(largest)};
            const uint32_t bound = reached_by<16>(mine, enough());
            if (bound > order_bits(-INFINITY)) threshold = just_below(order_value(bound));
        }
        // Within the chunk ids are not met in order, so the threshold stays as it is until its end.
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool wanted = v[j] > threshold;
            const uint64_t mask = __ballot(wanted);
            if (!mask) continue;
            const int n = int(__popcll(mask));
            if (waiting + n > 64) merge();
            if (wanted) batch[waiting + lanes_below(mask)] = list_key(v[j], id + j);
            waiting += n;
        }
        if (waiting < enough()) return;
        const int lane = threadIdx.x & 63;
        merge();
        const uint32_t last = __builtin_amdgcn_readlane(uint32_t(key >> 32), top - 1);
        if (last) threshold = fmaxf(threshold, order_value(last));
        if constexpr (WAVES > 2) {  // two waves gain less than it costs
            constexpr int kShow = 64 / WAVES;
            if (lane < kShow && lane < top) __hip_atomic_store(&shown[wave * kShow + lane], uint32_t(key >> 32), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            common();
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

    // Everything but what the whole chunks of ordinary rows need: element by element, with comparisons for the maximum (the
    // hardware's passes a signalling NaN on, quieted, and loses what it was compared with) and any size of values.
    template <typename LIST>
    __device__ __forceinline__ void slowly(const LogprobArgs& a, SoftmaxSums& sum, LIST& list, int id, int stop, float c) const {
        float v[8], most = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = id + j < stop ? value(id + j) : -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = v[j] > most ? v[j] : most;
        if (most > sum.m) sum = sum.at(most, c);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum.add(SoftmaxSums::distance(v[j], sum.m, c));
        if (a.top && __any(most > list.threshold)) list.take(v, id);
    }
    // The whole chunks, in pairs, with the next pair on its way. Past the end the last chunk is asked for again: a load under a
    // condition would make the compiler wait for all of them. One copy of the work on a chunk: unrolled over a ring of four it
    // was 45 KB of code, which a short call fetches as it goes. True if the sums are not to be trusted: a NaN, or nothing but far values.
    template <typename LIST>
    __device__ __forceinline__ bool quickly(const LogprobArgs& a, SoftmaxSums& sum, LIST& list, float c) const {
        const int lane = threadIdx.x & 63, final_chunk = part + (chunks - 1 - part) / parts * parts;
        auto ask = [&](int chunk) { return load(chunk < final_chunk ? chunk : final_chunk); };
        Raw first = ask(part), second = ask(part + parts);
        const SoftmaxSums ahead = sum;  // of the boundary
        sum = SoftmaxSums{};
        float r = 0.0f;
        for (int chunk = part; chunk <= final_chunk;) {
            const Raw third = ask(chunk + 2 * parts), fourth = ask(chunk + 3 * parts);
#pragma nounroll
            for (int i = 0; i < 2 && chunk <= final_chunk; ++i) {
                float v[8];
                widen(first, v);
                float most = v[0];
#pragma unroll
                for (int j = 1; j < 8; ++j) most = fmaxf(most, v[j]);
                if (__any(most > sum.m)) {
                    sum = sum.at_rounded(fmaxf(most, sum.m), c);
                    r = sum.m == -INFINITY ? 0.0f : -(sum.m * c);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) sum.add(__builtin_fmaf(v[j], c, r));
                if (a.top && __any(most > list.threshold)) list.take(v, head + chunk * kChunk + lane * 8);
                first = second;
                chunk += parts;
            }
            first = third;
            second = fourth;
        }
        // Lanes that saw nothing but masks: their far maximum does not matter beside the wave's.
        const float largest = wave_max(sum.m);
        if (SoftmaxSums::far(sum.m, c) && !SoftmaxSums::far(largest, c)) sum = sum.at_rounded(largest, c);
        const bool lost = __any(sum.z != sum.z || SoftmaxSums::far(sum.m, c));
        sum.join(ahead, c);
        return lost;
    }

    template <typename LIST>
    __device__ __forceinline__ void walk(const LogprobArgs& a, SoftmaxSums& sum, LIST& list) const {
        const int lane = threadIdx.x & 63, done = head + chunks * kChunk;
        const float c = a.scale * 1.44269504088896341f;
        // A part whose whole chunks turn out to hold a NaN, or nothing but far values, is gone through once more, slowly.
        for (bool careful = false, lost = false;; careful = true) {
            for (int phase = 0; phase < 3; ++phase) {  // ahead of the boundary; whole chunks; what is left behind them
                if (phase == 1 && !careful) {
                    if (part < chunks) lost = quickly(a, sum, list, c);
                    continue;
                }
                const bool mine = phase == 0 ? part == 0 : phase == 1 || part == parts - 1;
                const int stop = phase == 0 ? head : phase == 1 ? done : vocab;
                for (int id = phase == 0 ? 0 : phase == 1 ? head + part * kChunk : done; mine && id < stop; id += parts * kChunk)
                    slowly(a, sum, list, id + lane * 8, stop, c);
            }
            if (careful || !lost) break;
            sum = SoftmaxSums{};
            list.key = kNoKey;
            list.threshold = -INFINITY;
            list.waiting = 0;
        }
        sum.join_lanes(c);
        if (list.waiting) list.merge();
    }
};

// The logit of a row's i-th given token, asked for ahead of the rest; `there` false for an id outside the vocabulary or past the last.
struct GivenLogit {
    float v;
    bool there;
};
template <bool BF16>
__device__ __forceinline__ GivenLogit given_logit(const LogprobArgs& a, long row, int i) {
    const int id = i < a.n_given ? a.given[row * a.n_given + i] : -1;
    GivenLogit g{0.0f, id >= 0 && id < a.vocab};
    if (g.there) {
        const long at = row * a.pitch + id;
        if constexpr (BF16) g.v = __uint_as_float(uint32_t(static_cast<const uint16_t*>(a.logits)[at]) << 16);
        else g.v = static_cast<const float*>(a.logits)[at];
    }
    return g;
}

// What a workgroup of THREADS makes of a row's joined sums and the parts' keys: N a thread, kNoKey for none. Every thread of
// the workgroup comes here.
constexpr int kRoom = 256, kGroups = 128;
struct RowShared {
    uint64_t room[kRoom];
    uint32_t most[kGroups];
    int count, reached[64];
};
template <bool BF16, int THREADS, int N>
__device__ __forceinline__ void write_row(const LogprobArgs& a, long row, const SoftmaxSums& sum, GivenLogit given, const uint64_t (&key)[N], RowShared& sh) {
    const int tid = threadIdx.x, lane = tid & 63;
    const float c = a.scale * 1.44269504088896341f, log_z = log2f(sum.z);
    constexpr float kLn2 = 0.69314718055994531f;
    const bool empty = sum.m == -INFINITY && sum.z == 0.0f;
    // Z is relative to 2^r, r = m c rounded: what r is short of m c is exactly a fused product
    // Z relative to 2^(m c) is one at least and the entropy zero at least: what the roundings leave below counts as that (one token left)
    // and a NaN goes through.
    auto not_below_zero = [](float v) { return v <= 0.0f ? 0.0f : v; };
    const float ln_z = kLn2 * not_below_zero(SoftmaxSums::far(sum.m, c) || sum.m == -INFINITY ? log_z : log_z - __builtin_fmaf(sum.m, c, -(sum.m * c)));
    // halves, so that the difference of two numbers is one
    auto logprob = [&](float v) { return (0.5f * v - 0.5f * sum.m) * (2.0f * a.scale) - ln_z; };
    if (tid == 0 && a.entropy) a.entropy[row] = empty ? 0.0f : kLn2 * not_below_zero(log_z - sum.s / sum.z);
    for (int i = tid; i < a.n_given; i += THREADS) {
        if (i >= THREADS) given = given_logit<BF16>(a, row, i);
        a.given_logprob[row * a.n_given + i] = !given.there ? __builtin_nanf("") : empty ? -INFINITY : logprob(given.v);
    }
    if (!a.top) return;
    constexpr bool kFew = N == 1 && THREADS / 64 * kTopMost <= kRoom;
    if constexpr (kFew) {  // few enough to order as they are: a key's place is the number of larger ones
        const int all = THREADS / 64 * a.top;
        if (lane < a.top) sh.room[(tid >> 6) * a.top + lane] = key[0];
        __syncthreads();
        for (int i = tid; i < all; i += THREADS) {
            const uint64_t k = sh.room[i];
            int larger = 0, there = 0;
#pragma unroll 8
            for (int j = 0; j < all; ++j) {
                const uint64_t o = sh.room[j];
                larger += o > k;
                there += o != kNoKey;
            }
            if (k != kNoKey && larger < a.top) {
                a.top_ids[row * a.top + larger] = key_id(k);
                a.top_logprob[row * a.top + larger] = logprob(key_value(k));
            }
            if (i >= there && i < a.top) {
                a.top_ids[row * a.top + i] = -1;
                a.top_logprob[row * a.top + i] = -INFINITY;
            }
        }
    } else {
        // The bound: values alone, from the maxima of kGroups groups of threads.
        constexpr int kLanes = THREADS / kGroups;  // of a group
        static_assert(THREADS % kGroups == 0 && kLanes <= 8, "the lanes' exchanges below");
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) most = uint32_t(key[i] >> 32) > most ? uint32_t(key[i] >> 32) : most;
        auto larger_of = [&](uint32_t o) { most = o > most ? o : most; };
        if (kLanes > 1) larger_of(uint32_t(__builtin_amdgcn_update_dpp(0, int(most), kQuadXor1, 0xf, 0xf, false)));
        if (kLanes > 2) larger_of(uint32_t(__builtin_amdgcn_update_dpp(0, int(most), kQuadXor2, 0xf, 0xf, false)));
        if (kLanes > 4) larger_of(uint32_t(__builtin_amdgcn_update_dpp(0, int(most), kHalfRowMirror, 0xf, 0xf, false)));
        if (tid % kLanes == 0) sh.most[tid / kLanes] = most;
        if (tid >= THREADS - 64) sh.reached[lane] = 0;
        if (tid == 64) sh.count = 0;
        __syncthreads();
        const uint32_t two[2] = {sh.most[lane], sh.most[64 + lane]};
        uint64_t bound = uint64_t(reached_by<16>(two, a.top)) << 32;
        auto reach = [&](uint64_t k) {  // keys of this wave that reach k
            int n = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) n += int(__popcll(__ballot(key[i] != kNoKey && key[i] >= k)));
            return n;
        };
        auto gather = [&] {  // a key's place in the result does not depend on which wave is first here
            const int here = reach(bound);
            int at = 0;
            if (here && lane == 0) at = atomicAdd(&sh.count, here);
            at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const bool kept = key[i] != kNoKey && key[i] >= bound;
                const uint64_t mask = __ballot(kept);
                if (kept && at + lanes_below(mask) < kRoom) sh.room[at + lanes_below(mask)] = key[i];
                at += int(__popcll(mask));
            }
            __syncthreads();
            return sh.count;
        };
        int count = gather();
        if (count > kRoom) {  // many equal values, or lists that each hold all but one of the largest: bit by bit, until few enough are left
            bound = 0;
            for (int bit = 63; bit >= 0; --bit) {
                const int n = reach(bound | 1ull << bit);
                if (n && lane == 0) atomicAdd(&sh.reached[bit], n);
                __syncthreads();
                const int all = sh.reached[bit];
                if (all >= a.top) bound |= 1ull << bit;
                if (all >= a.top && all <= kRoom) break;
            }
            if (tid == 0) sh.count = 0;
            __syncthreads();
            count = gather();  // all there are, if that is fewer than `top`
        }
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
}

template <int WAVES>
struct ListShared {
    uint64_t batch[WAVES][64], turn[WAVES][64];
    uint32_t shown[64];
};
template <int WAVES>
__device__ __forceinline__ TopList<WAVES> empty_list(ListShared<WAVES>& sh, int top) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (WAVES > 2) {
        if (threadIdx.x < 64) sh.shown[threadIdx.x] = 0;
        __syncthreads();
    }
    return TopList<WAVES>{sh.shown, sh.batch[wave], sh.turn[wave], top, wave};
}

// A workgroup per row at a time, a part for each of its WAVES waves.
template <bool BF16, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) logprob_row_kernel(const LogprobArgs a) {
    __shared__ float4 sums[WAVES];
    __shared__ RowShared shared;
    __shared__ ListShared<WAVES> list_shared;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const GivenLogit given = given_logit<BF16>(a, row, threadIdx.x);
        SoftmaxSums sum;
        TopList<WAVES> list = empty_list(list_shared, a.top);
        RowPart<BF16>(a, row, wave, WAVES).walk(a, sum, list);
        if (lane == 0) sums[wave] = make_float4(sum.m, sum.z, sum.s, 0.0f);
        __syncthreads();
        const float c = a.scale * 1.44269504088896341f;
        sum = SoftmaxSums{};
        if (lane < WAVES) sum = SoftmaxSums{sums[lane].x, sums[lane].y, sums[lane].z};
        sum.join_lanes(c);
        const uint64_t key[1] = {lane < a.top ? list.key : kNoKey};
        write_row<BF16, 64 * WAVES>(a, row, sum, given, key, shared);
        __syncthreads();
    }
}

// A row over several workgroups: each wave leaves its part's sums and list in memory ...
constexpr int kPartWaves = 4;
template <bool BF16>
__global__ void __launch_bounds__(64 * kPartWaves) logprob_part_kernel(const LogprobArgs a) {
    __shared__ ListShared<kPartWaves> shared;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long cell = long(blockIdx.x) * kPartWaves + wave;  // parts is a multiple of kPartWaves: a workgroup is of one row
    SoftmaxSums sum;
    TopList<kPartWaves> list = empty_list(shared, a.top);
    RowPart<BF16>(a, cell / a.parts, int(cell % a.parts), a.parts).walk(a, sum, list);
    if (lane == 0) a.stats[cell] = make_float4(sum.m, sum.z, sum.s, 0.0f);
    if (lane < a.top) a.lists[cell * a.top + lane] = list.key;
}

// A part of CHUNKS chunks that lie one after another, held in registers: where rows are short or there are few of them, nothing
// is gained by walking, and what the walk does chunk by chunk (thresholds, merges, two forms of the sums) is done once. The
// maximum comes first, by comparisons, so the sums are right for any values; the bound is what `top` of the lanes' maxima
// reach; the few values that reach it are ordered by counting. `batch`: LDS, kBatch, this wave's; put(place, key) takes the list.
// About 45 of 1024 values reach the bound of a list of 32; with 64 places some wave of many goes the long way (4096 x 1000 BF16:
// 25 us against 11).
constexpr int kBatch = 128;
template <bool BF16, int CHUNKS, typename PUT>
__device__ __forceinline__ SoftmaxSums short_part(const LogprobArgs& a, long row, int part, uint64_t* batch, PUT put) {
    typedef typename std::conditional<BF16, uint16_t, float>::type T;
    constexpr int N = 8 * CHUNKS;
    const int lane = threadIdx.x & 63;
    const T* base = static_cast<const T*>(a.logits) + row * a.pitch;
    const int first = part * (CHUNKS * kChunk) + lane * 8;
    // Chunk i's values of this lane start at id(i); at the row's end they are the last eight, of which the first ones are not its own.
    auto id = [&](int i) { const int at = first + i * kChunk; return at < a.vocab - 8 ? at : a.vocab - 8; };
    float v[N];
    if (a.vocab >= 8) {
        v4u raw[CHUNKS][BF16 ? 1 : 2];
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
            for (int j = 0; j < (BF16 ? 1 : 2); ++j) raw[i][j] = *(reinterpret_cast<const v4u_any*>(base + id(i)) + j);
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint32_t bits;
                if constexpr (BF16) bits = j & 1 ? raw[i][0][j / 2] & 0xffff0000u : raw[i][0][j / 2] << 16;
                else bits = raw[i][j / 4][j % 4];
                v[8 * i + j] = id(i) + j >= first + i * kChunk ? __uint_as_float(bits) : -INFINITY;
            }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (id(0) + j < first || id(0) + j < 0) continue;
            if constexpr (BF16) v[j] = __uint_as_float(uint32_t(base[id(0) + j]) << 16);
            else v[j] = base[id(0) + j];
        }
    }
    const float c = a.scale * 1.44269504088896341f;
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) most = v[i] > most ? v[i] : most;  // a NaN takes no part
    SoftmaxSums sum;
    sum.m = wave_max(most);
#pragma unroll
    for (int i = 0; i < N; ++i) sum.add(SoftmaxSums::distance(v[i], sum.m, c));
    sum.z = wave_sum(sum.z);
    sum.s = wave_sum(sum.s);
    if (!a.top) return sum;
    uint32_t order[N];  // 0 for what is no alternative
#pragma unroll
    for (int i = 0; i < N; ++i) order[i] = v[i] > -INFINITY ? order_bits(v[i]) : 0;
    const uint32_t mine[1] = {order_bits(most)};
    uint32_t cut = reached_by<16>(mine, a.top), id_cut = 0;  // wanted: above the cut, or at it and ~id at least id_cut
    if (cut == 0) cut = 1;
    auto wanted = [&](int i) { return order[i] > cut || (order[i] == cut && uint32_t(~(id(i / 8) + i % 8)) >= id_cut); };
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n += int(__popcll(__ballot(order[i] >= cut)));
    if (n > kBatch) {  // many equal values, or too few lanes with any: bit by bit, until few enough are left
        cut = 0;
#pragma nounroll
        for (int bit = 31; bit >= 0 && n > kBatch; --bit) {
            const uint32_t higher = cut | 1u << bit;
            int m = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) m += int(__popcll(__ballot(order[i] >= higher)));
            if (m >= a.top) {
                cut = higher;
                n = m;
            }
        }
#pragma nounroll
        for (int bit = 31; bit >= 0 && n > kBatch; --bit) {  // equal ones by their ids
            const uint32_t before = id_cut;
            id_cut |= 1u << bit;
            int m = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) m += int(__popcll(__ballot(wanted(i))));
            if (m >= a.top) n = m;
            else id_cut = before;
        }
    }
    int at = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool mine_is = wanted(i);
        const uint64_t mask = __ballot(mine_is);
        if (mine_is) batch[at + lanes_below(mask)] = uint64_t(order[i]) << 32 | uint32_t(~(id(i / 8) + i % 8));
        at += int(__popcll(mask));
    }
    wave_fence();
    auto place = [&](int i) {
        if (i >= n) {
            if (i < a.top) put(i, kNoKey);
            return;
        }
        const uint64_t k = batch[i];
        int larger = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) larger += batch[j] > k;
        if (larger < a.top) put(larger, k);
    };
    place(lane);
    if (n > 64) place(64 + lane);
    return sum;
}

// A workgroup per row at a time, a short part for each of its waves.
template <bool BF16, int WAVES, int CHUNKS>
__global__ void __launch_bounds__(64 * WAVES) logprob_short_row_kernel(const LogprobArgs a) {
    __shared__ float4 sums[WAVES];
    __shared__ uint64_t batch[WAVES][kBatch], list[WAVES][kTopMost];
    __shared__ RowShared shared;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const GivenLogit given = given_logit<BF16>(a, row, threadIdx.x);
        SoftmaxSums sum = short_part<BF16, CHUNKS>(a, row, wave, batch[wave], [&](int place, uint64_t k) { list[wave][place] = k; });
        if (lane == 0) sums[wave] = make_float4(sum.m, sum.z, sum.s, 0.0f);
        __syncthreads();
        if (WAVES > 1) {
            sum = SoftmaxSums{};
            if (lane < WAVES) sum = SoftmaxSums{sums[lane].x, sums[lane].y, sums[lane].z};
            sum.join_lanes(a.scale * 1.44269504088896341f);
        }
        const uint64_t key[1] = {lane < a.top ? list[wave][lane] : kNoKey};
        write_row<BF16, 64 * WAVES>(a, row, sum, given, key, shared);
        __syncthreads();
    }
}

// A row over several workgroups of short parts.
template <bool BF16, int CHUNKS>
__global__ void __launch_bounds__(64 * kPartWaves) logprob_short_part_kernel(const LogprobArgs a) {
    __shared__ uint64_t batch[kPartWaves][kBatch];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long cell = long(blockIdx.x) * kPartWaves + wave;
    const SoftmaxSums sum = short_part<BF16, CHUNKS>(a, cell / a.parts, int(cell % a.parts), batch[wave],
                                                     [&](int place, uint64_t k) { a.lists[cell * a.top + place] = k; });
    if (lane == 0) a.stats[cell] = make_float4(sum.m, sum.z, sum.s, 0.0f);
}

// ... and a workgroup per row joins them, everything it reads asked for at once.
constexpr int kJoinThreads = 512;
template <bool BF16>
__global__ void __launch_bounds__(kJoinThreads) logprob_join_kernel(const LogprobArgs a) {
    constexpr int N = kPartsMost * kTopMost / kJoinThreads;
    __shared__ RowShared shared;
    const int lane = threadIdx.x & 63;
    const long row = blockIdx.x;
    const float c = a.scale * 1.44269504088896341f;
    const float4* stats = a.stats + row * a.parts;
    const uint64_t* lists = a.lists + row * a.parts * a.top;
    const GivenLogit given = given_logit<BF16>(a, row, threadIdx.x);
    // The groups whose maxima give the bound are each a part's list, or with fewer parts each `per`-th key of it: in order over
    // the threads, groups could hold nothing but last places (1 row x 131072, top 32: 28 us).
    constexpr int kLanes = kJoinThreads / kGroups;
    static_assert(kGroups >= kPartsMost && kLanes * N >= kTopMost, "a group takes a whole list");
    const int per = kGroups / a.parts, group = int(threadIdx.x) / kLanes, part = group / per, sub = group % per;
    float4 two[2];
    uint64_t key[N];
#pragma unroll
    for (int i = 0; i < 2; ++i) two[i] = lane + 64 * i < a.parts ? stats[lane + 64 * i] : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int rank = sub + per * (int(threadIdx.x) % kLanes + kLanes * i);
        key[i] = part < a.parts && rank < a.top ? lists[part * a.top + rank] : kNoKey;
    }
    SoftmaxSums sum{two[0].x, two[0].y, two[0].z};
    sum.join(SoftmaxSums{two[1].x, two[1].y, two[1].z}, c);
    sum.join_lanes(c);
    write_row<BF16, kJoinThreads>(a, row, sum, given, key, shared);
}

}  // namespace m26g

// Routing to the k best experts, and token rows to k experts and back.  The reference routes to one expert (top-k is a TODO
// there); these kernels stand beside its select / scatter / gather (plugin/cuda/moe.cu:147-258) for layers that route to k.
//
//   select   s = softmax(l) or sigmoid(l), c = s + bias; the k best c of the best groups, weights s / sum s of these.  65536 tokens,
//            8 of 256 experts in groups, FP32: 59 us, 5.4 times what its 71 MB take at the copy rate; bound by instructions (567
//            a token, the integer pipe 64 % busy).  Few tokens: 3 us.
//   scatter  routed[j] = x[pos[j] / k].  32768 rows of 8 KB: 55 to 57 us, 1.25 times its 287 MB; writes.
//   combine  out[t] = sum_s w[t, s] y[row(t, s)] + (1 - sum_s w[t, s]) x[t].  4096 tokens x 4 rows of 16 KB and their own: 62 us, its
//            389 MB at 6.3 TB/s.
#include <cfloat>
#include <type_traits>

#include "common.cuh"
#include "elem.cuh"
#include "kernels.h"

namespace infmoe {

namespace {

constexpr int SELECT_WARPS = 8;
// Experts of a token that 32 bits can choose: from there on lists of four keys run out too often, and all are chosen in 64 bits (65536 tokens
// of 256 experts by logits: 16 of them 55 us, 17 282).
constexpr int MAX_FAST_K = 16, MAX_ROUNDS = 18;

// Experts are laid out over the lanes of a warp so that a group's experts sit on lanes of their own: groups are padded to a
// power of two, group g has `lanes` = 32 / padded lanes, and each of these holds V consecutive experts of the group.  So
// lane order, and place order inside a lane, is expert order, and the lowest lane and place win ties.
struct SelectArgs {
    const void* logits;      // [T][ld]
    long long T, ld;
    int E, k, groups, top_groups, group_best, group_size, lanes, lanes_log2, width_log2;
    int sigmoid, renormalise, vec;     // vec: a lane's logits are read 16 bytes at a time
    float scale;
    const float* bias;       // [E] or NULL
    int* gate;               // [T][k]
    float* weight;           // [T][k]
    int* status;
};

template <typename T>
struct Lowest;
template <> struct Lowest<float> { static __device__ float value() { return -FLT_MAX; } };
template <> struct Lowest<__half> { static __device__ float value() { return -65504.f; } };
template <> struct Lowest<__nv_bfloat16> { static __device__ float value() { return __uint_as_float(0xff7f0000u); } };

__device__ __forceinline__ double shfl_xor(double v, int off) { return __shfl_xor_sync(0xffffffffu, v, off); }

// Expert indices of the k best in lanes 0..k-1, -1 where there are fewer, chosen by scores in 64 bits.
template <typename T, int V>
__device__ __noinline__ int select_in_64_bits(const SelectArgs& a, long long t, int lane) {
    const T* row = static_cast<const T*>(a.logits) + t * a.ld;
    const int g = lane / a.lanes, first = (lane - g * a.lanes) * V;
    const double none = -INFINITY;
    double c[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const bool in = g < a.groups && first + j < a.group_size;
        const float l = in ? to_float(row[g * a.group_size + first + j]) : -INFINITY;
        c[j] = l > Lowest<T>::value() ? (double)l : none;      // false for NaN too
    }
    // Without a bias the logits order the experts: scores would order them the same, but for those that round to one value.
    double top = none, sum = 0.0;
    if (!a.sigmoid && (a.bias || (a.groups > 1 && a.group_best == 2))) {
#pragma unroll
        for (int j = 0; j < V; ++j) top = fmax(top, c[j]);
        for (int off = 16; off >= 1; off >>= 1) top = fmax(top, shfl_xor(top, off));
#pragma unroll
        for (int j = 0; j < V; ++j) sum += c[j] == none ? 0.0 : c[j] == top ? 1.0 : exp(c[j] - top);
        for (int off = 16; off >= 1; off >>= 1) sum += shfl_xor(sum, off);
    }
    const auto score_of = [&](double l) {
        return a.sigmoid ? 1.0 / (1.0 + exp(-l)) : (l == top ? 1.0 : exp(l - top)) / sum;
    };
    if (a.bias) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (c[j] == none) continue;
            const float b = a.bias[g * a.group_size + first + j];
            c[j] = b > -INFINITY ? score_of(c[j]) + (double)b : none;
        }
    }
    if (a.groups > 1) {
        // the two best of the group, then the groups best first
        double b1 = none, b2 = none;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            b2 = fmax(b2, fmin(b1, c[j]));
            b1 = fmax(b1, c[j]);
        }
        for (int off = a.lanes >> 1; off >= 1; off >>= 1) {
            const double o1 = shfl_xor(b1, off), o2 = shfl_xor(b2, off);
            b2 = fmax(fmin(b1, o1), fmax(b2, o2));
            b1 = fmax(b1, o1);
        }
        double score = b1;
        if (a.group_best == 2 && b1 > none) {
            score = a.bias ? b1 : score_of(b1);
            if (b2 > none) score += a.bias ? b2 : score_of(b2);
        }
        int better = 0;
        for (int o = 0; o < a.groups; ++o) {
            const double other = __shfl_sync(0xffffffffu, score, o * a.lanes);
            better += other > score || (other == score && o < g);
        }
        if (better >= a.top_groups)
#pragma unroll
            for (int j = 0; j < V; ++j) c[j] = none;
    }
    int mine = -1;
    for (int i = 0; i < a.k; ++i) {
        double best = none;
#pragma unroll
        for (int j = 0; j < V; ++j) best = fmax(best, c[j]);
        // the largest of the lanes': numbers of 64 bits in the scores' order, upper halves first
        const long long w = __double_as_longlong(best + 0.0);       // -0 is 0
        const unsigned long long key = (unsigned long long)w ^ ((unsigned long long)(w >> 63) | 0x8000000000000000ull);
        const unsigned high = __reduce_max_sync(0xffffffffu, (unsigned)(key >> 32));
        const bool in = (unsigned)(key >> 32) == high;
        const unsigned low = __reduce_max_sync(0xffffffffu, in ? (unsigned)key : 0u);
        const int owner = __ffs(__ballot_sync(0xffffffffu, in && (unsigned)key == low)) - 1;
        if (high == 0x000fffffu) break;                             // -inf
        int place = 0;
#pragma unroll
        for (int j = V - 1; j >= 0; --j) place = c[j] == best ? j : place;
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (lane == owner && j == place) c[j] = none;
        const int e = __shfl_sync(0xffffffffu, g * a.group_size + first + place, owner);
        if (lane == i) mine = e;
    }
    return mine;
}

// The same from scores in 32 bits, as long as these tell all that matters apart; else false, and the choice has to be made in 64.
//
// A score becomes a 32-bit key whose order as an unsigned number is that of the scores; an expert that cannot be chosen has the
// score -inf, the keys up to NONE.  A key's lowest bits give way to the place in the lane, so that sorting keys carries the index
// along: with V = 8 that moves a score by 2^-20 of itself, no more than what exp and division leave uncertain.  By logits of 16
// bits nothing moves at all: their FP32 form has 13 bits to spare, which hold the whole index.  A lane sorts its keys (two
// instructions a comparison), and each round takes the largest of the 32 heads by one redux and moves that lane's list on.  Lists
// hold four or five keys; a lane that has more and uses up its list shows a last one that nothing exceeds, which counts as undecided
// (65536 tokens, 8 of 256 experts, of which 16 lanes hold what four of eight groups have: 277 undecided with lists of four, 149 of five).
template <int V>
struct Keys {
    static constexpr int PLACE_BITS = V <= 1 ? 0 : V <= 2 ? 1 : V <= 4 ? 2 : V <= 8 ? 3 : V <= 16 ? 4 : 5;
    static constexpr int DEPTH = V < 4 ? V : V == 8 ? 5 : 4;
    static constexpr uint32_t PLACES = (1u << PLACE_BITS) - 1, MORE = 0xffffffffu, NONE = 0x007fffffu;
};

__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t w = __float_as_uint(v);
    return w ^ ((uint32_t)((int)w >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key ^ ((uint32_t)(~(int)key >> 31) | 0x80000000u));
}
__device__ __forceinline__ void descending(uint32_t& a, uint32_t& b) {
    const uint32_t high = max(a, b);
    b = min(a, b);
    a = high;
}
__device__ __forceinline__ void sort4(uint32_t (&k)[4]) {
    descending(k[0], k[1]);
    descending(k[2], k[3]);
    descending(k[0], k[2]);
    descending(k[1], k[3]);
    descending(k[1], k[2]);
}
// The D largest of N keys, largest first: N <= 4 all of them, of eight up to five, else four.
template <int N, int D>
__device__ __forceinline__ void largest(const uint32_t* k, uint32_t (&out)[D]) {
    if constexpr (N <= 4) {
        static_assert(D == N, "all of them");
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = k[i];
        if constexpr (N == 2) descending(out[0], out[1]);
        if constexpr (N == 4) sort4(out);
    } else {
        uint32_t one[4], other[4];
        largest<N / 2, 4>(k, one);
        largest<N / 2, 4>(k + N / 2, other);
        // the larger of one's i-th and other's (3 - i)-th, the largest four of all eight, rise and fall; the fifth is the largest of the rest
        if constexpr (D == 5)
            out[4] = max(max(min(one[0], other[3]), min(one[1], other[2])), max(min(one[2], other[1]), min(one[3], other[0])));
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = max(one[i], other[3 - i]);
        descending(out[0], out[2]);
        descending(out[1], out[3]);
        descending(out[0], out[1]);
        descending(out[2], out[3]);
    }
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float reciprocal_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The lane whose first key is the warp's largest, unless that stands for none, leaves it and `base` in place i of `found` and moves its
// list on.  One predicate for all of it: a branch, or a select for every key, cost twice as much.
template <int DEPTH>
__device__ __forceinline__ void take_head(uint32_t (&head)[DEPTH], uint32_t rest, int& taken, uint32_t top, uint32_t none, uint32_t found,
                                          int i, uint32_t base) {
    const uint32_t to = found + 8 * i;
    if constexpr (DEPTH == 1)
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.gt.u32 q, %3, %4;\n\tsetp.eq.and.u32 p, %0, %3, q;\n\t"
                     "@p st.shared.v2.u32 [%5], {%3, %6};\n\t@p add.s32 %1, %1, 1;\n\t@p mov.u32 %0, %2;\n\t}"
                     : "+r"(head[0]), "+r"(taken)
                     : "r"(rest), "r"(top), "r"(none), "r"(to), "r"(base)
                     : "memory");
    else if constexpr (DEPTH == 2)
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.gt.u32 q, %4, %5;\n\tsetp.eq.and.u32 p, %0, %4, q;\n\t"
                     "@p st.shared.v2.u32 [%6], {%4, %7};\n\t@p add.s32 %2, %2, 1;\n\t@p mov.u32 %0, %1;\n\t@p mov.u32 %1, %3;\n\t}"
                     : "+r"(head[0]), "+r"(head[1]), "+r"(taken)
                     : "r"(rest), "r"(top), "r"(none), "r"(to), "r"(base)
                     : "memory");
    else if constexpr (DEPTH == 4)
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.gt.u32 q, %6, %7;\n\tsetp.eq.and.u32 p, %0, %6, q;\n\t"
                     "@p st.shared.v2.u32 [%8], {%6, %9};\n\t@p add.s32 %4, %4, 1;\n\t@p mov.u32 %0, %1;\n\t@p mov.u32 %1, %2;\n\t"
                     "@p mov.u32 %2, %3;\n\t@p mov.u32 %3, %5;\n\t}"
                     : "+r"(head[0]), "+r"(head[1]), "+r"(head[2]), "+r"(head[3]), "+r"(taken)
                     : "r"(rest), "r"(top), "r"(none), "r"(to), "r"(base)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.gt.u32 q, %7, %8;\n\tsetp.eq.and.u32 p, %0, %7, q;\n\t"
                     "@p st.shared.v2.u32 [%9], {%7, %10};\n\t@p add.s32 %5, %5, 1;\n\t@p mov.u32 %0, %1;\n\t@p mov.u32 %1, %2;\n\t"
                     "@p mov.u32 %2, %3;\n\t@p mov.u32 %3, %4;\n\t@p mov.u32 %4, %6;\n\t}"
                     : "+r"(head[0]), "+r"(head[1]), "+r"(head[2]), "+r"(head[3]), "+r"(head[4]), "+r"(taken)
                     : "r"(rest), "r"(top), "r"(none), "r"(to), "r"(base)
                     : "memory");
}

// What experts are chosen by: the logits themselves, or (with a bias, or groups that count with two experts) scores of them.
enum ChosenBy { LOGITS, SOFTMAX, SIGMOID };

// l[j]: the lane's logits, -inf where there is none to choose (SIGMOID: any that cannot be chosen); bias[j]: their biases; base: the lane's first expert; found: the
// warp's place for the rounds' keys and lanes.
template <typename T, int V, ChosenBy BY>
__device__ __forceinline__ bool select_in_32_bits(const SelectArgs& a, const float (&l)[V], const float (&bias)[V], int lane, int base,
                                                  uint2* found, int& mine) {
    using K = Keys<V>;
    constexpr bool SCORES = BY != LOGITS;
    constexpr bool WHOLE = !SCORES && sizeof(T) == 2;               // the key holds the expert's whole place
    constexpr uint32_t LOW = WHOLE ? 32 * V - 1 : K::PLACES;
    const uint32_t low0 = WHOLE ? (31 - lane) * V + V - 1 : V - 1;
    constexpr float LOG2E = 1.4426950408889634f;
    uint32_t key[V];
    float uncertain = 0.f;                                          // how far a score may be off, twice, beside what its size leaves
    if constexpr (SCORES) {
        float top = 0.f, part = 1.f;
        if constexpr (BY == SOFTMAX) {
            top = l[0];
#pragma unroll
            for (int j = 1; j < V; ++j) top = fmaxf(top, l[j]);
            top = warp_max(top);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j) sum += l[j] == top ? 1.f : exp2_fast((l[j] - top) * LOG2E);
            part = reciprocal_fast(warp_xor_sum(sum));
        }
        // Sigmoid: the exponential is off by (2 + 1.2 |l|) 2^-23, which comes to 0.8 of these units, sum, reciprocal and the sum
        // with the bias to 2.  Softmax: no score exceeds `part`; exponential, sum of up to 1024 of them and reciprocal come to
        // less than 34 units of it.
        uncertain = BY == SIGMOID ? 0x1p-20f : part * 0x1p-17f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float s;
            if constexpr (BY == SIGMOID)
                s = reciprocal_fast(1.f + exp2_fast(l[j] * -LOG2E));
            else
                s = (l[j] == top ? 1.f : exp2_fast((l[j] - top) * LOG2E)) * part;
            const float c = l[j] > (BY == SIGMOID ? Lowest<T>::value() : -INFINITY) ? s + bias[j] : -INFINITY;
            key[j] = (key_of(c) & ~LOW) | (low0 - j);
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) key[j] = (key_of(l[j] + 0.f) & ~LOW) | (low0 - j);     // -0 is 0
    }
    uint32_t head[K::DEPTH];
    largest<V, K::DEPTH>(key, head);
    uint32_t rest = V > K::DEPTH && head[K::DEPTH - 1] > K::NONE ? K::MORE : 0u;
    constexpr float SPREAD = SCORES ? (float)(1u << K::PLACE_BITS) * 0x1p-21f : 0.f;
    bool sure = true;
    if (a.groups > 1) {
        uint32_t b1 = head[0], b2 = K::DEPTH > 1 ? head[K::DEPTH > 1 ? 1 : 0] : 0u;
        for (int off = a.lanes >> 1; off >= 1; off >>= 1) {
            const uint32_t o1 = __shfl_xor_sync(0xffffffffu, b1, off), o2 = __shfl_xor_sync(0xffffffffu, b2, off);
            b2 = max(min(b1, o1), max(b2, o2));
            b1 = max(b1, o1);
        }
        uint32_t group = b1;
        float size = SCORES && b1 > K::NONE ? fabsf(value_of(b1 & ~LOW)) : 0.f;     // what the sum's uncertainty goes by
        if (SCORES && a.group_best == 2 && b2 > K::NONE) {
            group = key_of(value_of(b1 & ~LOW) + value_of(b2 & ~LOW));
            size += fabsf(value_of(b2 & ~LOW));
        }
        group = b1 > K::NONE ? (group & ~31u) | (31 - (lane >> a.lanes_log2)) : 0u;
        uint32_t left = group, last = 0u;
        for (int i = 0; i < a.top_groups; ++i) {
            last = __reduce_max_sync(0xffffffffu, left);
            left = left == last ? 0u : left;
        }
        const uint32_t next = __reduce_max_sync(0xffffffffu, left);
        if (next) {
            if constexpr (SCORES) {
                size = __uint_as_float(__reduce_max_sync(0xffffffffu, group >= next ? __float_as_uint(size) : 0u));
                sure = value_of(last & ~31u) - value_of(next & ~31u) > 2.f * uncertain + size * (SPREAD + 0x1p-16f);
            } else {
                sure = WHOLE || (last >> 5) != (next >> 5);
            }
        }
        if (group < last || group == 0u) {
#pragma unroll
            for (int i = 0; i < K::DEPTH; ++i) head[i] = 0u;
            rest = 0u;
        }
    }
    // Rounds, one past the last expert (and up to two more).  Lanes whose heads are equal move on together: the keys that are lost so
    // are counted, and leave it undecided.
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(found);
    if (lane < MAX_ROUNDS) found[lane] = make_uint2(0u, 0u);
    __syncwarp();
    int taken = 0;
#pragma unroll
    for (int i = 0; i < MAX_ROUNDS; ++i) {
        if (i % 3 == 0 && i > a.k) break;
        const uint32_t top = __reduce_max_sync(0xffffffffu, head[0]);
        take_head<K::DEPTH>(head, rest, taken, top, K::NONE, at, i, (uint32_t)base);
    }
    __syncwarp();
    const uint2 choice = lane < MAX_ROUNDS ? found[lane] : make_uint2(0u, 0u);
    const uint32_t best = choice.x, after = __shfl_down_sync(0xffffffffu, best, 1);
    const int rounds = __popc(__ballot_sync(0xffffffffu, best != 0u));
    __syncwarp();
    sure = sure && (lane > a.k || best != K::MORE);
    if (!WHOLE && lane < a.k && after) {
        if constexpr (SCORES) {
            const float high = value_of(best & ~LOW);
            sure = sure && high - value_of(after & ~LOW) > uncertain + fabsf(high) * SPREAD;
        } else {
            sure = sure && (best & ~LOW) != (after & ~LOW);
        }
    }
    if (__reduce_add_sync(0xffffffffu, (unsigned)taken + (sure ? 0u : 1u << 16)) != (unsigned)rounds) return false;
    mine = lane < a.k && best ? (int)(choice.y + ((LOW - (best & LOW)) & (V - 1))) : -1;
    return true;
}

// Weights of chosen experts, and the answer.  `width` lanes, a power of two, have the experts of one token (-1: none), rank r in
// the r-th of them; whole: the row's largest logit and sum of exponentials, for softmax weights that are not renormalised.
// Renormalised weights are computed from the chosen logits alone, relative to the largest, so they do not vanish
// where all scores do.
template <typename T>
__device__ __forceinline__ void store_choice(const SelectArgs& a, long long t, int r, int mine, int width, bool live, float2 whole) {
    const T* row = static_cast<const T*>(a.logits) + t * a.ld;
    const float l = live && mine >= 0 ? to_float(row[mine]) : -INFINITY;
    float w = 0.f;
    if (a.renormalise) {
        float top = l;
        for (int off = width >> 1; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        if (a.sigmoid && !(top > 0.f))
            w = mine >= 0 ? expf(l - top) / (1.f + expf(l)) : 0.f;
        else if (a.sigmoid)
            w = mine >= 0 ? 1.f / (1.f + expf(-l)) : 0.f;
        else
            w = mine >= 0 ? (l == top ? 1.f : expf(l - top)) : 0.f;
        float sum = w;
        for (int off = width >> 1; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        w = mine >= 0 ? w / sum : 0.f;
    } else if (a.sigmoid) {
        w = mine >= 0 ? 1.f / (1.f + expf(-l)) : 0.f;
    } else {
        w = mine >= 0 ? (l == whole.x ? 1.f : expf(l - whole.x)) / whole.y : 0.f;
    }
    if (live && r < a.k) {
        a.gate[t * a.k + r] = mine;
        a.weight[t * a.k + r] = w * a.scale;
        if (r == 0 && mine < 0 && a.status) atomicOr(a.status, STATUS_NO_EXPERT);
    }
}

// The lane's V logits of a row; -inf for an expert that is not there, or (MASK) cannot be chosen.
template <typename T, int V, bool MASK>
__device__ __forceinline__ void load_logits(const SelectArgs& a, long long t, int first, int count, float (&l)[V]) {
    const T* row = static_cast<const T*>(a.logits) + t * a.ld + first;
    constexpr int N = V * sizeof(T) >= 16 ? 16 / (int)sizeof(T) : V;
    if (a.vec && V * sizeof(T) >= 16) {
#pragma unroll
        for (int j = 0; j < V; j += N) {
            float e[N];
            load_elems<T, N>(row + j, e);
#pragma unroll
            for (int i = 0; i < N; ++i) l[j + i] = e[i];
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) l[j] = j < count ? to_float(row[j]) : -INFINITY;
    }
    if constexpr (MASK)
#pragma unroll
        for (int j = 0; j < V; ++j) l[j] = l[j] > Lowest<T>::value() ? l[j] : -INFINITY;    // NaN too
}

// A warp per token, tokens a grid apart, 32 to a warp before the block meets.  As many tokens as fit into the lanes (four with 5 to
// 8 experts each) then get their weights together: by token that took 10 of 45 us (65536 tokens, 8 of 256 experts).  Tokens
// that 32 bits leave undecided wait until the block's are done, and its warps share them; in the loop itself that choice cost every
// token its registers, 20 us, and by each warp after a few tokens 4 us more than so.  Of 59 us the undecided 149 take 9 (5 to 14 more
// by all threads of a block, an expert to each).
template <typename T, int V, ChosenBy BY>
__global__ void __launch_bounds__(SELECT_WARPS * 32, V <= 8 ? 4 : V <= 16 ? 3 : 2) select_topk_kernel(const __grid_constant__ SelectArgs a) {
    __shared__ uint2 s_found[SELECT_WARPS][MAX_ROUNDS];
    __shared__ int s_choice[SELECT_WARPS][32];
    __shared__ float2 s_row[SELECT_WARPS][32];                      // softmax of all experts, by turn: the largest logit, and the sum
    __shared__ int s_open[SELECT_WARPS * 32], s_open_count;         // undecided tokens: warp and turn
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> a.lanes_log2, place = (lane & (a.lanes - 1)) * V;
    const int first = g * a.group_size + place, count = g < a.groups ? a.group_size - place : 0;    // its experts
    float bias[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        bias[j] = BY != LOGITS && a.bias && j < count ? a.bias[first + j] : 0.f;
        if (bias[j] != bias[j]) bias[j] = -INFINITY;
    }
    const long long step = (long long)gridDim.x * SELECT_WARPS;
    const int width = 1 << a.width_log2, batch = 32 >> a.width_log2, r = lane & (width - 1);
    const bool whole_sum = !a.sigmoid && !a.renormalise;
    for (long long t0 = (long long)blockIdx.x * SELECT_WARPS; t0 < a.T; t0 += 32 * step) {      // the block's next 32 turns
        if (threadIdx.x == 0) s_open_count = 0;
        __syncthreads();
        for (int turn = 0; turn < 32 && t0 + warp + turn * step < a.T; turn += batch) {
            s_choice[warp][lane] = -2;
            __syncwarp();
            long long t = t0 + warp + turn * step;
            for (int i = 0; i < batch && t < a.T; ++i, t += step) {
                float l[V];
                load_logits<T, V, BY != SIGMOID>(a, t, first, count, l);
                if (BY != SIGMOID && whole_sum) {
                    float top = l[0], sum = 0.f;
#pragma unroll
                    for (int j = 1; j < V; ++j) top = fmaxf(top, l[j]);
                    top = warp_max(top);
#pragma unroll
                    for (int j = 0; j < V; ++j) sum += l[j] == top ? 1.f : expf(l[j] - top);
                    sum = warp_xor_sum(sum);
                    if (lane == 0) s_row[warp][turn + i] = make_float2(top, sum);
                }
                int mine = -1;
                if (a.k <= MAX_FAST_K && select_in_32_bits<T, V, BY>(a, l, bias, lane, first, s_found[warp], mine)) {
                    if (lane < width) s_choice[warp][i * width + lane] = mine;
                } else if (lane == 0) {
                    s_open[atomicAdd(&s_open_count, 1)] = warp * 32 + turn + i;
                }
            }
            __syncwarp();
            const int mine = s_choice[warp][lane], i = turn + (lane >> a.width_log2);
            store_choice<T>(a, min(t0 + warp + i * step, a.T - 1), r, mine, width, mine != -2, s_row[warp][i]);
            __syncwarp();
        }
        __syncthreads();
        const int open = s_open_count;
        for (int i = warp; i < open; i += SELECT_WARPS) {
            const int of = s_open[i] >> 5, turn = s_open[i] & 31;
            const long long t = t0 + of + turn * step;
            const int mine = select_in_64_bits<T, V>(a, t, lane);
            store_choice<T>(a, t, lane, mine, 32, true, s_row[of][turn]);
        }
        __syncthreads();
    }
}

template <typename T, int V, ChosenBy BY>
int launch_select_kernel(const SelectArgs& a, cudaStream_t stream) {
    const long long blocks = (a.T + SELECT_WARPS - 1) / SELECT_WARPS, most = 148 * (V <= 8 ? 4 : V <= 16 ? 3 : 2);   // as many as run at once
    INFMOE_CUDA_TRY(launch_chained(select_topk_kernel<T, V, BY>, (unsigned)(blocks < most ? blocks : most), SELECT_WARPS * 32, 0, 1,
                                   stream, a));
    note_launch();
    INFMOE_CUDA_TRY(cudaGetLastError());
    return INFMOE_OK;
}

template <typename T, int V>
int launch_select(SelectArgs a, cudaStream_t stream) {
    constexpr int bytes = V * (int)sizeof(T) < 16 ? V * (int)sizeof(T) : 16;
    a.vec = a.group_size == a.lanes * V && a.groups * a.lanes == 32 && (uintptr_t)a.logits % bytes == 0 &&
            a.ld * (long long)sizeof(T) % bytes == 0;
    if (!a.bias && (a.groups == 1 || a.group_best == 1)) return launch_select_kernel<T, V, LOGITS>(a, stream);
    if (a.sigmoid) return launch_select_kernel<T, V, SIGMOID>(a, stream);
    return launch_select_kernel<T, V, SOFTMAX>(a, stream);
}

template <typename T>
int launch_select_type(const SelectArgs& a, int per_lane, cudaStream_t stream) {
    if (per_lane <= 1) return launch_select<T, 1>(a, stream);
    if (per_lane <= 2) return launch_select<T, 2>(a, stream);
    if (per_lane <= 4) return launch_select<T, 4>(a, stream);
    if (per_lane <= 8) return launch_select<T, 8>(a, stream);
    if (per_lane <= 16) return launch_select<T, 16>(a, stream);
    return launch_select<T, 32>(a, stream);
}

// ---- rows to k experts and back ------------------------------------------------------------------

constexpr int ROW_THREADS = 256;
constexpr int MAX_TOKEN_LEN = 65535 * ROW_THREADS;   // parts of a row that a grid's second dimension can count, one element to a thread

// How a block of ROW_THREADS shares out rows of `vecs` vectors: rows_per_block whole rows, or (one row per block) parts of a
// row along grid.y.
struct RowSplit {
    int vecs, rows_per_block;
};

// routed[j] = x[pos[j] / k] and row_of[pos[j]] = j for the rows j below *valid_rows; row_of = -1 for the slots of the others.
// pos NULL: row j is slot j; valid_rows NULL: all rows.  A thread copies one vector of each of ROWS rows, all of them in flight.
template <typename Vec, int ROWS>
__global__ void __launch_bounds__(ROW_THREADS)
scatter_topk_kernel(long long rows, int k, RowSplit split, const Vec* x, long long ldx, const int* pos, const int* valid_rows,
                    Vec* __restrict__ routed, int* __restrict__ row_of) {
    pdl_wait();
    pdl_trigger();
    int local = 0, v = (int)threadIdx.x + (int)blockIdx.y * ROW_THREADS;
    if (split.rows_per_block > 1) {
        local = v / split.vecs;
        v -= local * split.vecs;
    }
    if (local >= split.rows_per_block || v >= split.vecs) return;
    const long long first = (long long)blockIdx.x * split.rows_per_block * ROWS + local, valid = valid_rows ? *valid_rows : rows;
    int slot[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const long long j = first + (long long)i * split.rows_per_block;
        slot[i] = j < rows ? (pos ? pos[j] : (int)j) : -1;
    }
    Vec value[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const long long j = first + (long long)i * split.rows_per_block;
        if (slot[i] >= rows) slot[i] = -1;
        if (slot[i] >= 0 && j < valid) value[i] = x[(long long)((unsigned)slot[i] / (unsigned)k) * ldx + v];
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const long long j = first + (long long)i * split.rows_per_block;
        if (slot[i] < 0) continue;
        if (v == 0 && row_of) row_of[slot[i]] = j < valid ? (int)j : -1;
        if (j < valid) routed[j * split.vecs + v] = value[i];
    }
}

// out[t] = sum_s w[t][s] y[row_of[t][s]] (+ (1 - sum_s w[t][s]) x[t]), slots without a row left out: a row outside [0, rows),
// or a gate outside [0, gates).
template <typename T, int N, bool RESIDUAL>
__global__ void __launch_bounds__(ROW_THREADS)
combine_topk_kernel(long long tokens, int k, RowSplit split, const T* y, long long rows, const float* weight, const int* gate,
                    unsigned gates, const int* row_of, const T* x, T* __restrict__ out) {
    pdl_trigger();
    pdl_wait();
    int local = 0, v = (int)threadIdx.x + (int)blockIdx.y * ROW_THREADS;
    if (split.rows_per_block > 1) {
        local = v / split.vecs;
        v -= local * split.vecs;
    }
    const long long t = (long long)blockIdx.x * split.rows_per_block + local;
    if (local >= split.rows_per_block || v >= split.vecs || t >= tokens) return;
    const long long D = (long long)split.vecs * N;
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    float rest = 1.f;
    for (int s = 0; s < k; ++s) {
        const long long slot = t * k + s;
        const long long row = row_of ? row_of[slot] : slot;
        if (row < 0 || row >= rows || (gate && (unsigned)gate[slot] >= gates)) continue;
        const float w = weight[slot];
        rest -= w;
        float e[N];
        load_elems<T, N>(y + row * D + (long long)v * N, e);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = fmaf(w, e[i], acc[i]);
    }
    if (RESIDUAL) {
        float e[N];
        load_elems<T, N>(x + t * D + (long long)v * N, e);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = fmaf(rest, e[i], acc[i]);
    }
    store_elems<T, N>(out + t * D + (long long)v * N, acc);
}

bool aligned(const void* p, size_t bytes) { return ((uintptr_t)p % bytes) == 0; }

RowSplit row_split(long long vecs) {
    return RowSplit{(int)vecs, vecs >= ROW_THREADS ? 1 : (int)(ROW_THREADS / vecs)};
}
dim3 row_split_grid(const RowSplit& s, long long rows) {
    return dim3((unsigned)((rows + s.rows_per_block - 1) / s.rows_per_block),
                s.rows_per_block > 1 ? 1u : (unsigned)((s.vecs + ROW_THREADS - 1) / ROW_THREADS));
}

template <typename Vec, int ROWS>
int launch_scatter_topk_rows(long long rows, int k, long long row_bytes, const void* x, long long ldx_bytes, const int* pos,
                             const int* valid_rows, void* routed, int* row_of, cudaStream_t stream) {
    const RowSplit s = row_split(row_bytes / (long long)sizeof(Vec));
    INFMOE_CUDA_TRY(launch_chained_2d(scatter_topk_kernel<Vec, ROWS>, row_split_grid(s, (rows + ROWS - 1) / ROWS), ROW_THREADS, stream,
                                      rows, k, s, (const Vec*)x, ldx_bytes / (long long)sizeof(Vec), pos, valid_rows, (Vec*)routed,
                                      row_of));
    note_launch();
    INFMOE_CUDA_TRY(cudaGetLastError());
    return INFMOE_OK;
}

template <typename Vec>
int launch_scatter_topk_vec(long long rows, int k, long long row_bytes, const void* x, long long ldx_bytes, const int* pos,
                            const int* valid_rows, void* routed, int* row_of, cudaStream_t stream) {
    // Four vectors to a thread where there is enough to do for all of them (32768 rows of 8 KB: one 82 us, two 61, four 57, eight 66;
    // four of one row instead of four rows: 16384 rows of 16 KB 69 instead of 60); one where blocks are few (512 rows of 8 KB: 4.7 us
    // either way, 64: 2.4).
    if (rows * row_bytes > (8 << 20))
        return launch_scatter_topk_rows<Vec, 4>(rows, k, row_bytes, x, ldx_bytes, pos, valid_rows, routed, row_of, stream);
    return launch_scatter_topk_rows<Vec, 1>(rows, k, row_bytes, x, ldx_bytes, pos, valid_rows, routed, row_of, stream);
}

template <typename T, int N>
int launch_combine_topk_vec(long long tokens, int k, int D, const void* y, long long rows, const float* weight, const int* gate,
                            unsigned gates, const int* row_of, const void* x, void* out, cudaStream_t stream) {
    const RowSplit s = row_split(D / N);
    const dim3 grid = row_split_grid(s, tokens);
    if (x)
        INFMOE_CUDA_TRY(launch_chained_2d(combine_topk_kernel<T, N, true>, grid, ROW_THREADS, stream, tokens, k, s, (const T*)y,
                                          rows, weight, gate, gates, row_of, (const T*)x, (T*)out));
    else
        INFMOE_CUDA_TRY(launch_chained_2d(combine_topk_kernel<T, N, false>, grid, ROW_THREADS, stream, tokens, k, s,
                                          (const T*)y, rows, weight, gate, gates, row_of, (const T*)x, (T*)out));
    note_launch();
    INFMOE_CUDA_TRY(cudaGetLastError());
    return INFMOE_OK;
}

template <typename T>
int launch_combine_topk_type(long long tokens, int k, int D, const void* y, long long rows, const float* weight,
                             const int* gate, unsigned gates, const int* row_of, const void* x, void* out, cudaStream_t stream) {
    constexpr int N = 16 / (int)sizeof(T);
    if (D % N == 0 && aligned(y, 16) && aligned(out, 16) && (!x || aligned(x, 16)))
        return launch_combine_topk_vec<T, N>(tokens, k, D, y, rows, weight, gate, gates, row_of, x, out, stream);
    return launch_combine_topk_vec<T, 1>(tokens, k, D, y, rows, weight, gate, gates, row_of, x, out, stream);
}

}  // namespace

int launch_scatter_topk(long long rows, int k, int D, int elem_bytes, const void* x, long long ldx, const int* pos,
                        const int* valid_rows, void* routed, int* row_of, cudaStream_t stream) {
    const long long row_bytes = (long long)D * elem_bytes, ldx_bytes = ldx * elem_bytes;
    if (row_bytes % 16 == 0 && ldx_bytes % 16 == 0 && aligned(x, 16) && aligned(routed, 16))
        return launch_scatter_topk_vec<uint4>(rows, k, row_bytes, x, ldx_bytes, pos, valid_rows, routed, row_of, stream);
    if (row_bytes % 4 == 0 && ldx_bytes % 4 == 0 && aligned(x, 4) && aligned(routed, 4))
        return launch_scatter_topk_vec<uint32_t>(rows, k, row_bytes, x, ldx_bytes, pos, valid_rows, routed, row_of, stream);
    return launch_scatter_topk_vec<uint16_t>(rows, k, row_bytes, x, ldx_bytes, pos, valid_rows, routed, row_of, stream);
}

int launch_combine_topk(long long tokens, int k, int D, int dtype, const void* y, long long rows, const float* weight,
                        const int* gate, unsigned gates, const int* row_of, const void* x, void* out, cudaStream_t stream) {
    if (dtype == INFMOE_F32)
        return launch_combine_topk_type<float>(tokens, k, D, y, rows, weight, gate, gates, row_of, x, out, stream);
    if (dtype == INFMOE_F16)
        return launch_combine_topk_type<__half>(tokens, k, D, y, rows, weight, gate, gates, row_of, x, out, stream);
    return launch_combine_topk_type<__nv_bfloat16>(tokens, k, D, y, rows, weight, gate, gates, row_of, x, out, stream);
}

}  // namespace infmoe

using namespace infmoe;

extern "C" {

int infmoe_expert_select_topk(const infmoe_topk_config* cfg, int64_t T, const void* d_logits, int32_t dtype, int64_t ld,
                              const float* d_bias, int32_t* d_gate, float* d_weight, int32_t* d_status, void* stream) {
    if (!cfg || T < 0 || T > 0x7fffffffLL || !known_dtype(dtype) || (T > 0 && (!d_logits || !d_gate || !d_weight))) {
        set_error("expert_select_topk: bad argument (T=%lld dtype=%d)", (long long)T, dtype);
        return INFMOE_ERR_INVALID_ARGUMENT;
    }
    const int E = cfg->expert_count, k = cfg->top_k, G = cfg->group_count;
    if (E <= 0 || ld < E || G <= 0 || G > E || E % G != 0 || cfg->top_groups <= 0 || cfg->top_groups > G || k <= 0 ||
        (int64_t)k > (int64_t)cfg->top_groups * (E / G) || (cfg->group_best != 1 && cfg->group_best != 2) ||
        (cfg->score != INFMOE_SCORE_SOFTMAX && cfg->score != INFMOE_SCORE_SIGMOID)) {
        set_error("expert_select_topk: bad configuration (experts %d, groups %d, top groups %d, top_k %d, best of a group %d, "
                  "score %d, row stride %lld)", E, G, cfg->top_groups, k, cfg->group_best, cfg->score, (long long)ld);
        return INFMOE_ERR_INVALID_ARGUMENT;
    }
    int padded = 1;
    while (padded < G) padded *= 2;
    const int size = E / G, lanes = padded <= 32 ? 32 / padded : 0;
    if (k > 32 || lanes == 0 || (size + lanes - 1) / lanes > 32) {
        set_error("expert_select_topk: at most 32 experts to a token, 32 groups and 32 experts to a lane (experts %d, groups %d, "
                  "top_k %d)", E, G, k);
        return INFMOE_ERR_UNSUPPORTED;
    }
    if (T == 0) return INFMOE_OK;
    SelectArgs a{};
    a.logits = d_logits;
    a.T = T;
    a.ld = ld;
    a.E = E;
    a.k = k;
    a.groups = G;
    a.top_groups = cfg->top_groups;
    a.group_best = cfg->group_best;
    a.group_size = size;
    a.lanes = lanes;
    a.lanes_log2 = 0;
    while ((1 << a.lanes_log2) < lanes) ++a.lanes_log2;
    while ((1 << a.width_log2) < k) ++a.width_log2;      // lanes that hold the experts of a token
    a.sigmoid = cfg->score == INFMOE_SCORE_SIGMOID;
    a.renormalise = cfg->renormalise != 0;
    a.scale = cfg->scale;
    a.bias = d_bias;
    a.gate = d_gate;
    a.weight = d_weight;
    a.status = d_status;
    const int per_lane = (size + lanes - 1) / lanes;
    if (dtype == INFMOE_F32) return launch_select_type<float>(a, per_lane, (cudaStream_t)stream);
    if (dtype == INFMOE_F16) return launch_select_type<__half>(a, per_lane, (cudaStream_t)stream);
    return launch_select_type<__nv_bfloat16>(a, per_lane, (cudaStream_t)stream);
}

int infmoe_expert_scatter_topk(int64_t T, int32_t top_k, int32_t token_len, int32_t dtype, const void* d_input, int64_t ld,
                               const int32_t* d_pos, const int32_t* d_valid_rows, void* d_routed, int32_t* d_row_of,
                               void* stream) {
    if (T < 0 || top_k <= 0 || token_len <= 0 || ld < token_len || !known_dtype(dtype) ||
        (T > 0 && (!d_input || !d_pos || !d_valid_rows || !d_routed))) {
        set_error("expert_scatter_topk: bad argument (T=%lld top_k=%d token_len=%d row stride %lld dtype=%d)", (long long)T, top_k,
                  token_len, (long long)ld, dtype);
        return INFMOE_ERR_INVALID_ARGUMENT;
    }
    if (T > 0x7fffffffLL / top_k || token_len > MAX_TOKEN_LEN) {
        set_error("expert_scatter_topk: %lld tokens of %d slots are too many for 32-bit slot indices, or rows of %d elements too long",
                  (long long)T, top_k, token_len);
        return INFMOE_ERR_UNSUPPORTED;
    }
    if (T == 0) return INFMOE_OK;
    return launch_scatter_topk(T * top_k, top_k, token_len, dtype_bytes(dtype), d_input, ld, d_pos, d_valid_rows, d_routed,
                               d_row_of, (cudaStream_t)stream);
}

int infmoe_expert_combine_topk(int64_t T, int32_t top_k, int32_t token_len, int32_t dtype, const void* d_rows, int64_t rows,
                               const float* d_weight, const int32_t* d_gate, const int32_t* d_row_of, const void* d_residual,
                               void* d_output, void* stream) {
    if (T < 0 || rows < 0 || top_k <= 0 || token_len <= 0 || !known_dtype(dtype) ||
        (T > 0 && ((rows > 0 && !d_rows) || !d_weight || !d_output)) || (T > 0 && d_rows == d_output)) {
        set_error("expert_combine_topk: bad argument (T=%lld rows=%lld top_k=%d token_len=%d dtype=%d)", (long long)T,
                  (long long)rows, top_k, token_len, dtype);
        return INFMOE_ERR_INVALID_ARGUMENT;
    }
    if (T > 0x7fffffffLL / top_k || token_len > MAX_TOKEN_LEN) {
        set_error("expert_combine_topk: %lld tokens of %d slots are too many for 32-bit slot indices, or rows of %d elements too long",
                  (long long)T, top_k, token_len);
        return INFMOE_ERR_UNSUPPORTED;
    }
    if (T == 0) return INFMOE_OK;
    return launch_combine_topk(T, top_k, token_len, dtype, d_rows, rows, d_weight, d_gate, 0x80000000u, d_row_of, d_residual,
                               d_output, (cudaStream_t)stream);
}

}  // extern "C"

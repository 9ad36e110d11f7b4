// Drawing items from a user's logits over the catalogue, by given uniform numbers.
//
// For a row of logits x, allowed items a (mask set, x neither NaN nor -inf), m = max x over a:
//   1. top-k   the k best, best first, equals in the order of their ids; k <= 0: all.
//              temperature t <= 0 (or NaN): k = 1
//   2. weight  w = exp((x - m) / t), and 1 where x = m
//   3. top-p   of them the shortest leading list with at least p of their weight; p <= 0: one item,
//              p >= 1: all
//   4. min-p   of it the items with w >= min_p
//   5. draw    the first item, in the order of the ids, at which the running sum of the weights
//              passes u times their total.
// Each step keeps a leading part of the same order (x descending, id ascending), so what a row keeps
// is described by a bound: all items above it, and the first `ties` of those equal to it.
//
// Weights are held as integers, round(w 2^S) with S = min(51, 62 - ceil(log2 n)): their sums are
// exact and the same in any order, so neither the split over lanes nor the order of atomics can
// change a draw, and a running sum can never pass the total.  Each weight is off by half a unit at most, so a
// running sum of n by n 2^-(S + 1) of the total (which is at least 1): the draw differs from real arithmetic only
// where u lands within n 2^-S of a border, 2^-22 at 1,000,000 items (S = 42), 2^-32 at 27,278 (S = 47).  An item
// of less than half a unit is never drawn.  w itself is computed in 64 bits.
//
// The reference keeps the best of a list by np.argsort (movierec/trt_client.py:50-57); drawing from
// the scores is an extension of that ranking.

#include <algorithm>
#include <cmath>

#include "ncf_common.h"
#include "ncf_internal.h"
#include "ncf_types.h"

namespace ncf {

struct DrawArgs {
    const void* logits;
    const uint8_t* mask;      // [rows][n] bytes, 0 = not allowed; NULL: all allowed
    int64_t ld, mask_ld;
    int64_t rows;
    int n, draws;
    const double* u;          // one of these two, [rows][draws]
    const float* u32;
    const float* temperature; // [rows] or NULL: the value below
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    double temperature_v, top_p_v, min_p_v;
    int32_t top_k_v;
    double unit;              // 2^S
    int32_t* items;
    float* probs;
};

// ----------------------------------------------------------------------------- keys and weights

// unsigned keys in the order of the floats
__device__ __forceinline__ uint32_t ukey(float x) {
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unukey(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

// w = exp(z), z = (x - m) / t, as an integer in units of 2^-S.  With z = (j + r) ln 2 / 2^BITS, |r| <= 1 / 2,
// w = 2^(j / 2^BITS) e^(r ln 2 / 2^BITS): the power of two from a table in LDS (its whole part into the exponent),
// the rest by its Taylor polynomial, to the third power for a table of 2,048 and to the fourth for one of 256
// (the next term is below 2^-54 in both).  Adding 1.5 2^52 rounds to j, adding 2^52 to the integer.  About 17
// instructions; exp() and a conversion take about 50.  A long row's workgroups of 1,024 fill the larger table
// (weights of 16 rows of 1,000,000: 24 us with 256 powers), a row in registers the smaller.
template <int BITS>
struct Weigher {
    static constexpr int kPowers = 1 << BITS;
    double m, a, unit;     // a = 2^BITS / (t ln 2), finite
    const double* power;   // [kPowers], times unit

    __device__ __forceinline__ Weigher(float top, double t, double unit, const double* power)
        // (under an infinite best item every finite one weighs nothing)
        : m(top < INFINITY ? (double)top : 1e300), a(fmin(1.0 / t, 1e280) * (kPowers * 1.4426950408889634074)),
          unit(unit), power(power) {}

    // w 2^S = e p
    __device__ __forceinline__ void factors(float x, double& e, double& p) const {
        constexpr double kMagic = 0x1.8p52, kStep = 0.69314718055994530942 / kPowers;
        // (at -60 less than half a unit; a NaN, of an infinite best item in an infinite temperature, becomes 0)
        const double y = fmax(fmin(((double)x - m) * a, 0.0), -60.0 * kPowers * 1.4426950408889634074);
        const double j = y + kMagic, r = y - (j - kMagic);
        e = BITS < 11 ? fma(r, kStep * kStep * kStep * kStep / 24.0, kStep * kStep * kStep / 6.0)
                      : kStep * kStep * kStep / 6.0;
        e = fma(r, e, kStep * kStep / 2.0);
        e = fma(r, e, kStep);
        e = fma(r, e, 1.0);
        const uint32_t n = (uint32_t)__double_as_longlong(j);
        p = power[n & (kPowers - 1)];
        p = __hiloint2double(__double2hiint(p) + (int)((n & ~(uint32_t)(kPowers - 1)) << (20 - BITS)),
                             __double2loint(p));
    }
    __device__ __forceinline__ static unsigned long long round(double e, double p) {
        return (unsigned long long)__double_as_longlong(fma(e, p, 0x1p52)) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ unsigned long long fixed(float x) const {
        double e, p;
        factors(x, e, p);
        return round(e, p);
    }
    // 0 where the weight does not reach `least`, which is min-p's
    __device__ __forceinline__ unsigned long long fixed(float x, unsigned long long least) const {
        const unsigned long long w = fixed(x);
        return w >= least ? w : 0ull;
    }
    __device__ __forceinline__ unsigned long long least(double min_p) const {
        return min_p > 0.0 ? (unsigned long long)ceil(min_p * unit) : 0ull;
    }
};
constexpr int kRowPowers = 8, kLongPowers = 11;   // BITS of a row in registers, and of a long one

template <int BITS>
__device__ __forceinline__ void fill_powers(double (&power)[1 << BITS], double unit, int threads) {
    for (int j = threadIdx.x; j < 1 << BITS; j += threads) power[j] = exp2(j * (1.0 / (1 << BITS))) * unit;
}

// (double)c >= p total, for a positive c: the one comparison that top-p makes
__device__ __forceinline__ bool reaches(unsigned long long c, double p, double total) {
    return c > 0 && (double)c >= p * total;
}

// ----------------------------------------------------------------------------- rows held in registers
//
// A workgroup of NT threads holds a row of up to EPT NT logits in registers (-inf: not allowed), each
// wave a contiguous part of it, reads it once, and works from there.  The bound of top-k (top-p) is
// found in two steps: a histogram of counts (weights) over 2 NT bins that are equal steps of the logit
// from the best down, which names the bin where the k-th item (the p-th part of the weight) lies; then
// that bin's few items are ranked against each other, one a thread.  A bin with more than NT items (many
// equal logits) goes digit by digit of the key instead.
// For top-k with k <= 4 NT the histogram sees one of V neighbours only and gives a limit that the k best
// most likely pass; the items that pass it, if they are at least k and at most 4 NT, move to a list in LDS
// in the order of the ids, and the row is not looked at again.  (Otherwise the whole row is counted.)
// 2,048 rows of 27,278 fp32 with a mask, top-1,000, top-p, min-p: 101 us, 2.8 TB/s: a row's
// barriers, LDS and ballots, which only the CU's other workgroup overlaps.  One row: 15 us.

__device__ __forceinline__ int lane_count(uint64_t mask) { return (int)__popcll(mask); }
// set bits of the mask below this lane, plus `more`
__device__ __forceinline__ uint32_t lanes_before(uint64_t mask, uint32_t more) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, more));
}

// inclusive sums over the lanes of a wave by data-parallel moves: within rows of 16, then across rows
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved32(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t lane_sums32(uint32_t x) {
    x += moved32<0x111, 0xf>(x);
    x += moved32<0x112, 0xf>(x);
    x += moved32<0x114, 0xf>(x);
    x += moved32<0x118, 0xf>(x);
    x += moved32<0x142, 0xa>(x);
    x += moved32<0x143, 0xc>(x);
    return x;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long moved64(unsigned long long x) {
    return (unsigned long long)moved32<CTRL, ROWS>((uint32_t)(x >> 32)) << 32 | moved32<CTRL, ROWS>((uint32_t)x);
}
__device__ __forceinline__ unsigned long long lane_sums64(unsigned long long x) {
    x += moved64<0x111, 0xf>(x);
    x += moved64<0x112, 0xf>(x);
    x += moved64<0x114, 0xf>(x);
    x += moved64<0x118, 0xf>(x);
    x += moved64<0x142, 0xa>(x);
    x += moved64<0x143, 0xc>(x);
    return x;
}
__device__ __forceinline__ uint32_t lane63(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)x, 63); }
__device__ __forceinline__ unsigned long long lane63(unsigned long long x) {
    return (unsigned long long)lane63((uint32_t)(x >> 32)) << 32 | lane63((uint32_t)x);
}

template <int NT>
struct RowShared {
    static constexpr int kBins = 2 * NT, kWaves = NT / 64, kPer = 4, kList = kPer * NT;
    union {
        uint32_t count[kBins];
        unsigned long long weight[kBins];
        unsigned long long before[kList];   // the list's running sums
    };
    float list_x[kList + 64];   // behind the list a place for what does not belong there, one a lane
    uint32_t list_id[kList + 64];
    unsigned long long member_w[NT];
    float member_x[NT];
    uint32_t member_id[NT];
    uint32_t members;
    float bound;
    uint32_t pick_bin, ties, equal;
    unsigned long long pick;
    unsigned long long wave64[kWaves];
    uint32_t wave32[kWaves];
    float wave_top[kWaves], wave_sum[kWaves], wave_n[kWaves];
    unsigned long long seg[NT / 4];         // weights ahead of each segment of the row: a wave's vector j
    uint32_t seg_ties[NT / 4];              // equals of the bound ahead of it
    double power[1 << kRowPowers];
};

// exclusive sums over the workgroup, the total to *sum
template <int NT>
__device__ __forceinline__ unsigned long long before64(unsigned long long v, RowShared<NT>& s,
                                                       unsigned long long* sum) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const unsigned long long inc = lane_sums64(v);
    if constexpr (NT == 64) {
        *sum = lane63(inc);
        return inc - v;
    }
    __syncthreads();
    if (lane == 63) s.wave64[w] = inc;
    __syncthreads();
    unsigned long long before = 0, all = 0;
#pragma unroll
    for (int j = 0; j < NT / 64; ++j) {
        const unsigned long long o = s.wave64[j];
        before += j < w ? o : 0ull;
        all += o;
    }
    *sum = all;
    return before + inc - v;
}

template <int NT>
__device__ __forceinline__ uint32_t before32(uint32_t v, RowShared<NT>& s, uint32_t* sum) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint32_t inc = lane_sums32(v);
    if constexpr (NT == 64) {
        *sum = lane63(inc);
        return inc - v;
    }
    __syncthreads();
    if (lane == 63) s.wave32[w] = inc;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int j = 0; j < NT / 64; ++j) {
        const uint32_t o = s.wave32[j];
        before += j < w ? o : 0u;
        all += o;
    }
    *sum = all;
    return before + inc - v;
}

// bins of equal width from the best logit down; what lies below the range shares the last
struct Bins {
    float top, scale, last;
    __device__ __forceinline__ int of(float x) const {
        return (int)fminf((top - x) * scale, last);   // (infinities on both sides: NaN, the last bin)
    }
    // every item of a bin up to b lies above this: the bin's lower edge, less the roundings of of()
    __device__ __forceinline__ float below(int b) const {
        if ((float)b >= last) return -3.402823466e38f;
        const float width = (float)(b + 1) / scale;
        return top - width - (fabsf(top) + width) * 0x1p-21f;
    }
};
__device__ __forceinline__ Bins make_bins(float top, float range, int bins) {
    range = range > 1e-30f && range < 1e30f ? range : 1.0f;
    return Bins{top, (float)bins / range, (float)(bins - 1)};
}

// what a row keeps: every item above `bound` and the first `ties` (in the order of the ids) equal to it
struct Cut {
    float bound;
    uint32_t ties;
    bool partial;   // more items equal the bound than `ties`
    uint32_t equal; // how many do (0: not known)
};
constexpr uint32_t kAllTies = 0xffffffffu;
__device__ __forceinline__ Cut keep_all() { return Cut{-3.402823466e38f, kAllTies, false, 0}; }

// Threads' sums of two neighbouring bins, from bin 0 (the best) up, in c0 and c1: the bin at which
// `found(before, before + bin)` holds goes to s.pick_bin, what lies before it to s.pick.
template <int NT, typename Found>
__device__ __forceinline__ void find_bin(unsigned long long b, unsigned long long c0, unsigned long long c1,
                                         RowShared<NT>& s, Found found) {
    if (found(b, b + c0)) {
        s.pick_bin = 2 * threadIdx.x;
        s.pick = b;
    } else if (found(b + c0, b + c0 + c1)) {
        s.pick_bin = 2 * threadIdx.x + 1;
        s.pick = b + c0;
    }
    __syncthreads();
}

// digits of a key, best first, log2(2 NT) bits each
template <int NT>
struct Digits {
    static constexpr int kBits = NT == 1024 ? 11 : NT == 512 ? 10 : NT == 256 ? 9 : 7;
    static constexpr int kLevels = (32 + kBits - 1) / kBits;
    static_assert(1 << kBits == 2 * NT, "a bin for every digit");
    __device__ static int shift(int level) { return 32 - kBits * (level + 1) > 0 ? 32 - kBits * (level + 1) : 0; }
    __device__ static uint32_t mask(int level) {
        return (1u << (level == kLevels - 1 ? 32 - kBits * (kLevels - 1) : kBits)) - 1u;
    }
    // 16-bit logits have bits only in the first 19 of the float, and so of the key: the rest are the sign's
    template <typename T> static constexpr int levels() { return sizeof(T) == 2 ? (19 + kBits - 1) / kBits : kLevels; }
    __device__ static uint32_t filled(uint32_t prefix, int levels) {
        return (prefix & 0x80000000u) || levels == kLevels ? prefix : prefix | ((1u << shift(levels - 1)) - 1u);
    }
    __device__ static bool same(uint32_t a, uint32_t b, int level) {
        return level == 0 || (a >> shift(level - 1)) == (b >> shift(level - 1));
    }
};

// The bin that holds the k-th best: returns false where all allowed items are no more than k.
// each(f) calls f(x, id) for the thread's items (-inf: not allowed).
struct CountBin {
    int bin;
    uint32_t above, in;   // items in better bins, and in this
};
template <int NT, typename Each>
__device__ __forceinline__ bool count_bin(uint32_t k, const Bins& bins, RowShared<NT>& s, Each each, CountBin* r) {
    const int tid = threadIdx.x;
    s.count[2 * tid] = s.count[2 * tid + 1] = 0;
    if (tid == 0) s.members = 0;
    __syncthreads();
    each([&](float x, uint32_t) {
        if (x > -INFINITY) atomicAdd(&s.count[bins.of(x)], 1u);
    });
    __syncthreads();
    const uint32_t c0 = s.count[2 * tid], c1 = s.count[2 * tid + 1];
    uint32_t all;
    const uint32_t b = before32(c0 + c1, s, &all);
    if (all <= k) return false;
    find_bin(b, c0, c1, s, [&](unsigned long long x, unsigned long long e) { return x < k && e >= k; });
    r->bin = (int)s.pick_bin;
    r->above = (uint32_t)s.pick;
    r->in = s.count[r->bin];
    return true;
}

// The k-th best of the items that each() gives, digit by digit of the key.
template <typename T, int NT, typename Each>
__device__ __forceinline__ Cut digits_count(uint32_t left, RowShared<NT>& s, Each each) {
    const int tid = threadIdx.x;
    uint32_t prefix = 0, equal = 0;
    constexpr int kLevels = Digits<NT>::template levels<T>();
    for (int level = 0; level < kLevels; ++level) {
        __syncthreads();
        s.count[2 * tid] = s.count[2 * tid + 1] = 0;
        __syncthreads();
        const uint32_t mask = Digits<NT>::mask(level);
        each([&](float x, uint32_t) {
            const uint32_t key = ukey(x + 0.0f);   // (-0 equals 0)
            if (x > -INFINITY && Digits<NT>::same(key, prefix, level))
                atomicAdd(&s.count[mask - ((key >> Digits<NT>::shift(level)) & mask)], 1u);
        });
        __syncthreads();
        const uint32_t c0 = s.count[2 * tid], c1 = s.count[2 * tid + 1];
        uint32_t all;
        const uint32_t before = before32(c0 + c1, s, &all);
        find_bin(before, c0, c1, s, [&](unsigned long long x, unsigned long long e) { return x < left && e >= left; });
        prefix |= (mask - s.pick_bin) << Digits<NT>::shift(level);
        left -= (uint32_t)s.pick;
        equal = s.count[s.pick_bin];
    }
    return Cut{unukey(Digits<NT>::filled(prefix, kLevels)), left, equal > left, equal};
}

// The item of those that each() gives at which the weight, from `ahead` on, reaches p of `all`; `over` is
// what those equals of was.bound weigh that are beyond its ties and among these items.
template <typename T, int NT, typename W, typename Each>
__device__ __forceinline__ Cut digits_weight(double p, double all, unsigned long long ahead, Cut was,
                                             unsigned long long over, const W& wt, RowShared<NT>& s, Each each) {
    const int tid = threadIdx.x;
    uint32_t prefix = 0;
    const uint32_t bound_key = ukey(was.bound + 0.0f);
    constexpr int kLevels = Digits<NT>::template levels<T>();
    for (int level = 0; level < kLevels; ++level) {
        __syncthreads();
        s.weight[2 * tid] = s.weight[2 * tid + 1] = 0;
        __syncthreads();
        const uint32_t mask = Digits<NT>::mask(level);
        each([&](float x, uint32_t) {
            const uint32_t key = ukey(x + 0.0f);
            if (x >= was.bound && Digits<NT>::same(key, prefix, level))
                atomicAdd(&s.weight[mask - ((key >> Digits<NT>::shift(level)) & mask)], wt.fixed(x));
        });
        __syncthreads();
        if (tid == 0 && over && Digits<NT>::same(bound_key, prefix, level))
            s.weight[mask - ((bound_key >> Digits<NT>::shift(level)) & mask)] -= over;
        __syncthreads();
        const unsigned long long c0 = s.weight[2 * tid], c1 = s.weight[2 * tid + 1];
        unsigned long long level_sum;
        const unsigned long long before = ahead + before64(c0 + c1, s, &level_sum);
        find_bin(before, c0, c1, s,
                 [&](unsigned long long x, unsigned long long e) { return !reaches(x, p, all) && reaches(e, p, all); });
        prefix |= (mask - s.pick_bin) << Digits<NT>::shift(level);
        ahead = s.pick;
    }
    const float bound = unukey(Digits<NT>::filled(prefix, kLevels));
    uint32_t equal = 0;
    each([&](float x, uint32_t) { equal += x == bound; });
    before32(equal, s, &equal);
    // of the equals of this logit, as many as it takes
    const uint32_t most = bound == was.bound && was.partial ? was.ties : equal;
    const unsigned long long w = wt.fixed(bound);
    const double want = ceil((p * all - (double)ahead) / (double)w);
    uint32_t j = want < 1.0 ? 1u : want > (double)most ? most : (uint32_t)want;
    while (j > 1 && reaches(ahead + (unsigned long long)(j - 1) * w, p, all)) --j;
    while (j < most && !reaches(ahead + (unsigned long long)j * w, p, all)) ++j;
    return Cut{bound, j, equal > j, equal};
}

// Its bound.
template <typename T, int NT, typename Each>
__device__ __forceinline__ Cut cut_count(uint32_t k, const CountBin& in, const Bins& bins, RowShared<NT>& s,
                                         Each each) {
    const int tid = threadIdx.x;
    if (in.in <= NT) {
        each([&](float x, uint32_t id) {
            if (x > -INFINITY && bins.of(x) == in.bin) {
                const uint32_t at = atomicAdd(&s.members, 1u);
                s.member_x[at] = x;
                s.member_id[at] = id;
            }
        });
        __syncthreads();
        if (tid < (int)in.in) {
            const float x = s.member_x[tid];
            const uint32_t id = s.member_id[tid];
            uint32_t rank = in.above, same = 0, equal = 0;
#pragma unroll 4
            for (uint32_t j = 0; j < in.in; ++j) {
                const float o = s.member_x[j];
                rank += o > x;
                equal += o == x;
                same += o == x && s.member_id[j] < id;
            }
            if (rank + same == k - 1) {
                s.bound = x;
                s.ties = same + 1;
                s.equal = equal;
            }
        }
        __syncthreads();
        return Cut{s.bound, s.ties, s.equal > s.ties, s.equal};
    }
    return digits_count<T>(k, s, each);
}

// The shortest leading list with at least p of the weight, inside what `was` keeps.
template <typename T, int NT, typename W, typename Each>
__device__ __forceinline__ Cut cut_weight(double p, Cut was, const Bins& bins, const W& wt, RowShared<NT>& s,
                                          Each each) {
    const int tid = threadIdx.x;
    // equals of the bound beyond its ties: counted with the others, then taken off
    uint32_t extra = 0;
    if (was.partial) {
        each([&](float x, uint32_t) { extra += x == was.bound; });
        before32(extra, s, &extra);
        extra -= was.ties;
    }
    const unsigned long long over = (unsigned long long)extra * wt.fixed(was.bound);
    __syncthreads();
    s.weight[2 * tid] = s.weight[2 * tid + 1] = 0;
    if (tid == 0) s.members = 0;
    __syncthreads();
    each([&](float x, uint32_t) {
        if (x >= was.bound) atomicAdd(&s.weight[bins.of(x)], wt.fixed(x));
    });
    __syncthreads();
    if (was.partial) {
        if (tid == 0) s.weight[bins.of(was.bound)] -= over;
        __syncthreads();
    }
    unsigned long long c0 = s.weight[2 * tid], c1 = s.weight[2 * tid + 1], total;
    const unsigned long long b = before64(c0 + c1, s, &total);
    const double all = (double)total;
    auto found = [&](unsigned long long x, unsigned long long e) { return !reaches(x, p, all) && reaches(e, p, all); };
    find_bin(b, c0, c1, s, found);
    const int bin = (int)s.pick_bin;
    const unsigned long long above = s.pick;
    each([&](float x, uint32_t id) {
        if (x >= was.bound && bins.of(x) == bin) {
            const uint32_t at = atomicAdd(&s.members, 1u);
            if (at < NT) {
                s.member_x[at] = x;
                s.member_id[at] = id;
                s.member_w[at] = wt.fixed(x);
            }
        }
    });
    __syncthreads();
    const uint32_t in_bin = s.members;
    if (in_bin <= NT) {
        if (tid < (int)in_bin) {
            const float x = s.member_x[tid];
            const uint32_t id = s.member_id[tid];
            unsigned long long ahead = above;
            uint32_t same = 0, equal = 0;
#pragma unroll 4
            for (uint32_t j = 0; j < in_bin; ++j) {
                const float o = s.member_x[j];
                const bool before = o == x && s.member_id[j] < id;
                ahead += o > x || before ? s.member_w[j] : 0ull;
                equal += o == x;
                same += before;
            }
            if (!(x == was.bound && same >= was.ties) && found(ahead, ahead + s.member_w[tid])) {
                s.bound = x;
                s.ties = same + 1;
                s.equal = equal;
            }
        }
        __syncthreads();
        return Cut{s.bound, s.ties, s.equal > s.ties, s.equal};
    }
    return digits_weight<T>(p, all, 0ull, was, over, wt, s, each);
}

struct RowSettings {
    double t, p, min_p;
    uint32_t k;     // 0: all
    bool all_p;     // top-p keeps everything
};
__device__ __forceinline__ RowSettings row_settings(const DrawArgs& a, int64_t row) {
    RowSettings r;
    r.t = a.temperature ? (double)a.temperature[row] : a.temperature_v;
    r.p = a.top_p ? (double)a.top_p[row] : a.top_p_v;
    r.min_p = a.min_p ? (double)a.min_p[row] : a.min_p_v;
    r.min_p = r.min_p > 1.0 ? 1.0 : r.min_p;   // the best item always stays
    const int k = a.top_k ? a.top_k[row] : a.top_k_v;
    r.k = k > 0 ? (uint32_t)k : 0u;
    if (!(r.t > 0.0) || r.p <= 0.0) r.k = 1;
    if (!(r.t > 0.0)) r.t = 1.0;
    r.all_p = !(r.p > 0.0 && r.p < 1.0);
    return r;
}

// u total, held inside [0, total)
__device__ __forceinline__ unsigned long long draw_target(const DrawArgs& a, int64_t o, unsigned long long total) {
    const double at = (a.u ? a.u[o] : (double)a.u32[o]) * (double)total;
    const unsigned long long t = at > 0.0 ? (at >= 9.2e18 ? ~0ull >> 1 : (unsigned long long)at) : 0ull;
    return t >= total ? total - 1 : t;
}

// V neighbours' logits as they are stored (-inf past the row's end) and their mask bytes: loaded ahead, settled
// when they are used.  (Settled as they came, a row's vectors were loaded one behind the other: 2,048 rows of 27,278
// fp32 with a mask 138 us, so 101.)
template <typename T>
struct RawLogits {
    static constexpr int V = Elem<T>::kVec;
    typedef T own __attribute__((ext_vector_type(V)));
    own v;
    uint32_t on[V / 4];

    // from item i on
    __device__ __forceinline__ void load(const DrawArgs& a, int64_t row, int i) {
        const T* x = static_cast<const T*>(a.logits) + row * a.ld;
        const uint8_t* mask = a.mask ? a.mask + row * a.mask_ld : nullptr;
        if (i + V <= a.n) {
            v = *reinterpret_cast<const typename Elem<T>::vec*>(x + i);
            if (mask) __builtin_memcpy(on, mask + i, V);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = i + e < a.n ? x[i + e] : (T)(-INFINITY);
            if (mask) {
#pragma unroll
                for (int w = 0; w < V / 4; ++w) on[w] = 0;
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (i + e < a.n) on[e / 4] |= (uint32_t)mask[i + e] << (8 * (e & 3));
            }
        }
    }
    // -inf where not allowed
    __device__ __forceinline__ void settle(const DrawArgs& a, float* r) const {
#pragma unroll
        for (int e = 0; e < V; ++e) r[e] = fmaxf((float)v[e], -INFINITY);   // (a NaN becomes -inf)
        if (a.mask) {
#pragma unroll
            for (int e = 0; e < V; ++e) r[e] = (on[e / 4] >> (8 * (e & 3)) & 0xffu) ? r[e] : -INFINITY;
        }
    }
};
template <typename T>
__device__ __forceinline__ void load_logits(const DrawArgs& a, int64_t row, int i, float* r) {
    RawLogits<T> raw;
    raw.load(a, row, i);
    raw.settle(a, r);
}

// a copy the compiler takes for a new value: what one pass over the row derives from its logits (bins,
// weights) is computed again by the next and not kept in registers, for which there is no room
__device__ __forceinline__ float fresh(float x) {
    asm volatile("" : "+v"(x));
    return x;
}

template <typename T, int NT, int EPT>
__global__ __launch_bounds__(NT) void k_draw_row(DrawArgs a) {
    __shared__ RowShared<NT> s;
    constexpr int V = Elem<T>::kVec, J = EPT / V, W = NT / 64, P = RowShared<NT>::kPer;
    static_assert(J * W <= NT / 4, "a thread and a place for every segment");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t row = blockIdx.x;
    const RowSettings set = row_settings(a, row);
    // a wave's vectors, of 64 V neighbours each: the row spread evenly over the waves
    const int jn = (a.n + NT * V - 1) / (NT * V), segs = jn * W;
    const int first = wave * jn * 64 * V + lane * V;   // of the thread's vector 0; vector j: 64 V j further
    RawLogits<T> raw[J];
#pragma unroll
    for (int j = 0; j < J; ++j)
        if (j < jn) raw[j].load(a, row, first + 64 * V * j);
    __builtin_amdgcn_sched_barrier(0);
    float x[EPT];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        if (j < jn) {
            raw[j].settle(a, x + V * j);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) x[V * j + e] = -INFINITY;
        }
    }
    fill_powers<kRowPowers>(s.power, a.unit, NT);

    // the best item, and the mean of the first logits of every thread for the bins' range
    float top = -INFINITY, sum = 0.0f, num = 0.0f;
#pragma unroll
    for (int e = 0; e < EPT; ++e) top = fmaxf(top, x[e]);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const bool usual = fabsf(x[e]) < 1e30f;   // (no mask by the lowest value)
        sum += usual ? x[e] : 0.0f;
        num += usual ? 1.0f : 0.0f;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        top = fmaxf(top, __shfl_xor(top, d, 64));
        sum += __shfl_xor(sum, d, 64);
        num += __shfl_xor(num, d, 64);
    }
    if constexpr (NT > 64) {
        if (lane == 0) {
            s.wave_top[wave] = top;
            s.wave_sum[wave] = sum;
            s.wave_n[wave] = num;
        }
        __syncthreads();
        sum = num = 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            top = fmaxf(top, s.wave_top[j]);
            sum += s.wave_sum[j];
            num += s.wave_n[j];
        }
    }
    __syncthreads();
    if (!(top > -INFINITY)) {
        for (int d = tid; d < a.draws; d += NT) {
            a.items[row * a.draws + d] = -1;
            a.probs[row * a.draws + d] = 0.0f;
        }
        return;
    }
    const Weigher<kRowPowers> wt(top, set.t, a.unit, s.power);
    const unsigned long long least = wt.least(set.min_p);
    // twice the way from the best to the mean holds what top-k and top-p cut between
    const float range = 2.0f * (top - sum / num);
    const Bins bins = make_bins(top, range, 2 * NT);

    auto each = [&](auto f) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if (j < jn) {
#pragma unroll
                for (int e = 0; e < V; ++e) f(fresh(x[V * j + e]), (uint32_t)(first + 64 * V * j + e));
            }
            __builtin_amdgcn_sched_barrier(0);   // (a vector at a time: registers for one)
        }
    };
    constexpr int kList = RowShared<NT>::kList;
    constexpr float kLowest = -3.402823466e38f;
    const bool top_k = set.k > 0 && set.k < (uint32_t)a.n;
    // items not below a limit: in the workgroup, and (at) in the waves ahead of this one
    uint32_t at = 0;
    auto count_from = [&](float limit) {
        int mine = 0;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if (j < jn) {
#pragma unroll
                for (int e = 0; e < V; ++e) mine += lane_count(__ballot(x[V * j + e] >= limit));
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (NT == 64) return (uint32_t)mine;
        __syncthreads();
        if (lane == 0) s.wave32[wave] = (uint32_t)mine;
        __syncthreads();
        uint32_t all = 0;
        at = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const uint32_t o = s.wave32[w];
            at += w < wave ? o : 0u;
            all += o;
        }
        return all;
    };
    float limit = kLowest;
    uint32_t count = kList + 1;   // of the list
    if (a.n <= kList) {
        count = count_from(limit);
    } else if (top_k && set.k <= (uint32_t)kList) {
        auto sample = [&](auto f) {
#pragma unroll
            for (int j = 0; j < J; ++j)
                if (j < jn) f(fresh(x[V * j + j % V]), 0u);
        };
        // k / V of the sample, and four deviations more
        const float part = (float)set.k / V;
        CountBin cb;
        if (count_bin((uint32_t)(part + 4.0f * sqrtf(part) + 4.0f), bins, s, sample, &cb)) limit = bins.below(cb.bin);
        count = count_from(limit);
        if (count < set.k && limit > kLowest) count = kList + 1;
    }
    Cut cut = keep_all();
    if (top_k && count > (uint32_t)kList) {
        CountBin cb;
        if (count_bin(set.k, bins, s, each, &cb)) {
            limit = bins.below(cb.bin);
            if (cb.above + cb.in <= (uint32_t)kList) count = count_from(limit);
            if (count > (uint32_t)kList) cut = cut_count<T>(set.k, cb, bins, s, each);
        }
    }
    if (count <= (uint32_t)kList) {
        // ---- from a list in LDS
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if (j < jn) {
                uint64_t m[V], any = 0;
#pragma unroll
                for (int e = 0; e < V; ++e) any |= m[e] = __ballot(x[V * j + e] >= limit);
                if (any != 0) {
                    uint32_t mine = at;
                    int id = first + 64 * V * j;
                    asm volatile("" : "+v"(id));   // (computed here, not kept from the passes before)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        mine = lanes_before(m[e], mine);
                        at += (uint32_t)lane_count(m[e]);
                    }
#pragma unroll
                    for (int e = 0; e < V; ++e) {   // (without a branch)
                        const bool in = x[V * j + e] >= limit;
                        const uint32_t to = in ? mine : (uint32_t)(kList + lane);
                        s.list_x[to] = x[V * j + e];
                        s.list_id[to] = (uint32_t)(id + e);
                        mine += in;
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
        float y[P];   // the thread's neighbours in the list
#pragma unroll
        for (int e = 0; e < P; ++e) y[e] = P * tid + e < (int)count ? s.list_x[P * tid + e] : -INFINITY;
        auto each_listed = [&](auto f) {
#pragma unroll
            for (int e = 0; e < P; ++e) f(y[e], (uint32_t)(P * tid + e));
        };
        const Bins fine = make_bins(top, limit > kLowest ? top - limit : range, 2 * NT);
        Cut in = keep_all();
        CountBin cb;
        if (top_k && count > set.k && count_bin(set.k, fine, s, each_listed, &cb))
            in = cut_count<T>(set.k, cb, fine, s, each_listed);
        if (!set.all_p) in = cut_weight<T>(set.p, in, fine, wt, s, each_listed);
        __syncthreads();
        // weights in the order of the ids, which is the list's
        uint32_t seen = 0;
        if (in.partial) {
            uint32_t mine = 0, ties;
#pragma unroll
            for (int e = 0; e < P; ++e) mine += y[e] == in.bound;
            seen = before32(mine, s, &ties);
        }
        unsigned long long w[P], mine = 0, total;
#pragma unroll
        for (int e = 0; e < P; ++e) {
            const bool out = y[e] < in.bound || (in.partial && y[e] == in.bound && seen++ >= in.ties);
            w[e] = out ? 0ull : wt.fixed(y[e], least);
            mine += w[e];
        }
        unsigned long long c = before64(mine, s, &total);
        __syncthreads();
#pragma unroll
        for (int e = 0; e < P; ++e) s.before[P * tid + e] = c += w[e];   // running sums
        __syncthreads();
        for (int d = tid; d < a.draws; d += NT) {
            const int64_t o = row * a.draws + d;
            const unsigned long long target = draw_target(a, o, total);
            int lo = 0, hi = (int)count - 1;   // the first running sum above the target
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (s.before[mid] > target) hi = mid;
                else lo = mid + 1;
            }
            const unsigned long long got = s.before[lo] - (lo ? s.before[lo - 1] : 0ull);
            a.items[o] = (int32_t)s.list_id[lo];
            a.probs[o] = (float)((double)got / (double)total);
        }
        return;
    }

    // ---- from the registers
    if (!set.all_p) cut = cut_weight<T>(set.p, cut, bins, wt, s, each);
    // equals of the bound ahead of the lane's first of V neighbours
    auto ties_before = [&](const float* y, uint32_t ahead) {
#pragma unroll
        for (int e = 0; e < V; ++e) ahead = lanes_before(__ballot(y[e] == cut.bound), ahead);
        return ahead;
    };
    if (cut.partial) {   // s.seg_ties: equals of the bound ahead of each segment
        __syncthreads();
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if (j < jn) {
                int mine = 0;
#pragma unroll
                for (int e = 0; e < V; ++e) mine += lane_count(__ballot(fresh(x[V * j + e]) == cut.bound));
                if (lane == 0) s.seg_ties[wave * jn + j] = (uint32_t)mine;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
        uint32_t all;
        const uint32_t b = before32(tid < segs ? s.seg_ties[tid] : 0u, s, &all);
        __syncthreads();
        if (tid < segs) s.seg_ties[tid] = b;
    }
    __syncthreads();
    auto weigh = [&](float y, uint32_t& seen) -> unsigned long long {
        if (y < cut.bound) return 0;   // (-inf too)
        if (cut.partial && y == cut.bound && seen++ >= cut.ties) return 0;
        return wt.fixed(y, least);
    };
#pragma unroll
    for (int j = 0; j < J; ++j) {
        if (j < jn) {
            uint32_t seen = cut.partial ? ties_before(x + V * j, s.seg_ties[wave * jn + j]) : 0u;
            unsigned long long mine = 0;
#pragma unroll
            for (int e = 0; e < V; ++e) mine += weigh(fresh(x[V * j + e]), seen);
            mine = lane_sums64(mine);
            if (lane == 63) s.seg[wave * jn + j] = mine;
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    unsigned long long total;
    const unsigned long long seg_b = before64(tid < segs ? s.seg[tid] : 0ull, s, &total);
    __syncthreads();
    if (tid < segs) s.seg[tid] = seg_b;
    __syncthreads();
    // a wave takes a draw: the segment in which its sum passes the target, read once more
    for (int d = wave; d < a.draws; d += W) {
        const int64_t o = row * a.draws + d;
        const unsigned long long target = draw_target(a, o, total);
        int lo = 0, hi = segs - 1;   // the last segment with no more than the target ahead of it
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (s.seg[mid] <= target) lo = mid;
            else hi = mid - 1;
        }
        const int at = (lo * 64 + lane) * V;
        float y[V];
        load_logits<T>(a, row, at, y);
        uint32_t seen = cut.partial ? ties_before(y, s.seg_ties[lo]) : 0u;
        unsigned long long w[V], mine = 0;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            w[e] = weigh(y[e], seen);
            mine += w[e];
        }
        unsigned long long c = s.seg[lo] + lane_sums64(mine) - mine;
        if (c <= target && target < c + mine) {
            bool open = true;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (open && target < c + w[e]) {
                    open = false;
                    a.items[o] = at + e;
                    a.probs[o] = (float)((double)w[e] / (double)total);
                }
                c += w[e];
            }
        }
    }
}

// ----------------------------------------------------------------------------- long rows
//
// A row longer than the registers of a workgroup is cut into parts, a workgroup each, and passed over by
// a few launches that hand on what they find in a workspace: the best item; per cut (top-k by counts,
// top-p by weights) the histogram over kLongBins steps of the logit, the items of the bin that holds the
// cut, and the bound among them (one workgroup a row; where the items outgrow their list it reads the row
// again instead); the weight of every segment of 64 vectors; the draws.  The row comes from memory once
// and from the caches after that (1,000,000 items are 2 or 4 MB).  16 rows of 1,000,000 bf16, top-p: 87 us, of them
// histogram 23, segments' weights 22 (64-bit exponentials both), gather 14, bound 11, draws 9, best 8.  Workgroups of
// 1,024: of 256 the same, but four times as many histograms to join.

constexpr int kLongThreads = 1024;
constexpr int kLongWaves = kLongThreads / 64;
constexpr int kLongBins = 2048;
constexpr int kResolveThreads = 512;

struct LongRow {
    float bound;
    uint32_t ties, partial, equal;            // the cut so far
    uint32_t members;                         // items of the bin, as far as they are gathered
    int bin;                                  // -1: no cut to make
    uint32_t above_n;
    unsigned long long above_w, total_w;
};

struct LongArgs {
    DrawArgs a;
    int parts, part;          // parts of a row, items of a part (whole segments)
    int segs;                 // segments of a row
    uint32_t cap;             // of a row's list
    float* tops;              // [rows][parts] best, sum and number of usual logits
    float* sums;
    float* nums;
    uint32_t* count;          // [rows][kLongBins]
    unsigned long long* weight;
    LongRow* row;
    uint2* list;              // [rows][cap] logit bits, id
    unsigned long long* seg;  // [rows][segs]
    uint32_t* seg_ties;
};

template <typename T>
__host__ __device__ constexpr int seg_items() { return 64 * Elem<T>::kVec; }

// the segments of this wave in a part
template <typename T>
__device__ __forceinline__ void wave_segments(const LongArgs& l, int part, int* s0, int* s1) {
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), waves = (int)(blockDim.x >> 6);
    const int n = l.part / seg_items<T>(), per = (n + waves - 1) / waves, end = min(l.segs, (part + 1) * n);
    *s0 = min(part * n + wave * per, end);
    *s1 = min(*s0 + per, end);
}

// the part's logits, a vector at a time: f(logits, first id); a wave takes a contiguous part of it
template <typename T, typename F>
__device__ __forceinline__ void each_vector(const LongArgs& l, int64_t r, int part, F f) {
    constexpr int V = Elem<T>::kVec, U = 4;
    const int lane = threadIdx.x & 63;
    int s0, s1;
    wave_segments<T>(l, part, &s0, &s1);
    for (int sg = s0; sg < s1; sg += U) {
        RawLogits<T> raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (sg + u < s1) raw[u].load(l.a, r, (sg + u) * seg_items<T>() + lane * V);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (sg + u >= s1) break;
            float y[V];
            raw[u].settle(l.a, y);
            f(y, (sg + u) * seg_items<T>() + lane * V);
        }
    }
}

struct LongShared {
    union {
        uint32_t count[kLongBins];
        unsigned long long weight[kLongBins];
        uint2 staged[kLongBins];
    };
    double power[1 << kLongPowers];
    unsigned long long wave64[kLongWaves], pick;
    uint32_t wave32[kLongWaves];
    float wavef[3][kLongWaves];
    int pick_bin;
    uint32_t items;
};

template <typename T>
__global__ __launch_bounds__(kLongThreads) void k_long_top(LongArgs l) {
    __shared__ LongShared s;
    const int64_t r = blockIdx.x / l.parts;
    const int part = (int)(blockIdx.x - r * l.parts), tid = threadIdx.x;
    for (int b = part * kLongThreads + tid; b < kLongBins; b += l.parts * kLongThreads) {
        l.count[r * kLongBins + b] = 0;
        l.weight[r * kLongBins + b] = 0;
    }
    float top = -INFINITY, sum = 0.0f, num = 0.0f;
    each_vector<T>(l, r, part, [&](const float* y, int) {
#pragma unroll
        for (int e = 0; e < Elem<T>::kVec; ++e) {
            top = fmaxf(top, y[e]);
            const bool usual = fabsf(y[e]) < 1e30f;
            sum += usual ? y[e] : 0.0f;
            num += usual ? 1.0f : 0.0f;
        }
    });
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        top = fmaxf(top, __shfl_xor(top, d, 64));
        sum += __shfl_xor(sum, d, 64);
        num += __shfl_xor(num, d, 64);
    }
    if ((tid & 63) == 0) {
        s.wavef[0][tid >> 6] = top;
        s.wavef[1][tid >> 6] = sum;
        s.wavef[2][tid >> 6] = num;
    }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kLongWaves; ++w) {
            top = fmaxf(top, s.wavef[0][w]);
            sum += s.wavef[1][w];
            num += s.wavef[2][w];
        }
        l.tops[blockIdx.x] = top;
        l.sums[blockIdx.x] = sum;
        l.nums[blockIdx.x] = num;
        if (part == 0) {
            LongRow z{};
            const Cut all = keep_all();
            z.bound = all.bound;
            z.ties = all.ties;
            z.bin = -1;
            l.row[r] = z;
        }
    }
}

// the row's best logit and its bins, from the parts' (every workgroup in the same order)
__device__ __forceinline__ Bins long_bins(const LongArgs& l, int64_t r) {
    const int lane = threadIdx.x & 63;
    float top = -INFINITY, sum = 0.0f, num = 0.0f;
    for (int p = lane; p < l.parts; p += 64) {
        top = fmaxf(top, l.tops[r * l.parts + p]);
        sum += l.sums[r * l.parts + p];
        num += l.nums[r * l.parts + p];
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        top = fmaxf(top, __shfl_xor(top, d, 64));
        sum += __shfl_xor(sum, d, 64);
        num += __shfl_xor(num, d, 64);
    }
    return make_bins(top, 2.0f * (top - sum / num), kLongBins);
}
__device__ __forceinline__ Weigher<kLongPowers> long_weigher(const LongArgs& l, const Bins& bins, const RowSettings& set,
                                                const double* power) {
    return Weigher<kLongPowers>(bins.top, set.t, l.a.unit, power);
}
__device__ __forceinline__ Cut row_cut(const LongRow& w) { return Cut{w.bound, w.ties, w.partial != 0, w.equal}; }
__device__ __forceinline__ bool wants_cut(const LongArgs& l, const RowSettings& set, bool weights) {
    return weights ? !set.all_p : set.k > 0 && set.k < (uint32_t)l.a.n;
}

template <typename T, bool WEIGHTS>
__global__ __launch_bounds__(kLongThreads) void k_long_histogram(LongArgs l) {
    __shared__ LongShared s;
    const int64_t r = blockIdx.x / l.parts;
    const int part = (int)(blockIdx.x - r * l.parts), tid = threadIdx.x;
    const RowSettings set = row_settings(l.a, r);
    if (!wants_cut(l, set, WEIGHTS)) return;
    const Bins bins = long_bins(l, r);
    if (!(bins.top > -INFINITY)) return;
    for (int b = tid; b < kLongBins; b += kLongThreads) {
        if constexpr (WEIGHTS) s.weight[b] = 0;
        else s.count[b] = 0;
    }
    fill_powers<kLongPowers>(s.power, l.a.unit, kLongThreads);
    __syncthreads();
    const Weigher<kLongPowers> wt = long_weigher(l, bins, set, s.power);
    const float bound = l.row[r].bound;
    each_vector<T>(l, r, part, [&](const float* y, int) {
        constexpr int V = Elem<T>::kVec;
        unsigned long long w[V];
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = WEIGHTS ? wt.fixed(y[e]) : 1ull;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (!(y[e] >= bound)) continue;   // (-inf too)
            if constexpr (WEIGHTS) atomicAdd(&s.weight[bins.of(y[e])], w[e]);
            else atomicAdd(&s.count[bins.of(y[e])], 1u);
        }
    });
    __syncthreads();
    for (int b = tid; b < kLongBins; b += kLongThreads) {
        if constexpr (WEIGHTS) {
            if (s.weight[b]) atomicAdd(&l.weight[r * kLongBins + b], s.weight[b]);
        } else {
            if (s.count[b]) atomicAdd(&l.count[r * kLongBins + b], s.count[b]);
        }
    }
}

// exclusive sums over the workgroup
__device__ __forceinline__ unsigned long long long_before(unsigned long long v, LongShared& s,
                                                          unsigned long long* sum) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const unsigned long long inc = lane_sums64(v);
    __syncthreads();
    if (lane == 63) s.wave64[w] = inc;
    __syncthreads();
    unsigned long long before = 0, all = 0;
#pragma unroll
    for (int j = 0; j < kLongWaves; ++j) {
        before += j < w ? s.wave64[j] : 0ull;
        all += s.wave64[j];
    }
    *sum = all;
    return before + inc - v;
}

// The bin of the cut (every workgroup of a row finds the same), and its items to the row's list.
template <typename T, bool WEIGHTS>
__global__ __launch_bounds__(kLongThreads) void k_long_gather(LongArgs l) {
    __shared__ LongShared s;
    constexpr int kPer = kLongBins / kLongThreads;
    const int64_t r = blockIdx.x / l.parts;
    const int part = (int)(blockIdx.x - r * l.parts), tid = threadIdx.x;
    const RowSettings set = row_settings(l.a, r);
    if (!wants_cut(l, set, WEIGHTS)) return;
    const Bins bins = long_bins(l, r);
    if (!(bins.top > -INFINITY)) return;
    const Cut was = row_cut(l.row[r]);
    if (WEIGHTS && was.partial) fill_powers<kLongPowers>(s.power, l.a.unit, kLongThreads);
    if (tid == 0) {
        s.pick_bin = -1;
        s.items = 0;
    }
    __syncthreads();
    unsigned long long c[kPer], mine = 0, total;
#pragma unroll
    for (int b = 0; b < kPer; ++b) {
        const int64_t at = r * kLongBins + kPer * tid + b;
        c[b] = WEIGHTS ? l.weight[at] : (unsigned long long)l.count[at];
    }
    if (WEIGHTS && was.partial) {   // equals of top-k's bound beyond its ties
        const Weigher<kLongPowers> wt = long_weigher(l, bins, set, s.power);
        const int at = bins.of(was.bound);
#pragma unroll
        for (int b = 0; b < kPer; ++b)
            if (kPer * tid + b == at) c[b] -= (unsigned long long)(was.equal - was.ties) * wt.fixed(was.bound);
    }
#pragma unroll
    for (int b = 0; b < kPer; ++b) mine += c[b];
    unsigned long long ahead = long_before(mine, s, &total);
    const double all = (double)total;
    if (WEIGHTS || total > set.k) {
#pragma unroll
        for (int b = 0; b < kPer; ++b) {
            const unsigned long long e = ahead + c[b];
            const bool found = WEIGHTS ? !reaches(ahead, set.p, all) && reaches(e, set.p, all)
                                       : ahead < set.k && e >= set.k;
            if (found) {
                s.pick_bin = kPer * tid + b;
                s.pick = ahead;
            }
            ahead = e;
        }
    }
    __syncthreads();
    const int bin = s.pick_bin;
    if (part == 0 && tid == 0) {
        l.row[r].bin = bin;
        l.row[r].above_n = (uint32_t)s.pick;
        l.row[r].above_w = s.pick;
        l.row[r].total_w = total;
    }
    if (bin < 0) return;
    // to LDS first: one place in the row's list for all of them (with an atomic on it for each wave's items this
    // kernel took 57 us, counted in a pass of its own 20; 16 rows of 1,000,000)
    each_vector<T>(l, r, part, [&](const float* y, int id) {
#pragma unroll
        for (int e = 0; e < Elem<T>::kVec; ++e)
            if (y[e] >= was.bound && bins.of(y[e]) == bin) {
                const uint32_t at = atomicAdd(&s.items, 1u);
                if (at < kLongBins) s.staged[at] = make_uint2(__float_as_uint(y[e]), (uint32_t)(id + e));
            }
    });
    __syncthreads();
    const uint32_t items = s.items;
    if (items == 0) return;
    if (tid == 0) s.wave32[0] = atomicAdd(&l.row[r].members, items);
    __syncthreads();
    const uint32_t first = s.wave32[0];
    if (first >= l.cap) return;   // (the list is not used then)
    if (items <= (uint32_t)kLongBins) {
        for (uint32_t at = tid; at < items; at += kLongThreads)
            if (first + at < l.cap) l.list[r * l.cap + first + at] = s.staged[at];
        return;
    }
    if (tid == 0) s.items = 0;
    __syncthreads();
    each_vector<T>(l, r, part, [&](const float* y, int id) {
#pragma unroll
        for (int e = 0; e < Elem<T>::kVec; ++e)
            if (y[e] >= was.bound && bins.of(y[e]) == bin) {
                const uint32_t at = first + atomicAdd(&s.items, 1u);
                if (at < l.cap) l.list[r * l.cap + at] = make_uint2(__float_as_uint(y[e]), (uint32_t)(id + e));
            }
    });
}

// The bound among the items of the bin; a workgroup a row.
template <typename T, bool WEIGHTS>
__global__ __launch_bounds__(kResolveThreads) void k_long_resolve(LongArgs l) {
    __shared__ RowShared<kResolveThreads> s;
    __shared__ double power[1 << kLongPowers];
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x;
    const RowSettings set = row_settings(l.a, r);
    if (!wants_cut(l, set, WEIGHTS)) return;
    const LongRow w = l.row[r];
    const Bins bins = long_bins(l, r);
    if (!(bins.top > -INFINITY) || w.bin < 0) return;
    fill_powers<kLongPowers>(power, l.a.unit, kResolveThreads);
    __syncthreads();
    const Cut was = row_cut(w);
    const Weigher<kLongPowers> wt = long_weigher(l, bins, set, power);
    const unsigned long long over =
        WEIGHTS && was.partial && bins.of(was.bound) == w.bin
            ? (unsigned long long)(was.equal - was.ties) * wt.fixed(was.bound) : 0ull;
    auto bound_of = [&](auto each) {
        if constexpr (WEIGHTS)
            return digits_weight<T>(set.p, (double)w.total_w, w.above_w, was, over, wt, s, each);
        else
            return digits_count<T>(set.k - w.above_n, s, each);
    };
    Cut cut;
    if (w.members <= l.cap) {
        cut = bound_of([&](auto f) {
            for (uint32_t i = tid; i < w.members; i += kResolveThreads) {
                const uint2 m = l.list[r * l.cap + i];
                f(__uint_as_float(m.x), m.y);
            }
        });
    } else {
        LongArgs whole = l;   // (the row as one part)
        whole.part = l.segs * seg_items<T>();
        cut = bound_of([&](auto f) {
            each_vector<T>(whole, r, 0, [&](const float* y, int id) {
#pragma unroll
                for (int e = 0; e < Elem<T>::kVec; ++e)
                    if (y[e] >= was.bound && bins.of(y[e]) == w.bin) f(y[e], (uint32_t)(id + e));
            });
        });
    }
    __syncthreads();
    if (tid == 0) {
        LongRow n = w;
        n.bound = cut.bound;
        n.ties = cut.ties;
        n.partial = cut.partial;
        n.equal = cut.equal;
        n.members = 0;
        n.bin = -1;
        l.row[r] = n;
    }
}

// weights of V neighbours, of which `seen` equals of the bound lie ahead
template <int V>
__device__ __forceinline__ unsigned long long weigh_vector(const float* y, uint32_t seen, const Cut& cut,
                                                           const Weigher<kLongPowers>& wt, unsigned long long least,
                                                           unsigned long long* w) {
    unsigned long long sum = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        w[e] = 0;
        if (y[e] >= cut.bound && !(cut.partial && y[e] == cut.bound && seen++ >= cut.ties)) w[e] = wt.fixed(y[e], least);
        sum += w[e];
    }
    return sum;
}

// The weight of every segment; under a partial bound that of what lies above it, and the number of its equals.
template <typename T>
__global__ __launch_bounds__(kLongThreads) void k_long_weigh(LongArgs l) {
    __shared__ double power[1 << kLongPowers];
    constexpr int V = Elem<T>::kVec;
    const int64_t r = blockIdx.x / l.parts;
    const int part = (int)(blockIdx.x - r * l.parts), lane = threadIdx.x & 63;
    const RowSettings set = row_settings(l.a, r);
    const Bins bins = long_bins(l, r);
    if (!(bins.top > -INFINITY)) return;
    fill_powers<kLongPowers>(power, l.a.unit, kLongThreads);
    __syncthreads();
    const Weigher<kLongPowers> wt = long_weigher(l, bins, set, power);
    const unsigned long long least = wt.least(set.min_p);
    const Cut cut = row_cut(l.row[r]);
    each_vector<T>(l, r, part, [&](const float* y, int id) {
        const int64_t g = r * l.segs + id / seg_items<T>();
        unsigned long long sum = 0;
#pragma unroll
        for (int e = 0; e < V; ++e) {   // (of all, without a branch: the chains of a vector side by side)
            const unsigned long long w = wt.fixed(y[e], least);
            sum += y[e] > cut.bound || (!cut.partial && y[e] == cut.bound) ? w : 0ull;
        }
        sum = lane_sums64(sum);
        if (lane == 63) l.seg[g] = sum;
        if (cut.partial) {
            int n = 0;
#pragma unroll
            for (int e = 0; e < V; ++e) n += lane_count(__ballot(y[e] == cut.bound));
            if (lane == 0) l.seg_ties[g] = (uint32_t)n;
        }
    });
}

// A draw of a row: the segment in which the running sum passes the target, then the item in it; the draws from `first` on.
template <typename T>
__global__ __launch_bounds__(kLongThreads) void k_long_draw(LongArgs l, int64_t first) {
    __shared__ LongShared s;
    constexpr int V = Elem<T>::kVec;
    const int64_t o = first + blockIdx.x, r = o / l.a.draws;
    const int tid = threadIdx.x, lane = tid & 63;
    const RowSettings set = row_settings(l.a, r);
    const Bins bins = long_bins(l, r);
    if (!(bins.top > -INFINITY)) {
        if (tid == 0) {
            l.a.items[o] = -1;
            l.a.probs[o] = 0.0f;
        }
        return;
    }
    fill_powers<kLongPowers>(s.power, l.a.unit, kLongThreads);
    const Weigher<kLongPowers> wt = long_weigher(l, bins, set, s.power);
    const Cut cut = row_cut(l.row[r]);
    const unsigned long long least = wt.least(set.min_p);
    // a thread's share of the segments
    const int per = (l.segs + kLongThreads - 1) / kLongThreads;
    const int g0 = min(tid * per, l.segs), g1 = min(g0 + per, l.segs);
    const unsigned long long* seg = l.seg + r * l.segs;
    const uint32_t* equals = l.seg_ties + r * l.segs;
    uint32_t ties = 0;          // equals of a partial bound ahead of the share
    unsigned long long tie_w = 0;
    if (cut.partial) {
        for (int g = g0; g < g1; ++g) ties += equals[g];
        unsigned long long all;
        ties = (uint32_t)long_before(ties, s, &all);   // (and the powers)
        tie_w = wt.fixed(cut.bound, least);
    }
    // a segment's weight, `ahead` equals of the bound before it
    auto weight = [&](int g, uint32_t ahead) {
        unsigned long long w = seg[g];
        if (cut.partial && ahead < cut.ties) w += tie_w * min(equals[g], cut.ties - ahead);
        return w;
    };
    unsigned long long mine = 0, total;
    {
        uint32_t ahead = ties;
        for (int g = g0; g < g1; ++g) {
            mine += weight(g, ahead);
            if (cut.partial) ahead += equals[g];
        }
    }
    unsigned long long c = long_before(mine, s, &total);
    const unsigned long long target = draw_target(l.a, o, total);
    if (c <= target && target < c + mine) {
        for (int g = g0; g < g1; ++g) {
            const unsigned long long w = weight(g, ties);
            if (target < c + w) {
                s.pick_bin = g;
                s.pick = c;
                s.items = ties;
                break;
            }
            c += w;
            if (cut.partial) ties += equals[g];
        }
    }
    __syncthreads();
    if (tid >= 64) return;
    const int g = s.pick_bin, at = g * seg_items<T>() + lane * V;
    float y[V];
    load_logits<T>(l.a, r, at, y);
    uint32_t seen = 0;
    if (cut.partial) {
        seen = s.items;
#pragma unroll
        for (int e = 0; e < V; ++e) seen = lanes_before(__ballot(y[e] == cut.bound), seen);
    }
    unsigned long long w[V];
    const unsigned long long sum = weigh_vector<V>(y, seen, cut, wt, least, w);
    c = s.pick + lane_sums64(sum) - sum;
    if (c <= target && target < c + sum) {
        bool open = true;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (open && target < c + w[e]) {
                open = false;
                l.a.items[o] = at + e;
                l.a.probs[o] = (float)((double)w[e] / (double)total);
            }
            c += w[e];
        }
    }
}

// workspace of the long path (sizes by the narrower vector, so it serves every element type)
struct LongLayout {
    int64_t parts, segs, cap;
    size_t tops, count, weight, row, list, seg, seg_ties, total;
};
static LongLayout long_layout(int64_t rows, int64_t n, int vec) {
    LongLayout l{};
    const int64_t seg = 64 * vec;
    l.segs = (n + seg - 1) / seg;
    // about 4,096 waves, four a SIMD, of at least four segments each
    l.parts = 4096 / kLongWaves / rows;
    const int64_t most = (l.segs + 4 * kLongWaves - 1) / (4 * kLongWaves);
    l.parts = l.parts < 1 ? 1 : l.parts > most ? most : l.parts;
    // lists of 64 MB together: 2,048 items at least, 65,536 at most
    l.cap = ((int64_t)8 << 20) / rows;
    l.cap = l.cap < 2048 ? 2048 : l.cap > 65536 ? 65536 : l.cap;
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t at = off;
        off = (off + bytes + 255) / 256 * 256;
        return at;
    };
    l.tops = take((size_t)rows * l.parts * 3 * sizeof(float));
    l.count = take((size_t)rows * kLongBins * sizeof(uint32_t));
    l.weight = take((size_t)rows * kLongBins * sizeof(unsigned long long));
    l.row = take((size_t)rows * sizeof(LongRow));
    l.list = take((size_t)rows * l.cap * sizeof(uint2));
    l.seg = take((size_t)rows * l.segs * sizeof(unsigned long long));
    l.seg_ties = take((size_t)rows * l.segs * sizeof(uint32_t));
    l.total = off;
    return l;
}

constexpr int kRowMost = 512 * 56;   // the longest row that two workgroups a CU hold; behind it one of 1,024 does,
// up to so many logits a thread (nothing spilled)
constexpr int items_most(size_t size) { return size == 4 ? 40 : 32; }

// Workgroups of one launch at most: HIP counts a launch's threads in 32 bits, and 2^21 workgroups have up to 2^31.
// More rows (draws over long rows) go in several launches, one behind the other, that share the workspace.
constexpr int64_t kLaunchMost = (int64_t)1 << 21;

size_t draw_workspace(int64_t rows, int64_t n, size_t size) {
    return rows > 0 && n > 1024 * items_most(size) ? long_layout(std::min(rows, kLaunchMost), n, Elem<float>::kVec).total : 0;
}
int64_t draw_count(const ncf_draw_t& d) {
    return d.rows > INT64_MAX / (d.draws > 0 ? d.draws : 1) ? INT64_MAX : d.rows * d.draws;
}

template <typename T>
static void draw_long(const DrawArgs& a, void* ws, bool may_k, bool may_p, hipStream_t st) {
    const LongLayout y = long_layout(a.rows, a.n, Elem<T>::kVec);
    LongArgs l{};
    l.a = a;
    l.parts = (int)y.parts;
    l.segs = (int)y.segs;
    l.part = (int)((y.segs + y.parts - 1) / y.parts) * seg_items<T>();
    l.cap = (uint32_t)y.cap;
    l.tops = at<float>(ws, y.tops);
    l.sums = l.tops + a.rows * y.parts;
    l.nums = l.sums + a.rows * y.parts;
    l.count = at<uint32_t>(ws, y.count);
    l.weight = at<unsigned long long>(ws, y.weight);
    l.row = at<LongRow>(ws, y.row);
    l.list = at<uint2>(ws, y.list);
    l.seg = at<unsigned long long>(ws, y.seg);
    l.seg_ties = at<uint32_t>(ws, y.seg_ties);
    const dim3 grid((unsigned)(a.rows * y.parts)), rows((unsigned)a.rows);
    launch(k_long_top<T>, grid, kLongThreads, 0, st, l);
    if (may_k) {
        launch(k_long_histogram<T, false>, grid, kLongThreads, 0, st, l);
        launch(k_long_gather<T, false>, grid, kLongThreads, 0, st, l);
        launch(k_long_resolve<T, false>, rows, kResolveThreads, 0, st, l);
    }
    if (may_p) {
        launch(k_long_histogram<T, true>, grid, kLongThreads, 0, st, l);
        launch(k_long_gather<T, true>, grid, kLongThreads, 0, st, l);
        launch(k_long_resolve<T, true>, rows, kResolveThreads, 0, st, l);
    }
    launch(k_long_weigh<T>, grid, kLongThreads, 0, st, l);
    const int64_t draws = a.rows * a.draws;
    for (int64_t o = 0; o < draws; o += kLaunchMost)
        launch(k_long_draw<T>, dim3((unsigned)std::min(draws - o, kLaunchMost)), kLongThreads, 0, st, l, o);
}

// The smallest workgroup that holds a row, and the next one (us for 4,096 rows, top-50, top-p 0.9): 500 items 15.2
// and 15.6, 2,000 20.6 and 41.5, 8,000 58 and 115.  A row in registers, and by the launches over parts of it: one row
// of 27,278 17.3 and 59.5, 2,048 88 and 408; one of 40,000 18.9 and 57.5, 1,024 84 and 269 (fp32).
template <typename T>
static void draw_t(const DrawArgs& a, void* ws, bool may_k, bool may_p, hipStream_t st) {
    constexpr int kMost = items_most(sizeof(T));
    const dim3 grid((unsigned)a.rows);
    if (a.n <= 64 * 8) launch(k_draw_row<T, 64, 8>, grid, 64, 0, st, a);
    else if (a.n <= 64 * 32) launch(k_draw_row<T, 64, 32>, grid, 64, 0, st, a);
    else if (a.n <= 256 * 32) launch(k_draw_row<T, 256, 32>, grid, 256, 0, st, a);
    else if (a.n <= kRowMost) launch(k_draw_row<T, 512, 56>, grid, 512, 0, st, a);
    else if (a.n <= 1024 * kMost) launch(k_draw_row<T, 1024, kMost>, grid, 1024, 0, st, a);
    else draw_long<T>(a, ws, may_k, may_p, st);
}

hipError_t launch_draw(const ncf_draw_t& c, hipStream_t st) {
    if (c.rows <= 0 || c.draws <= 0) return hipSuccess;
    DrawArgs a{};
    a.logits = c.logits;
    a.mask = c.mask;
    a.ld = c.ld;
    a.mask_ld = c.mask_ld;
    a.rows = c.rows;
    a.n = (int)c.n;
    a.draws = (int)c.draws;
    a.u = c.u64 ? static_cast<const double*>(c.u) : nullptr;
    a.u32 = c.u64 ? nullptr : static_cast<const float*>(c.u);
    a.temperature = c.temperature_rows;
    a.top_k = c.top_k_rows;
    a.top_p = c.top_p_rows;
    a.min_p = c.min_p_rows;
    a.temperature_v = c.temperature;
    a.top_k_v = c.top_k <= 0 ? 0 : c.top_k < c.n ? (int)c.top_k : (int)c.n;
    a.top_p_v = c.top_p;
    a.min_p_v = c.min_p;
    a.items = c.items;
    a.probs = c.probs;
    int bits = 0;
    while ((int64_t)1 << bits < c.n) ++bits;
    a.unit = std::ldexp(1.0, 62 - bits < 51 ? 62 - bits : 51);
    // which cuts some row may ask for
    const bool greedy = c.temperature_rows || !(c.temperature > 0.0) || c.top_p_rows || !(c.top_p > 0.0);
    const bool may_k = c.top_k_rows || c.top_k > 0 || greedy, may_p = c.top_p_rows || c.top_p < 1.0;
    const DrawArgs all = a;
    for (int64_t r = 0; r < all.rows; r += kLaunchMost) {
        auto from = [&](auto* p, int64_t step) { return p ? p + r * step : nullptr; };
        a.rows = std::min(all.rows - r, kLaunchMost);
        a.logits = static_cast<const char*>(all.logits) + r * all.ld * (c.dtype == NCF_F32 ? 4 : 2);
        a.mask = from(all.mask, all.mask_ld);
        a.u = from(all.u, all.draws);
        a.u32 = from(all.u32, all.draws);
        a.temperature = from(all.temperature, 1);
        a.top_k = from(all.top_k, 1);
        a.top_p = from(all.top_p, 1);
        a.min_p = from(all.min_p, 1);
        a.items = all.items + r * all.draws;
        a.probs = all.probs + r * all.draws;
        if (c.dtype == NCF_F32) draw_t<float>(a, c.ws, may_k, may_p, st);
        else if (c.dtype == NCF_BF16) draw_t<__bf16>(a, c.ws, may_k, may_p, st);
        else draw_t<_Float16>(a, c.ws, may_k, may_p, st);
        if (hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
}

}  // namespace ncf

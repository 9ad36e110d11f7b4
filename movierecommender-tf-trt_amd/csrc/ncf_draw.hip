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
// change a draw, and a running sum can never pass the total.  The draw differs from real arithmetic
// only where u lands within 2^-S of a border.  w itself is computed in 64 bits.
//
// The reference keeps the best of a list by np.argsort (movierec/trt_client.py:50-57); drawing from
// the scores is an extension of that ranking.

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
    int shift;                // S
    int32_t* items;
    float* probs;
};

// ----------------------------------------------------------------------------- keys and weights

// unsigned keys in the order of the floats; 0 stands for an item that is not allowed
__device__ __forceinline__ uint32_t ukey(float x) {
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unukey(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

// -0 and 0 are equal logits: one key
template <typename T>
__device__ __forceinline__ uint32_t item_key(T x, bool allowed) {
    const float f = (float)x + 0.0f;
    return (allowed && f > -INFINITY) ? ukey(f) : 0u;   // (a NaN compares false)
}

struct Weigher {
    double m, t, scale;
    uint32_t top;  // key of the best item

    __device__ __forceinline__ double real(uint32_t key) const {
        if (key == top) return 1.0;
        return fmax(exp(((double)unukey(key) - m) / t), 0.0);   // (infinities in both: NaN, no weight)
    }
    __device__ __forceinline__ uint64_t fixed(double w) const { return (uint64_t)rint(w * scale); }
};

// ----------------------------------------------------------------------------- one workgroup per row

constexpr int kDrawThreads = 1024;
constexpr int kDrawBins = 2048;

struct DrawShared {
    union {
        uint32_t count[kDrawBins];
        unsigned long long weight[kDrawBins];
    };
    unsigned long long wave64[kDrawThreads / 64];
    uint32_t wave32[kDrawThreads / 64];
    unsigned long long pick64;
    uint32_t pick_bin;
};

__device__ __forceinline__ unsigned long long shfl_up64(unsigned long long v, int d) {
    return (unsigned long long)__shfl_up((long long)v, d, 64);
}

// exclusive prefix over the workgroup, total to *sum
__device__ __forceinline__ unsigned long long block_before64(unsigned long long v, DrawShared& s,
                                                             unsigned long long* sum) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    unsigned long long inc = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned long long o = shfl_up64(inc, d);
        if (lane >= d) inc += o;
    }
    __syncthreads();
    if (lane == 63) s.wave64[w] = inc;
    __syncthreads();
    unsigned long long before = 0, all = 0;
    for (int j = 0; j < kDrawThreads / 64; ++j) {
        if (j < w) before += s.wave64[j];
        all += s.wave64[j];
    }
    *sum = all;
    return before + inc - v;
}

__device__ __forceinline__ uint32_t block_before32(uint32_t v, DrawShared& s, uint32_t* sum) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint32_t inc = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = (uint32_t)__shfl_up((int)inc, d, 64);
        if (lane >= d) inc += o;
    }
    __syncthreads();
    if (lane == 63) s.wave32[w] = inc;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (int j = 0; j < kDrawThreads / 64; ++j) {
        if (j < w) before += s.wave32[j];
        all += s.wave32[j];
    }
    *sum = all;
    return before + inc - v;
}

// (double)c >= p total, for a positive c: the one comparison that top-p makes
__device__ __forceinline__ bool reaches(unsigned long long c, double p, double total) {
    return c > 0 && (double)c >= p * total;
}

template <typename T>
struct RowView {
    const T* x;
    const uint8_t* mask;
    int n;
    __device__ __forceinline__ uint32_t key(int i) const {
        return item_key(x[i], mask == nullptr || mask[i] != 0);
    }
};

// key digits, most significant first: 11, 11 and 10 bits
__device__ __forceinline__ int digit_shift(int level) { return level == 0 ? 21 : level == 1 ? 10 : 0; }
__device__ __forceinline__ uint32_t digit_mask(int level) { return level == 2 ? 1023u : 2047u; }
__device__ __forceinline__ bool same_prefix(uint32_t a, uint32_t b, int level) {
    return level == 0 || (a >> digit_shift(level - 1)) == (b >> digit_shift(level - 1));
}

template <typename T>
__global__ __launch_bounds__(kDrawThreads) void k_draw(DrawArgs a) {
    __shared__ DrawShared s;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const RowView<T> r{static_cast<const T*>(a.logits) + row * a.ld, a.mask ? a.mask + row * a.mask_ld : nullptr,
                       a.n};
    const double t = a.temperature ? (double)a.temperature[row] : a.temperature_v;
    const double p = a.top_p ? (double)a.top_p[row] : a.top_p_v;
    double min_p = a.min_p ? (double)a.min_p[row] : a.min_p_v;
    min_p = min_p > 1.0 ? 1.0 : min_p;   // the best item always stays
    int k = a.top_k ? a.top_k[row] : a.top_k_v;
    if (!(t > 0.0) || p <= 0.0) k = 1;

    // the best item and how many are allowed
    uint32_t top = 0, allowed = 0;
    for (int i = tid; i < a.n; i += kDrawThreads) {
        const uint32_t key = r.key(i);
        top = max(top, key);
        allowed += key != 0;
    }
    block_before32(allowed, s, &allowed);
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
    __syncthreads();
    if ((tid & 63) == 0) s.wave32[tid >> 6] = top;
    __syncthreads();
    for (int j = 0; j < kDrawThreads / 64; ++j) top = max(top, s.wave32[j]);
    __syncthreads();
    if (allowed == 0) {
        for (int d = tid; d < a.draws; d += kDrawThreads) {
            a.items[row * a.draws + d] = -1;
            a.probs[row * a.draws + d] = 0.0f;
        }
        return;
    }
    const Weigher wt{(double)unukey(top), t > 0.0 ? t : 1.0, exp2((double)a.shift), top};

    // top-k: the k-th largest key, digit by digit
    uint32_t bound = 1, ties = 0xffffffffu;   // all allowed items
    if (k > 0 && (uint32_t)k < allowed) {
        uint32_t left = (uint32_t)k, prefix = 0;
        for (int level = 0; level < 3; ++level) {
            for (int b = tid; b < kDrawBins; b += kDrawThreads) s.count[b] = 0;
            __syncthreads();
            for (int i = tid; i < a.n; i += kDrawThreads) {
                const uint32_t key = r.key(i);
                if (key != 0 && same_prefix(key, prefix, level))
                    atomicAdd(&s.count[(key >> digit_shift(level)) & digit_mask(level)], 1u);
            }
            __syncthreads();
            // from the best digit down, two bins a thread
            const uint32_t c0 = s.count[kDrawBins - 1 - 2 * tid], c1 = s.count[kDrawBins - 2 - 2 * tid];
            uint32_t all;
            const uint32_t before = block_before32(c0 + c1, s, &all);
            if (before < left && before + c0 + c1 >= left) {
                const bool first = before + c0 >= left;
                s.pick_bin = kDrawBins - 1 - 2 * tid - (first ? 0 : 1);
                s.pick64 = before + (first ? 0 : c0);
            }
            __syncthreads();
            prefix |= s.pick_bin << digit_shift(level);
            left -= (uint32_t)s.pick64;
            __syncthreads();
        }
        bound = prefix;
        ties = left;
    }

    // top-p: the same over weights; of the bound's equals only `ties` count
    if (p > 0.0 && p < 1.0) {
        uint32_t equal = 0;
        if (ties != 0xffffffffu) {
            for (int i = tid; i < a.n; i += kDrawThreads) equal += r.key(i) == bound;
            block_before32(equal, s, &equal);
        }
        const unsigned long long over =
            ties != 0xffffffffu ? (unsigned long long)(equal - ties) * wt.fixed(wt.real(bound)) : 0;
        uint32_t prefix = 0;
        unsigned long long above = 0;
        double total = 0.0;
        for (int level = 0; level < 3; ++level) {
            for (int b = tid; b < kDrawBins; b += kDrawThreads) s.weight[b] = 0;
            __syncthreads();
            for (int i = tid; i < a.n; i += kDrawThreads) {
                const uint32_t key = r.key(i);
                if (key >= bound && same_prefix(key, prefix, level))
                    atomicAdd(&s.weight[(key >> digit_shift(level)) & digit_mask(level)],
                              (unsigned long long)wt.fixed(wt.real(key)));
            }
            __syncthreads();
            if (tid == 0 && over && same_prefix(bound, prefix, level))
                s.weight[(bound >> digit_shift(level)) & digit_mask(level)] -= over;
            __syncthreads();
            const unsigned long long c0 = s.weight[kDrawBins - 1 - 2 * tid], c1 = s.weight[kDrawBins - 2 - 2 * tid];
            unsigned long long all;
            const unsigned long long before = above + block_before64(c0 + c1, s, &all);
            if (level == 0) total = (double)all;
            if (!reaches(before, p, total) && reaches(before + c0 + c1, p, total)) {
                const bool first = reaches(before + c0, p, total);
                s.pick_bin = kDrawBins - 1 - 2 * tid - (first ? 0 : 1);
                s.pick64 = before + (first ? 0 : c0);
            }
            __syncthreads();
            prefix |= s.pick_bin << digit_shift(level);
            above = s.pick64;
            __syncthreads();
        }
        // of the equals of this key, as many as it takes
        const unsigned long long w = wt.fixed(wt.real(prefix));
        double want = ceil((p * total - (double)above) / (double)w);
        uint32_t j = want < 1.0 ? 1u : want > (double)a.n ? (uint32_t)a.n : (uint32_t)want;
        while (j > 1 && reaches(above + (unsigned long long)(j - 1) * w, p, total)) --j;
        while (j < (uint32_t)a.n && !reaches(above + (unsigned long long)j * w, p, total)) ++j;
        if (prefix > bound) {
            bound = prefix;
            ties = j;
        } else {
            ties = min(ties, j);
        }
    }

    // segments of the row: their weight and their equals of the bound
    const int per = (a.n + kDrawThreads - 1) / kDrawThreads;   // items of a thread, neighbours
    const int i0 = min(tid * per, a.n), i1 = min(i0 + per, a.n);
    uint32_t equal = 0, all32;
    for (int i = i0; i < i1; ++i) equal += r.key(i) == bound;
    const uint32_t ties_before = block_before32(equal, s, &all32);
    auto weigh = [&](int i, uint32_t& seen) -> unsigned long long {
        const uint32_t key = r.key(i);
        if (key < bound || key == 0) return 0;
        if (key == bound && seen++ >= ties) return 0;
        const double w = wt.real(key);
        return w >= min_p || !(min_p > 0.0) ? (unsigned long long)wt.fixed(w) : 0ull;
    };
    unsigned long long mine = 0, total;
    {
        uint32_t seen = ties_before;
        for (int i = i0; i < i1; ++i) mine += weigh(i, seen);
    }
    const unsigned long long before = block_before64(mine, s, &total);
    for (int d = 0; d < a.draws; ++d) {
        const int64_t o = row * a.draws + d;
        const double u = a.u ? a.u[o] : (double)a.u32[o];
        const double at = u * (double)total;
        // the first running sum above u total; a u outside [0, 1) takes the nearest end
        unsigned long long target = at > 0.0 ? (at >= 9.2e18 ? ~0ull >> 1 : (unsigned long long)at) : 0ull;
        if (target >= total) target = total - 1;
        if (target >= before && target < before + mine) {
            unsigned long long c = before;
            uint32_t seen = ties_before;
            for (int i = i0; i < i1; ++i) {
                const unsigned long long w = weigh(i, seen);
                c += w;
                if (c > target) {
                    a.items[o] = i;
                    a.probs[o] = (float)((double)w / (double)total);
                    break;
                }
            }
        }
    }
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
    a.shift = 62 - bits < 51 ? 62 - bits : 51;
    const dim3 grid((unsigned)c.rows);
    if (c.dtype == NCF_F32) launch(k_draw<float>, grid, kDrawThreads, 0, st, a);
    else if (c.dtype == NCF_BF16) launch(k_draw<__bf16>, grid, kDrawThreads, 0, st, a);
    else launch(k_draw<_Float16>, grid, kDrawThreads, 0, st, a);
    return hipGetLastError();
}

}  // namespace ncf

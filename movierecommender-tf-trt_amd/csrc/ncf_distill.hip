// Distillation from a teacher's best items: loss and gradient for a student's logits over the catalogue.
//
// For a row of student logits x over v items, temperature t and a teacher's list (item i_k, logit y_k):
//     p = softmax(x / t)                       q_k = exp(y_k / t - ref)
//     loss = sum_k q_k (log q_k - log p[i_k])  [ + q0 (log q0 - log p0) ]
//     d loss / d x_j = (p_j c_j - q(j)) / t,   q(j) = the q of the entries that name j
// ref is the log-sum-exp of the list's y / t (then c = sum q = 1), or, given the teacher's log-sum-exp
// over its whole catalogue, that: the mass outside the list is one more class, q0 = 1 - sum q against
// p0 = the student's mass outside, c = sum q + q0 inside the list and sum q + q0 - q0 / p0 outside.
// Left out: entries whose item lies outside [0, v) (padding), entries of no mass (y = -inf), the last
// class where either side has no mass there; a row without a list entry or whose logits are all -inf
// has loss and gradient 0.  An item named twice counts with both entries.
//
// The exponentials are fp32; their sums, the logarithms and everything of a list's length are 64 bits,
// because the loss is a small difference of large logarithms and q0 of numbers near one.  Inside and
// outside mass are summed apart, never by subtraction, both relative to the row's best logit; where that leaves
// less than 2^-28 of the mass outside (the list leads by 19 t), it is formed again relative to its own best, so it
// does not vanish however far the list leads.  With s_j = w_j / (its class's sum) the gradient outside is
//     s_j ((sum q + q0) p0 - q0) / t = s_j (sum q - q0 r) / (1 + r) / t,   r = inside mass / outside mass,
// and inside (s_j (sum q + q0) r / (1 + r) - q(j)) / t.  y / t and x / t are 64 bits: a q is off by |y / t| 2^-53 of
// itself, a loss by |x / t| 2^-53, nothing at ordinary temperatures (1e-9 at t = 1e-6).
//
// The reference trains on labels alone (binary cross-entropy, movierec/model.py:213-214).

#include <algorithm>
#include <cmath>

#include "ncf_common.h"
#include "ncf_internal.h"
#include "ncf_types.h"

namespace ncf {

constexpr int kDistThreads = 256;
constexpr int kDistItems = 32;                             // logits of a thread, in registers
constexpr int kDistChunk = kDistThreads * kDistItems;      // logits of a workgroup
constexpr int kDistWords = kDistChunk / 32;
constexpr int kState = NCF_DISTILL_STATE;                  // doubles of a row kept for the gradient

struct DistArgs {
    const void* x;
    int64_t ld;
    int64_t rows;
    int v, k, chunks;
    const void* idx;      // [rows][k], int32 or int64
    int idx64;
    const float* y;       // [rows][k]
    int64_t idx_ld, y_ld;
    const float* ref;     // [rows] or NULL
    double inv_t;
    float c2;             // log2(e) / t
    double2* sums;        // per chunk: mass outside and inside the list, each relative to its base
    float2* tops;         // per chunk: these bases; -inf for no mass
    double* state;        // [rows][kState]: both bases (32 bits each), factors outside and inside, sum q, ref
    float* loss;
    const float* gl;      // [rows] or NULL: gl_v
    float gl_v;
    void* grad;
    int64_t grad_ld;
};

__device__ __forceinline__ int64_t list_item(const DistArgs& a, int64_t row, int k) {
    return a.idx64 ? static_cast<const int64_t*>(a.idx)[row * a.idx_ld + k]
                   : (int64_t)static_cast<const int32_t*>(a.idx)[row * a.idx_ld + k];
}

__device__ __forceinline__ double wave_sum64(double x) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) x += __shfl_xor(x, d, 64);
    return x;
}
__device__ __forceinline__ double wave_max64(double x) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) x = fmax(x, __shfl_xor(x, d, 64));
    return x;
}
__device__ __forceinline__ float wave_max32(float x) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) x = fmaxf(x, __shfl_xor(x, d, 64));
    return x;
}

// over a workgroup of NT threads, in the same order for every thread
template <int NT>
struct BlockRed {
    double d[2][NT / 64];
    float f[NT / 64];
};
template <int NT>
__device__ __forceinline__ double block_sum64(double x, BlockRed<NT>& r) {
    x = wave_sum64(x);
    if constexpr (NT == 64) return x;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) r.d[0][threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0.0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) x += r.d[0][w];
    return x;
}
template <int NT>
__device__ __forceinline__ void block_sum64(double& x, double& y, BlockRed<NT>& r) {
    x = wave_sum64(x);
    y = wave_sum64(y);
    if constexpr (NT == 64) return;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        r.d[0][threadIdx.x >> 6] = x;
        r.d[1][threadIdx.x >> 6] = y;
    }
    __syncthreads();
    x = y = 0.0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        x += r.d[0][w];
        y += r.d[1][w];
    }
}
template <int NT>
__device__ __forceinline__ double block_max64(double x, BlockRed<NT>& r) {
    x = wave_max64(x);
    if constexpr (NT == 64) return x;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) r.d[0][threadIdx.x >> 6] = x;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) x = fmax(x, r.d[0][w]);
    return x;
}
template <int NT>
__device__ __forceinline__ float block_max32(float x, BlockRed<NT>& r) {
    x = wave_max32(x);
    if constexpr (NT == 64) return x;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) r.f[threadIdx.x >> 6] = x;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) x = fmaxf(x, r.f[w]);
    return x;
}

// one instruction, right to a unit in the last place; below 2^-126 it may give 0
__device__ __forceinline__ float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

// a thread's vectors of kVec neighbours: vector j starts at kVec (j kDistThreads + thread)
template <typename T, int NT = kDistThreads>
__device__ __forceinline__ int vec_at(int j) {
    return Elem<T>::kVec * (j * NT + (int)threadIdx.x);
}

// a thread's EPT logits as they are stored, and as floats; -inf past the end
template <int EPT, typename T>
struct Raw {
    static constexpr int V = Elem<T>::kVec, J = EPT / V;
    typedef T vec __attribute__((ext_vector_type(V)));
    vec v[J];
};
template <int NT, int EPT, typename T>
__device__ __forceinline__ void load_chunk(const T* x, int left, Raw<EPT, T>& r) {
    constexpr int V = Elem<T>::kVec;
#pragma unroll
    for (int j = 0; j < EPT / V; ++j) {
        const int o = vec_at<T, NT>(j);
        if (o + V <= left) {
            r.v[j] = *reinterpret_cast<const typename Elem<T>::vec*>(x + o);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) r.v[j][e] = o + e < left ? x[o + e] : (T)(-INFINITY);
        }
    }
}
template <int EPT, typename T>
__device__ __forceinline__ void to_floats(const Raw<EPT, T>& r, float (&x)[EPT]) {
    constexpr int V = Elem<T>::kVec;
#pragma unroll
    for (int j = 0; j < EPT / V; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) x[V * j + e] = (float)r.v[j][e];
}

// the list's bits of the items [first, first + 32 WORDS)
template <int NT, int WORDS>
__device__ __forceinline__ void mark_list(const DistArgs& a, int64_t row, int first, uint32_t* bits) {
    for (int w = threadIdx.x; w < WORDS; w += NT) bits[w] = 0;
    __syncthreads();
    for (int k = threadIdx.x; k < a.k; k += NT) {
        const int64_t i = list_item(a, row, k) - first;
        if (i >= 0 && i < 32 * WORDS) atomicOr(&bits[i >> 5], 1u << (i & 31));
    }
    __syncthreads();
}

__device__ __forceinline__ float base_of(float m) { return m > -INFINITY ? m : 0.0f; }

// The least mass outside, relative to the row's best logit, that is not formed again.  (A sum's relative error is
// that of its weights on the average, 1.5 2^-23 z / ln 2 with z <= ln n + 19 < 42 then.)  A row that needs it is
// read twice more (2,048 x 27,278 bf16, lists of 32 in every row 60 ahead: 145 us, so 62), others pay a comparison.
// (A base for each class from the start: a pass over the list's bits for the maxima, 62 -> 97.)
constexpr double kRestLeast = 0x1p-28;

// A row's best logit, the bases of its masses outside and inside the list, and the masses.
struct RowMass {
    float top, base_out, base_in;
    double out, in;
};

// f(item, logit) for those of v items that `bits` does not mark, a vector at a time: what a rare row needs once more.
template <int NT, typename T, typename F>
__device__ __forceinline__ void each_outside(const T* x, int v, const uint32_t* bits, F f) {
    constexpr int V = Elem<T>::kVec;
#pragma unroll 1
    for (int o = V * (int)threadIdx.x; o < v; o += V * NT) {
        Raw<V, T> raw;
        if (o + V <= v) {
            raw.v[0] = *reinterpret_cast<const typename Elem<T>::vec*>(x + o);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) raw.v[0][e] = o + e < v ? x[o + e] : (T)(-INFINITY);
        }
        const uint32_t b = bits[o >> 5] >> (o & 31);
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (o + e < v && !(b >> e & 1u)) f(o + e, (float)raw.v[0][e]);
    }
}
// The mass outside relative to its own best logit.
template <int NT, typename T>
__device__ __forceinline__ void outside_again(const T* x, int v, const uint32_t* bits, float c2, float& base, double& sum,
                                              BlockRed<NT>& red) {
    float top = -INFINITY;
    each_outside<NT>(x, v, bits, [&](int, float y) { top = fmaxf(top, y); });
    const float b = base_of(block_max32(top, red));
    double s = 0.0;
    each_outside<NT>(x, v, bits, [&](int, float y) { s += (double)pow2((y - b) * c2); });
    sum = block_sum64(s, red);
    base = b;
}
// Whether a row (chunk) is such: most of it lies in the list.
__device__ __forceinline__ bool little_outside(const DistArgs& a, double out, double in) {
    return a.ref && out < kRestLeast && in != 0.0;
}

// Maxima and masses of one chunk of a row.
template <typename T>
__global__ __launch_bounds__(kDistThreads) void k_distill_sums(DistArgs a) {
    __shared__ BlockRed<kDistThreads> red;
    __shared__ uint32_t bits[kDistWords];
    constexpr int V = Elem<T>::kVec;
    const int64_t row = blockIdx.x / a.chunks;
    const int chunk = (int)(blockIdx.x - row * a.chunks), first = chunk * kDistChunk;
    Raw<kDistItems, T> raw;
    load_chunk<kDistThreads>(static_cast<const T*>(a.x) + row * a.ld + first, a.v - first, raw);
    if (a.ref) mark_list<kDistThreads, kDistWords>(a, row, first, bits);
    float x[kDistItems];
    to_floats(raw, x);
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < kDistItems; ++e) m = fmaxf(m, x[e]);
    m = block_max32(m, red);
    float base = base_of(m);
    double out = 0.0, in = 0.0;
#pragma unroll
    for (int j = 0; j < kDistItems / V; ++j) {
        const int o = vec_at<T>(j);
        const uint32_t b = a.ref ? bits[o >> 5] >> (o & 31) : 0u;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const double w = (double)pow2((x[V * j + e] - base) * a.c2);
            if (b >> e & 1u) in += w;
            else out += w;
        }
    }
    block_sum64(out, in, red);
    if (little_outside(a, out, in))
        outside_again<kDistThreads>(static_cast<const T*>(a.x) + row * a.ld + first, min(a.v - first, kDistChunk), bits,
                                    a.c2, base, out, red);
    if (threadIdx.x == 0) {
        a.tops[blockIdx.x] = make_float2(out != 0.0 ? base : -INFINITY, m);
        a.sums[blockIdx.x] = make_double2(out, in);
    }
}

// What depends on a row's list alone: the teacher's reference, sum q, sum q log q and sum q x.
struct ListSums {
    double ref, q, q_log_q, q_x;
};

// y / t, rounded: fused into a later subtraction it would no longer equal itself (where y / t is large, a best entry's
// q would be e to the half step that its own reference was rounded by)
__device__ __forceinline__ double list_z(float y, double inv_t) {
#pragma clang fp contract(off)
    return (double)y * inv_t;
}

// A thread's first entry of the list, loaded ahead of the row.
struct ListEntry {
    int64_t item;   // -1: none
    double z;       // y / t
    float x;
};
template <typename T>
__device__ __forceinline__ ListEntry list_entry(const DistArgs& a, int64_t row, const T* x, int k) {
    ListEntry e{-1, 0.0, 0.0f};
    if (k < a.k) {
        const int64_t i = list_item(a, row, k);
        if (i >= 0 && i < a.v) {
            e.item = i;
            e.z = list_z(a.y[row * a.y_ld + k], a.inv_t);
            e.x = (float)x[i];
        }
    }
    return e;
}
// f(entry) for the thread's entries k = thread, thread + NT, ..
template <int NT, typename T, typename F>
__device__ __forceinline__ void each_entry(const DistArgs& a, int64_t row, const T* x, const ListEntry& first, F f) {
    if (first.item >= 0) f(first);
    for (int k = threadIdx.x + NT; k < a.k; k += NT) {
        const ListEntry e = list_entry(a, row, x, k);
        if (e.item >= 0) f(e);
    }
}

template <int NT, typename T>
__device__ __forceinline__ ListSums list_sums(const DistArgs& a, int64_t row, const T* x, const ListEntry& first,
                                              BlockRed<NT>& red) {
    ListSums l{};
    if (a.ref) {   // the teacher's reference: given, or the list's own
        l.ref = (double)a.ref[row];
    } else {
        double top = -INFINITY, s = 0.0;
        each_entry<NT>(a, row, x, first, [&](const ListEntry& e) { top = fmax(top, e.z); });
        top = block_max64(top, red);
        each_entry<NT>(a, row, x, first, [&](const ListEntry& e) {
            if (top > -INFINITY) s += exp(e.z - top);
        });
        s = block_sum64(s, red);
        l.ref = s != 0.0 ? top + log(s) : INFINITY;   // no entry: q = 0
    }
    each_entry<NT>(a, row, x, first, [&](const ListEntry& e) {
        const double lq = e.z - l.ref, q = exp(lq);
        l.q += q;
        if (q != 0.0) {
            l.q_log_q += q * lq;
            l.q_x += q * (double)e.x;
        }
    });
    block_sum64(l.q, l.q_log_q, red);
    l.q_x = block_sum64(l.q_x, red);
    return l;
}

// What the gradient of a row needs: an item's is factor * exp2((x - base) c2) - q(item), each side of the list with
// its own.  And for the loss what lies between the two sides.
struct RowState {
    float base_out, base_in;
    double f_out, f_in, ref;
    double way;     // (base_in - base_out) / t: 0, or positive where the mass outside has a base of its own
    double less;    // inside mass / outside mass, its inverse where way > 0
    bool rest;      // the mass outside is a class
    bool dead;      // no logit left
};

__device__ __forceinline__ RowState row_state(const DistArgs& a, const RowMass& m, const ListSums& l) {
    RowState st{};
    st.base_out = m.base_out;
    st.base_in = m.base_in;
    st.ref = l.ref;
    st.dead = !(m.top > -INFINITY) && m.out + m.in == 0.0;   // (NaN logits: a NaN sum)
    if (st.dead) {
        st.ref = INFINITY;
        return st;
    }
    if (!a.ref) {   // one class, the one outside
        st.f_out = st.f_in = 1.0 / m.out * l.q;
        return st;
    }
    const double q0 = 1.0 - l.q;
    st.rest = q0 > 0.0 && !(m.out <= 0.0);
    st.way = ((double)m.base_in - (double)m.base_out) * a.inv_t;
    const bool own = st.way > 0.0 || m.out == 0.0;
    st.less = m.out == 0.0 ? 0.0 : own ? exp(-st.way) * (m.out / m.in) : m.in / m.out;
    const double part = 1.0 / (1.0 + st.less), p0 = own ? st.less * part : part, p1 = own ? part : st.less * part;
    const double c = st.rest ? l.q + q0 : l.q;
    // (c p0 - q0 without its cancellation)
    st.f_out = st.rest ? (own ? l.q * st.less - q0 : l.q - q0 * st.less) * part : c * p0;
    st.f_out = m.out == 0.0 ? 0.0 : st.f_out / m.out;
    st.f_in = m.in == 0.0 ? 0.0 : c * p1 / m.in;
    return st;
}

// Its loss, by one thread; and the state, for a gradient later.
__device__ __forceinline__ void write_row(const DistArgs& a, int64_t row, const RowState& st, const RowMass& m,
                                          const ListSums& l) {
    // sum q (log q - log p) with log p = (x - base) / t - log sum
    const bool own = a.ref && (st.way > 0.0 || m.out == 0.0);
    const double sum = (own ? m.in : m.out) * (1.0 + st.less);
    double loss = l.q_log_q - (l.q_x - l.q * (double)st.base_in) * a.inv_t + l.q * log(sum);
    if (st.rest) {   // q0 (log q0 - log p0)
        const double log_p0 = own ? -(st.way + log(m.in / m.out) + log1p(st.less)) : -log1p(st.less);
        loss += (1.0 - l.q) * (log1p(-l.q) - log_p0);
    }
    if (a.state) {
        double* to = a.state + row * kState;
        to[0] = __hiloint2double(__float_as_int(st.base_in), __float_as_int(st.base_out));
        to[1] = st.f_out;
        to[2] = st.f_in;
        to[3] = l.q;
        to[4] = st.ref;
    }
    a.loss[row] = st.dead || (l.q == 0.0 && !a.ref) ? 0.0f : (float)loss;
}

// The row's loss and what its gradient needs.
template <typename T>
__global__ __launch_bounds__(kDistThreads) void k_distill_loss(DistArgs a) {
    __shared__ BlockRed<kDistThreads> red;
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ld;
    const ListEntry entry = list_entry(a, row, x, threadIdx.x);
    float top = -INFINITY, top_out = -INFINITY;
    for (int c = threadIdx.x; c < a.chunks; c += kDistThreads) {
        const float2 t = a.tops[row * a.chunks + c];
        top_out = fmaxf(top_out, t.x);
        top = fmaxf(top, t.y);
    }
    top = block_max32(top, red);
    top_out = block_max32(top_out, red);
    RowMass m{top, base_of(top_out), base_of(top), 0.0, 0.0};
    for (int c = threadIdx.x; c < a.chunks; c += kDistThreads) {
        const float2 t = a.tops[row * a.chunks + c];
        const double2 s = a.sums[row * a.chunks + c];
        m.out += s.x * (t.x > -INFINITY ? exp(((double)t.x - (double)m.base_out) * a.inv_t) : 1.0);
        m.in += s.y * (t.y > -INFINITY ? exp(((double)t.y - (double)m.base_in) * a.inv_t) : 1.0);
    }
    block_sum64(m.out, m.in, red);
    const ListSums sums = list_sums<kDistThreads>(a, row, x, entry, red);
    if (threadIdx.x == 0) write_row(a, row, row_state(a, m, sums), m, sums);
}

// The list's q by item: a bit map, the marked items ahead of each of its words, and the q of each marked item as an
// integer (the sum of an item's entries does not depend on their order), in units of 2^-51 times a power of two above
// the whole list's q: that may be as large or small as the teacher's log-sum-exp makes it.
template <int NT, int WORDS>
struct ItemQ {
    uint32_t bits[WORDS];
    uint32_t before[WORDS];
    unsigned long long q[NCF_DISTILL_MAX_K];
    uint32_t wave[NT / 64];
    int power;   // of that

    __device__ __forceinline__ uint32_t slot(int o) const {
        return before[o >> 5] + __popc(bits[o >> 5] & ((1u << (o & 31)) - 1u));
    }
    __device__ __forceinline__ double at(int o) const { return ldexp((double)q[slot(o)], power - 51); }

    // (no finite sum: c inside and outside the list are not finite either, and so is no gradient)
    __device__ __forceinline__ static int power_of(double sum_q) {
        return sum_q > 0.0 && sum_q < INFINITY ? ilogb(sum_q) + 1 : 0;
    }

    // from the marked bits (mark_list)
    __device__ __forceinline__ void fill(const DistArgs& a, int64_t row, int first, double ref, double sum_q) {
        constexpr int W = (WORDS + NT - 1) / NT;
        const int lane = threadIdx.x & 63, w0 = W * (int)threadIdx.x;
        uint32_t n[W], mine = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            n[w] = w0 + w < WORDS ? __popc(bits[w0 + w]) : 0;
            mine += n[w];
        }
        uint32_t inc = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = (uint32_t)__shfl_up((int)inc, d, 64);
            if (lane >= d) inc += o;
        }
        if (lane == 63) wave[threadIdx.x >> 6] = inc;
        if (threadIdx.x == 0) power = power_of(sum_q);
        __syncthreads();
        uint32_t ahead = inc - mine, total = 0;
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) {
            ahead += w < (int)(threadIdx.x >> 6) ? wave[w] : 0;
            total += wave[w];
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w0 + w < WORDS) before[w0 + w] = ahead;
            ahead += n[w];
        }
        for (uint32_t s = threadIdx.x; s < total; s += NT) q[s] = 0;
        __syncthreads();
        for (int k = threadIdx.x; k < a.k; k += NT) {
            const int64_t i = list_item(a, row, k) - first;
            if (i < 0 || i >= 32 * WORDS || i + first >= a.v) continue;
            const double e = ldexp(exp(list_z(a.y[row * a.y_ld + k], a.inv_t) - ref), 51 - power_of(sum_q));
            atomicAdd(&q[slot((int)i)], (unsigned long long)rint(fmin(e, 0x1p52)));
        }
        __syncthreads();
    }
};

// V neighbours' gradients from their weights, o items behind `first`
template <typename T, typename Q>
__device__ __forceinline__ void store_grad(T* out, int o, int left, const float* w, uint32_t b, float p_in,
                                           float p_out, double g, const Q& l) {
    constexpr int V = Elem<T>::kVec;
    float r[V];
#pragma unroll
    for (int e = 0; e < V; ++e) r[e] = w[e] * ((b >> e & 1u) ? p_in : p_out);
    if (b & ((1u << V) - 1u)) {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (b >> e & 1u) r[e] -= (float)(l.at(o + e) * g);
    }
    if (o + V <= left) {
        typename Elem<T>::vec y;
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = (T)r[e];
        *reinterpret_cast<typename Elem<T>::vec*>(out + o) = y;
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (o + e < left) out[o + e] = (T)r[e];
    }
}

// 64 rows of 1,000,000 fp32: sums 62 us (4.1 TB/s), gradient 79 (6.5 TB/s, part of the logits from the cache).
// Gradient of NT EPT items of a row, `chunks` such a row.  From the last row to the first: what the pass over
// the sums read last is still in the cache.
template <typename T, int NT, int EPT>
__global__ __launch_bounds__(NT) void k_distill_grad(DistArgs a, int chunks) {
    constexpr int V = Elem<T>::kVec, WORDS = NT * EPT / 32;
    __shared__ ItemQ<NT, WORDS> l;
    const int64_t at = (int64_t)gridDim.x - 1 - blockIdx.x, row = at / chunks;
    const int first = (int)(at - row * chunks) * NT * EPT;
    Raw<EPT, T> raw;
    load_chunk<NT>(static_cast<const T*>(a.x) + row * a.ld + first, a.v - first, raw);
    const double* st = a.state + row * kState;
    const float base_out = __int_as_float(__double2loint(st[0])), base_in = __int_as_float(__double2hiint(st[0]));
    const double g = (double)(a.gl ? a.gl[row] : a.gl_v) * a.inv_t;
    const float p_out = (float)(st[1] * g), p_in = (float)(st[2] * g);
    mark_list<NT, WORDS>(a, row, first, l.bits);
    l.fill(a, row, first, st[4], st[3]);
    T* out = static_cast<T*>(a.grad) + row * a.grad_ld + first;
    float x[EPT];
    to_floats(raw, x);
#pragma unroll
    for (int j = 0; j < EPT / V; ++j) {
        const int o = vec_at<T, NT>(j);
        const uint32_t b = l.bits[o >> 5] >> (o & 31) & ((1u << V) - 1u);
        float w[V];
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = pow2((x[V * j + e] - base_out) * a.c2);
        if (b != 0 && base_in != base_out) {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (b >> e & 1u) w[e] = pow2((x[V * j + e] - base_in) * a.c2);
        }
        store_grad(out, o, a.v - first, w, b, p_in, p_out, g, l);
    }
}

// A whole row in a workgroup's registers: read once, its loss, and its gradient written.  NT EPT items at
// most; 56 of a thread leave two workgroups of 512 a CU.
template <typename T, int NT, int EPT, bool GRAD>
__global__ __launch_bounds__(NT, 4) void k_distill_row(DistArgs a) {
    constexpr int V = Elem<T>::kVec, WORDS = NT * EPT / 32;
    __shared__ BlockRed<NT> red;
    __shared__ ItemQ<NT, WORDS> l;
    const int64_t row = blockIdx.x;
    const T* px = static_cast<const T*>(a.x) + row * a.ld;
    // the list first: its arithmetic and the row do not fit the registers together (the CU's other workgroup
    // reads meanwhile)
    const ListSums sums = list_sums<NT>(a, row, px, list_entry(a, row, px, threadIdx.x), red);
    if (GRAD || a.ref) mark_list<NT, WORDS>(a, row, 0, l.bits);
    if constexpr (GRAD) l.fill(a, row, 0, sums.ref, sums.q);
    __builtin_amdgcn_sched_barrier(0);
    Raw<EPT, T> raw;
    load_chunk<NT>(px, a.v, raw);
    float x[EPT];
    to_floats(raw, x);
    RowMass m{};
    m.top = -INFINITY;
#pragma unroll
    for (int e = 0; e < EPT; ++e) m.top = fmaxf(m.top, x[e]);
    m.top = block_max32(m.top, red);
    m.base_out = m.base_in = base_of(m.top);
#pragma unroll
    for (int j = 0; j < EPT / V; ++j) {
        const int o = vec_at<T, NT>(j);
        const uint32_t b = a.ref ? l.bits[o >> 5] >> (o & 31) & ((1u << V) - 1u) : 0u;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            x[V * j + e] = pow2((x[V * j + e] - m.base_in) * a.c2);
            if (b == 0) m.out += (double)x[V * j + e];
        }
        if (b != 0) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (b >> e & 1u) m.in += (double)x[V * j + e];
                else m.out += (double)x[V * j + e];
            }
        }
        __builtin_amdgcn_sched_barrier(0);   // (a vector at a time: registers for one)
    }
    block_sum64(m.out, m.in, red);
    const bool again = little_outside(a, m.out, m.in);
    if (again) outside_again<NT>(px, a.v, l.bits, a.c2, m.base_out, m.out, red);
    const RowState st = row_state(a, m, sums);
    if (GRAD && again) {
        const double g = (double)(a.gl ? a.gl[row] : a.gl_v) * a.inv_t;
        const float p_in = (float)(st.f_in * g), p_out = (float)(st.f_out * g);
        T* to = static_cast<T*>(a.grad) + row * a.grad_ld;
        each_outside<NT>(px, a.v, l.bits, [&](int o, float y) { to[o] = (T)(pow2((y - st.base_out) * a.c2) * p_out); });
        for (int k = threadIdx.x; k < a.k; k += NT) {   // (entries that name one item write the same there)
            const ListEntry e = list_entry(a, row, px, k);
            if (e.item >= 0)
                to[e.item] = (T)(pow2((e.x - st.base_in) * a.c2) * p_in - (float)(l.at((int)e.item) * g));
        }
    } else if constexpr (GRAD) {
        const double g = (double)(a.gl ? a.gl[row] : a.gl_v) * a.inv_t;
        const float p_in = (float)(st.f_in * g), p_out = (float)(st.f_out * g);
        const double q_g = st.dead ? 0.0 : g;   // (a row with no logit left has no gradient)
        T* to = static_cast<T*>(a.grad) + row * a.grad_ld;
#pragma unroll
        for (int j = 0; j < EPT / V; ++j) {
            const int o = vec_at<T, NT>(j);
            store_grad(to, o, a.v, x + V * j, l.bits[o >> 5] >> (o & 31), p_in, p_out, q_g, l);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // (the logarithms last: they and the row do not fit the registers together)
    if (threadIdx.x == 0) write_row(a, row, st, m, sums);
}

// The same for lists of up to 64 entries: the first wave holds the list, an entry a lane, and works on it
// while the row is on its way, without a barrier; the gradient's q are taken off the written row at the end.
// 2,048 rows of 27,278 bf16 logits, lists of 32: 59 us (kernel 53, 4.2 TB/s), by the kernel above 88; fp32 96 and
// 125.  Bound by memory, a workgroup's reads, sums and writes one behind the other.
constexpr int kWaveList = 64;

template <typename T, int NT, int EPT, bool GRAD>
__global__ __launch_bounds__(NT, 4) void k_distill_row_wave(DistArgs a) {
    constexpr int V = Elem<T>::kVec, WORDS = NT * EPT / 32;
    __shared__ BlockRed<NT> red;
    __shared__ uint32_t bits[WORDS];
    __shared__ ListSums list;
    __shared__ double list_q[kWaveList];
    __shared__ int list_at[kWaveList];
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const T* px = static_cast<const T*>(a.x) + row * a.ld;
    ListEntry entry{-1, 0.0, 0.0f};
    if (wave == 0) entry = list_entry(a, row, px, lane);
    __builtin_amdgcn_sched_barrier(0);
    Raw<EPT, T> raw;
    load_chunk<NT>(px, a.v, raw);
    __builtin_amdgcn_sched_barrier(0);
    if (a.ref) {
        for (int w = threadIdx.x; w < WORDS; w += NT) bits[w] = 0;
        __syncthreads();
    }
    if (wave == 0) {
        const bool in = entry.item >= 0;
        ListSums l{};
        if (a.ref) {
            l.ref = (double)a.ref[row];
            if (in) atomicOr(&bits[entry.item >> 5], 1u << (entry.item & 31));
        } else {
            const double top = wave_max64(in ? entry.z : -INFINITY);
            const double s = wave_sum64(in && top > -INFINITY ? exp(entry.z - top) : 0.0);
            l.ref = s != 0.0 ? top + log(s) : INFINITY;   // no entry: q = 0
        }
        const double lq = entry.z - l.ref, q = in ? exp(lq) : 0.0;
        l.q = wave_sum64(q);
        l.q_log_q = wave_sum64(q != 0.0 ? q * lq : 0.0);
        l.q_x = wave_sum64(q != 0.0 ? q * (double)entry.x : 0.0);
        list_q[lane] = q;
        list_at[lane] = in ? (int)entry.item : -1;
        if (lane == 0) list = l;
    }
    __builtin_amdgcn_sched_barrier(0);
    float x[EPT];
    to_floats(raw, x);
    RowMass m{};
    m.top = -INFINITY;
#pragma unroll
    for (int e = 0; e < EPT; ++e) m.top = fmaxf(m.top, x[e]);
    m.top = block_max32(m.top, red);
    __syncthreads();   // (and the list)
    m.base_out = m.base_in = base_of(m.top);
#pragma unroll
    for (int j = 0; j < EPT / V; ++j) {
        const int o = vec_at<T, NT>(j);
        const uint32_t b = a.ref ? bits[o >> 5] >> (o & 31) & ((1u << V) - 1u) : 0u;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            x[V * j + e] = pow2((x[V * j + e] - m.base_in) * a.c2);
            if (b == 0) m.out += (double)x[V * j + e];
        }
        if (b != 0) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (b >> e & 1u) m.in += (double)x[V * j + e];
                else m.out += (double)x[V * j + e];
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    block_sum64(m.out, m.in, red);
    const bool again = little_outside(a, m.out, m.in);
    if (again) outside_again<NT>(px, a.v, bits, a.c2, m.base_out, m.out, red);
    const RowState st = row_state(a, m, list);
    if constexpr (GRAD) {
        const double g = (double)(a.gl ? a.gl[row] : a.gl_v) * a.inv_t;
        const float p_in = (float)(st.f_in * g), p_out = (float)(st.f_out * g);
        T* to = static_cast<T*>(a.grad) + row * a.grad_ld;
        if (again) {
            each_outside<NT>(px, a.v, bits,
                             [&](int o, float y) { to[o] = (T)(pow2((y - st.base_out) * a.c2) * p_out); });
        } else {
#pragma unroll
            for (int j = 0; j < EPT / V; ++j) {
                const int o = vec_at<T, NT>(j);
                if (o + V <= a.v) {
                    typename Elem<T>::vec y;
#pragma unroll
                    for (int e = 0; e < V; ++e) y[e] = (T)(x[V * j + e] * p_out);
                    *reinterpret_cast<typename Elem<T>::vec*>(to + o) = y;
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (o + e < a.v) to[o + e] = (T)(x[V * j + e] * p_out);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // the list's items once more, when every wave's stores of the row have arrived
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (wave == 0 && entry.item >= 0) {
            double q = 0.0;   // of all entries that name the item, in their order
            for (int k = 0; k < a.k; ++k) q += list_at[k] == (int)entry.item ? list_q[k] : 0.0;
            const float w = pow2((entry.x - st.base_in) * a.c2);
            to[entry.item] = (T)(w * p_in - (float)(q * (st.dead ? 0.0 : g)));
        }
    }
    if (threadIdx.x == 0) write_row(a, row, st, m, list);
}

static DistArgs dist_args(const ncf_distill_t& c, void* ws) {
    DistArgs a{};
    a.x = c.logits;
    a.ld = c.ld;
    a.rows = c.rows;
    a.v = (int)c.v;
    a.k = (int)c.k;
    a.chunks = (a.v + kDistChunk - 1) / kDistChunk;
    a.idx = c.teacher_items;
    a.idx64 = c.items64;
    a.idx_ld = c.items_ld;
    a.y = c.teacher_logits;
    a.y_ld = c.teacher_ld;
    a.ref = c.teacher_lse;
    a.inv_t = 1.0 / c.temperature;
    a.c2 = (float)(1.4426950408889634 / c.temperature);
    a.state = c.state;
    a.loss = c.loss;
    a.gl = c.grad_loss;
    a.gl_v = c.grad_loss_value;
    a.grad = c.grad;
    a.grad_ld = c.grad_ld;
    a.sums = static_cast<double2*>(ws);
    if (ws) {
        const int64_t n = c.rows * a.chunks;
        a.tops = reinterpret_cast<float2*>(a.sums + n);
        if (!a.state) a.state = reinterpret_cast<double*>(a.tops + n);
    }
    return a;
}

// A row goes to one workgroup where its registers hold it, however few the rows (27,278 fp32 logits by chunks:
// one row 18.7 us, so 13.1; 512 rows 44 and 23; 2,048 rows 146 and 96).
// Twice as long a row, a CU's registers full, only with a list that a wave holds (40,000 logits, lists of 32: one
// row 18.7 us, so 14.6; 1,024 rows 93 and 86).
constexpr int64_t kRowMost = 512 * 56;
static bool by_row(int64_t v, int64_t k) { return v <= kRowMost || (v <= 2 * kRowMost && k <= kWaveList); }

// Rows of one launch at most: HIP counts a launch's threads in 32 bits, and 2^21 workgroups have up to 2^31.  More
// rows go in several launches, one behind the other, that share the workspace.
static int64_t launch_rows(int64_t v) {
    return std::max<int64_t>(1, ((int64_t)1 << 21) / ((v + kDistChunk - 1) / kDistChunk));
}

// for the chunks' sums and, behind them, the state where the caller takes none
size_t distill_workspace(int64_t rows, int v, int64_t k) {
    if (by_row(v, k)) return 0;
    rows = std::min(rows, launch_rows(v));
    const size_t n = (size_t)rows * ((v + kDistChunk - 1) / kDistChunk);
    return n * (sizeof(double2) + sizeof(float2)) + (size_t)rows * kState * sizeof(double);
}
int64_t distill_chunks(int64_t rows, int v) {
    const int64_t c = (v + kDistChunk - 1) / kDistChunk;
    return rows > INT64_MAX / c ? INT64_MAX : rows * c;
}

template <typename T, int NT, int EPT>
static void distill_row(const DistArgs& a, bool backward, hipStream_t st) {
    const dim3 grid((unsigned)a.rows);
    if (a.k <= kWaveList) {
        if (backward) launch(k_distill_row_wave<T, NT, EPT, true>, grid, NT, 0, st, a);
        else launch(k_distill_row_wave<T, NT, EPT, false>, grid, NT, 0, st, a);
        return;
    }
    if (backward) launch(k_distill_row<T, NT, EPT, true>, grid, NT, 0, st, a);
    else launch(k_distill_row<T, NT, EPT, false>, grid, NT, 0, st, a);
}

// The smallest workgroup that holds a row, and the next one (us for 4,096 rows, lists of 32): 500 logits 13.7 and
// 16.5, 2,000 18.5 and 33, 8,000 47 and 104.
template <typename T>
static hipError_t distill_t(const DistArgs& a, bool forward, bool backward, hipStream_t st) {
    const unsigned grid = (unsigned)(a.rows * a.chunks);
    if (forward && by_row(a.v, a.k)) {
        if (a.v <= 64 * 8) distill_row<T, 64, 8>(a, backward, st);
        else if (a.v <= 64 * 32) distill_row<T, 64, 32>(a, backward, st);
        else if (a.v <= 256 * 32) distill_row<T, 256, 32>(a, backward, st);
        else if (a.v <= 512 * 56) distill_row<T, 512, 56>(a, backward, st);
        else if (backward) launch(k_distill_row_wave<T, 1024, 56, true>, dim3((unsigned)a.rows), 1024, 0, st, a);
        else launch(k_distill_row_wave<T, 1024, 56, false>, dim3((unsigned)a.rows), 1024, 0, st, a);
        return hipGetLastError();
    }
    if (forward) {
        launch(k_distill_sums<T>, dim3(grid), kDistThreads, 0, st, a);
        launch(k_distill_loss<T>, dim3((unsigned)a.rows), kDistThreads, 0, st, a);
    }
    if (backward) {
        if (a.v <= 64 * 8) launch(k_distill_grad<T, 64, 8>, dim3((unsigned)a.rows), 64, 0, st, a, 1);
        else if (a.v <= 64 * 32) launch(k_distill_grad<T, 64, 32>, dim3((unsigned)a.rows), 64, 0, st, a, 1);
        else launch(k_distill_grad<T, kDistThreads, kDistItems>, dim3(grid), kDistThreads, 0, st, a, a.chunks);
    }
    return hipGetLastError();
}

hipError_t launch_distill(const ncf_distill_t& c, void* ws, bool forward, bool backward, hipStream_t st) {
    const int64_t size = c.dtype == NCF_F32 ? 4 : 2, most = launch_rows(c.v);
    for (int64_t r = 0; r < c.rows; r += most) {
        auto from = [&](auto* p, int64_t step) { return p ? p + r * step : nullptr; };
        ncf_distill_t part = c;
        part.rows = std::min(c.rows - r, most);
        part.logits = static_cast<const char*>(c.logits) + r * c.ld * size;
        part.teacher_items = static_cast<const char*>(c.teacher_items) + r * c.items_ld * (c.items64 ? 8 : 4);
        part.teacher_logits = c.teacher_logits + r * c.teacher_ld;
        part.teacher_lse = from(c.teacher_lse, 1);
        part.grad_loss = from(c.grad_loss, 1);
        part.loss = from(c.loss, 1);
        part.state = from(c.state, kState);
        part.grad = from(static_cast<char*>(c.grad), c.grad_ld * size);
        const DistArgs a = dist_args(part, ws);
        hipError_t e = c.dtype == NCF_F32 ? distill_t<float>(a, forward, backward, st)
                       : c.dtype == NCF_BF16 ? distill_t<__bf16>(a, forward, backward, st)
                                             : distill_t<_Float16>(a, forward, backward, st);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace ncf

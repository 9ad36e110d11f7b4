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
// outside mass are summed apart, never by subtraction.
//
// The reference trains on labels alone (binary cross-entropy, movierec/model.py:213-214).

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
    double2* sums;        // per chunk: mass outside and inside the list, relative to the chunk's max
    float* tops;          // per chunk: its max
    double* state;        // [rows][kState]: max, 1 / sum, c inside, c outside, ref
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

template <int NT, int EPT, typename T>
__device__ __forceinline__ void load_chunk(const T* x, int left, float (&r)[EPT]) {
    constexpr int V = Elem<T>::kVec;
#pragma unroll
    for (int j = 0; j < EPT / V; ++j) {
        const int o = vec_at<T, NT>(j);
        if (o + V <= left) {
            const typename Elem<T>::vec w = *reinterpret_cast<const typename Elem<T>::vec*>(x + o);
#pragma unroll
            for (int e = 0; e < V; ++e) r[V * j + e] = (float)w[e];
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) r[V * j + e] = o + e < left ? (float)x[o + e] : -INFINITY;
        }
    }
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

// Max and masses of one chunk of a row.
template <typename T>
__global__ __launch_bounds__(kDistThreads) void k_distill_sums(DistArgs a) {
    __shared__ BlockRed<kDistThreads> red;
    __shared__ uint32_t bits[kDistWords];
    constexpr int V = Elem<T>::kVec;
    const int64_t row = blockIdx.x / a.chunks;
    const int chunk = (int)(blockIdx.x - row * a.chunks), first = chunk * kDistChunk;
    float x[kDistItems];
    load_chunk<kDistThreads, kDistItems>(static_cast<const T*>(a.x) + row * a.ld + first, a.v - first, x);
    if (a.ref) mark_list<kDistThreads, kDistWords>(a, row, first, bits);
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < kDistItems; ++e) m = fmaxf(m, x[e]);
    m = block_max32(m, red);
    const float base = m > -INFINITY ? m : 0.0f;
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
    if (threadIdx.x == 0) {
        a.tops[blockIdx.x] = m;
        a.sums[blockIdx.x] = make_double2(out, in);
    }
}

// What the gradient of a row needs.
struct RowState {
    float base;             // the largest logit
    double inv_sum, c_in, c_out, ref;
};

// The row's loss and state from its max m and its masses outside and inside the list; NT threads.
template <int NT, typename T>
__device__ __forceinline__ RowState finish_row(const DistArgs& a, int64_t row, const T* x, float m, double out,
                                               double in, BlockRed<NT>& red) {
    const float base = m > -INFINITY ? m : 0.0f;
    const double sum = out + in;
    // the teacher's reference: given, or the list's own
    double ref;
    if (a.ref) {
        ref = (double)a.ref[row];
    } else {
        double top = -INFINITY;
        for (int k = threadIdx.x; k < a.k; k += NT) {
            const int64_t i = list_item(a, row, k);
            if (i >= 0 && i < a.v) top = fmax(top, (double)a.y[row * a.y_ld + k] * a.inv_t);
        }
        top = block_max64(top, red);
        double s = 0.0;
        for (int k = threadIdx.x; k < a.k; k += NT) {
            const int64_t i = list_item(a, row, k);
            if (i >= 0 && i < a.v && top > -INFINITY) s += exp((double)a.y[row * a.y_ld + k] * a.inv_t - top);
        }
        s = block_sum64(s, red);
        ref = s != 0.0 ? top + log(s) : INFINITY;   // no entry: q = 0
    }
    const double log_sum = log(sum);
    double loss = 0.0, q_sum = 0.0;
    for (int k = threadIdx.x; k < a.k; k += NT) {
        const int64_t i = list_item(a, row, k);
        if (i < 0 || i >= a.v) continue;
        const double lq = (double)a.y[row * a.y_ld + k] * a.inv_t - ref, q = exp(lq);
        q_sum += q;
        if (q != 0.0) loss += q * (lq - (((double)(float)x[i] - (double)base) * a.inv_t - log_sum));
    }
    block_sum64(loss, q_sum, red);
    double inside = q_sum, outside = q_sum;
    if (a.ref) {
        const double q0 = 1.0 - q_sum;
        if (q0 > 0.0 && !(out <= 0.0)) {
            loss += q0 * (log1p(-q_sum) + log1p(in / out));
            inside = q_sum + q0;
            outside = inside - q0 * (sum / out);
        }
    }
    const bool none = !(m > -INFINITY) && sum == 0.0;   // (a NaN logit leaves a NaN sum)
    const RowState st = none ? RowState{base, 0.0, 0.0, 0.0, INFINITY}
                             : RowState{base, 1.0 / sum, inside, outside, ref};
    if (threadIdx.x == 0) {
        double* to = a.state + row * kState;
        to[0] = st.base;
        to[1] = st.inv_sum;
        to[2] = st.c_in;
        to[3] = st.c_out;
        to[4] = st.ref;
        a.loss[row] = none ? 0.0f : (float)loss;
    }
    return st;
}

// The row's loss and what its gradient needs.
template <typename T>
__global__ __launch_bounds__(kDistThreads) void k_distill_loss(DistArgs a) {
    __shared__ BlockRed<kDistThreads> red;
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ld;
    float m = -INFINITY;
    for (int c = threadIdx.x; c < a.chunks; c += kDistThreads) m = fmaxf(m, a.tops[row * a.chunks + c]);
    m = block_max32(m, red);
    const float base = m > -INFINITY ? m : 0.0f;
    double out = 0.0, in = 0.0;
    for (int c = threadIdx.x; c < a.chunks; c += kDistThreads) {
        const float mc = a.tops[row * a.chunks + c];
        const double f = mc > -INFINITY ? exp(((double)mc - (double)base) * a.inv_t) : 1.0;
        const double2 s = a.sums[row * a.chunks + c];
        out += s.x * f;
        in += s.y * f;
    }
    block_sum64(out, in, red);
    finish_row<kDistThreads>(a, row, x, m, out, in, red);
}

// The list's q by item: a bit map, the marked items ahead of each of its words, and the q of each marked
// item in units of 2^-51 (integers: the sum of an item's entries does not depend on their order).
template <int NT, int WORDS>
struct ItemQ {
    uint32_t bits[WORDS];
    uint32_t before[WORDS];
    unsigned long long q[NCF_DISTILL_MAX_K];
    uint32_t wave[NT / 64];

    __device__ __forceinline__ uint32_t slot(int o) const {
        return before[o >> 5] + __popc(bits[o >> 5] & ((1u << (o & 31)) - 1u));
    }
    __device__ __forceinline__ double at(int o) const { return (double)q[slot(o)] * 0x1p-51; }

    // from the marked bits (mark_list)
    __device__ __forceinline__ void fill(const DistArgs& a, int64_t row, int first, double ref) {
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
            // (no q of a log-sum-exp passes 1, up to its rounding; a NaN has made c inside and outside NaN)
            const double e = exp((double)a.y[row * a.y_ld + k] * a.inv_t - ref);
            atomicAdd(&q[slot((int)i)], (unsigned long long)rint(fmin(e, 2.0) * 0x1p51));
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

// Gradient of one chunk of a row.
template <typename T>
__global__ __launch_bounds__(kDistThreads) void k_distill_grad(DistArgs a) {
    __shared__ ItemQ<kDistThreads, kDistWords> l;
    constexpr int V = Elem<T>::kVec;
    const int64_t row = blockIdx.x / a.chunks;
    const int chunk = (int)(blockIdx.x - row * a.chunks), first = chunk * kDistChunk;
    float x[kDistItems];
    load_chunk<kDistThreads, kDistItems>(static_cast<const T*>(a.x) + row * a.ld + first, a.v - first, x);
    const double* st = a.state + row * kState;
    const float base = (float)st[0];
    const double g = (double)(a.gl ? a.gl[row] : a.gl_v) * a.inv_t;
    const float p_in = (float)(st[1] * st[2] * g), p_out = (float)(st[1] * st[3] * g);
    mark_list<kDistThreads, kDistWords>(a, row, first, l.bits);
    l.fill(a, row, first, st[4]);
    T* out = static_cast<T*>(a.grad) + row * a.grad_ld + first;
#pragma unroll
    for (int j = 0; j < kDistItems / V; ++j) {
        const int o = vec_at<T>(j);
        float w[V];
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = pow2((x[V * j + e] - base) * a.c2);
        store_grad(out, o, a.v - first, w, l.bits[o >> 5] >> (o & 31), p_in, p_out, g, l);
    }
}

// A whole row in a workgroup's registers: read once, its loss, and its gradient written.  NT EPT items at
// most; 56 of a thread leave two workgroups of 512 a CU.
template <typename T, int NT, int EPT, bool GRAD>
__global__ __launch_bounds__(NT) void k_distill_row(DistArgs a) {
    constexpr int V = Elem<T>::kVec, WORDS = NT * EPT / 32;
    __shared__ BlockRed<NT> red;
    __shared__ ItemQ<NT, WORDS> l;
    const int64_t row = blockIdx.x;
    const T* px = static_cast<const T*>(a.x) + row * a.ld;
    float x[EPT];
    load_chunk<NT, EPT>(px, a.v, x);
    if (GRAD || a.ref) mark_list<NT, WORDS>(a, row, 0, l.bits);
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < EPT; ++e) m = fmaxf(m, x[e]);
    m = block_max32(m, red);
    const float base = m > -INFINITY ? m : 0.0f;
    double out = 0.0, in = 0.0;
#pragma unroll
    for (int j = 0; j < EPT / V; ++j) {
        const int o = vec_at<T, NT>(j);
        const uint32_t b = a.ref ? l.bits[o >> 5] >> (o & 31) & ((1u << V) - 1u) : 0u;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float w = pow2((x[V * j + e] - base) * a.c2);
            x[V * j + e] = w;
            if (b == 0) out += (double)w;
        }
        if (b != 0) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (b >> e & 1u) in += (double)x[V * j + e];
                else out += (double)x[V * j + e];
            }
        }
    }
    block_sum64(out, in, red);
    const RowState st = finish_row<NT>(a, row, px, m, out, in, red);
    if constexpr (GRAD) {
        const double g = (double)(a.gl ? a.gl[row] : a.gl_v) * a.inv_t;
        const float p_in = (float)(st.inv_sum * st.c_in * g), p_out = (float)(st.inv_sum * st.c_out * g);
        l.fill(a, row, 0, st.ref);
        T* to = static_cast<T*>(a.grad) + row * a.grad_ld;
#pragma unroll
        for (int j = 0; j < EPT / V; ++j) {
            const int o = vec_at<T, NT>(j);
            store_grad(to, o, a.v, x + V * j, l.bits[o >> 5] >> (o & 31), p_in, p_out, g, l);
        }
    }
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
    a.tops = ws ? reinterpret_cast<float*>(a.sums + c.rows * a.chunks) : nullptr;
    return a;
}

size_t distill_workspace(int64_t rows, int v) {
    const size_t n = (size_t)rows * ((v + kDistChunk - 1) / kDistChunk);
    return n * (sizeof(double2) + sizeof(float));
}
int64_t distill_blocks(int64_t rows, int v) {
    const int64_t c = (v + kDistChunk - 1) / kDistChunk;
    return rows > INT64_MAX / c ? INT64_MAX : rows * c;
}

template <typename T, int NT, int EPT>
static void distill_row(const DistArgs& a, bool backward, hipStream_t st) {
    const dim3 grid((unsigned)a.rows);
    if (backward) launch(k_distill_row<T, NT, EPT, true>, grid, NT, 0, st, a);
    else launch(k_distill_row<T, NT, EPT, false>, grid, NT, 0, st, a);
}

template <typename T>
static hipError_t distill_t(const DistArgs& a, bool forward, bool backward, hipStream_t st) {
    const unsigned grid = (unsigned)(a.rows * a.chunks);
    // few rows of more than a chunk each would leave CUs idle: those go by chunks
    const bool by_row = a.v <= kDistChunk || (a.v <= 512 * 56 && a.rows >= 128);
    if (forward && by_row) {
        if (a.v <= 64 * 8) distill_row<T, 64, 8>(a, backward, st);
        else if (a.v <= 64 * 32) distill_row<T, 64, 32>(a, backward, st);
        else if (a.v <= 256 * 32) distill_row<T, 256, 32>(a, backward, st);
        else distill_row<T, 512, 56>(a, backward, st);
        return hipGetLastError();
    }
    if (forward) {
        launch(k_distill_sums<T>, dim3(grid), kDistThreads, 0, st, a);
        launch(k_distill_loss<T>, dim3((unsigned)a.rows), kDistThreads, 0, st, a);
    }
    if (backward) launch(k_distill_grad<T>, dim3(grid), kDistThreads, 0, st, a);
    return hipGetLastError();
}

hipError_t launch_distill(const ncf_distill_t& c, void* ws, bool forward, bool backward, hipStream_t st) {
    if (c.rows <= 0) return hipSuccess;
    const DistArgs a = dist_args(c, ws);
    if (c.dtype == NCF_F32) return distill_t<float>(a, forward, backward, st);
    if (c.dtype == NCF_BF16) return distill_t<__bf16>(a, forward, backward, st);
    return distill_t<_Float16>(a, forward, backward, st);
}

}  // namespace ncf

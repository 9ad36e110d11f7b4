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

struct BlockRed {
    double d[kDistThreads / 64];
    float f[kDistThreads / 64];
};
__device__ __forceinline__ double block_sum64(double x, BlockRed& r) {
    x = wave_sum64(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) r.d[threadIdx.x >> 6] = x;
    __syncthreads();
    return (r.d[0] + r.d[1]) + (r.d[2] + r.d[3]);
}
__device__ __forceinline__ double block_max64(double x, BlockRed& r) {
    x = wave_max64(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) r.d[threadIdx.x >> 6] = x;
    __syncthreads();
    return fmax(fmax(r.d[0], r.d[1]), fmax(r.d[2], r.d[3]));
}
__device__ __forceinline__ float block_max32(float x, BlockRed& r) {
    x = wave_max32(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) r.f[threadIdx.x >> 6] = x;
    __syncthreads();
    return fmaxf(fmaxf(r.f[0], r.f[1]), fmaxf(r.f[2], r.f[3]));
}

// a thread's vectors of kVec neighbours: vector j starts at kVec (j kDistThreads + thread)
template <typename T>
__device__ __forceinline__ int vec_at(int j) {
    return Elem<T>::kVec * (j * kDistThreads + (int)threadIdx.x);
}

template <typename T>
__device__ __forceinline__ void load_chunk(const T* x, int left, float (&r)[kDistItems]) {
    constexpr int V = Elem<T>::kVec;
#pragma unroll
    for (int j = 0; j < kDistItems / V; ++j) {
        const int o = vec_at<T>(j);
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

// the chunk's bits of the list
__device__ __forceinline__ void mark_list(const DistArgs& a, int64_t row, int first, uint32_t* bits) {
    for (int w = threadIdx.x; w < kDistWords; w += kDistThreads) bits[w] = 0;
    __syncthreads();
    for (int k = threadIdx.x; k < a.k; k += kDistThreads) {
        const int64_t i = list_item(a, row, k) - first;
        if (i >= 0 && i < kDistChunk) atomicOr(&bits[i >> 5], 1u << (i & 31));
    }
    __syncthreads();
}

// Max and masses of one chunk of a row.
template <typename T>
__global__ __launch_bounds__(kDistThreads) void k_distill_sums(DistArgs a) {
    __shared__ BlockRed red;
    __shared__ uint32_t bits[kDistWords];
    constexpr int V = Elem<T>::kVec;
    const int64_t row = blockIdx.x / a.chunks;
    const int chunk = (int)(blockIdx.x - row * a.chunks), first = chunk * kDistChunk;
    float x[kDistItems];
    load_chunk(static_cast<const T*>(a.x) + row * a.ld + first, a.v - first, x);
    if (a.ref) mark_list(a, row, first, bits);
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
            const double w = (double)exp2f((x[V * j + e] - base) * a.c2);
            if (b >> e & 1u) in += w;
            else out += w;
        }
    }
    out = block_sum64(out, red);
    in = block_sum64(in, red);
    if (threadIdx.x == 0) {
        a.tops[blockIdx.x] = m;
        a.sums[blockIdx.x] = make_double2(out, in);
    }
}

// The row's loss and what its gradient needs.
template <typename T>
__global__ __launch_bounds__(kDistThreads) void k_distill_loss(DistArgs a) {
    __shared__ BlockRed red;
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
    out = block_sum64(out, red);
    in = block_sum64(in, red);
    const double sum = out + in;
    // the teacher's reference: given, or the list's own
    double ref;
    if (a.ref) {
        ref = (double)a.ref[row];
    } else {
        double top = -INFINITY;
        for (int k = threadIdx.x; k < a.k; k += kDistThreads) {
            const int64_t i = list_item(a, row, k);
            if (i >= 0 && i < a.v) top = fmax(top, (double)a.y[row * a.y_ld + k] * a.inv_t);
        }
        top = block_max64(top, red);
        double s = 0.0;
        for (int k = threadIdx.x; k < a.k; k += kDistThreads) {
            const int64_t i = list_item(a, row, k);
            if (i >= 0 && i < a.v && top > -INFINITY) s += exp((double)a.y[row * a.y_ld + k] * a.inv_t - top);
        }
        s = block_sum64(s, red);
        ref = s != 0.0 ? top + log(s) : INFINITY;   // no entry: q = 0
    }
    const double log_sum = log(sum);
    double loss = 0.0, q_sum = 0.0;
    for (int k = threadIdx.x; k < a.k; k += kDistThreads) {
        const int64_t i = list_item(a, row, k);
        if (i < 0 || i >= a.v) continue;
        const double lq = (double)a.y[row * a.y_ld + k] * a.inv_t - ref, q = exp(lq);
        q_sum += q;
        if (q != 0.0) loss += q * (lq - (((double)(float)x[i] - (double)base) * a.inv_t - log_sum));
    }
    loss = block_sum64(loss, red);
    q_sum = block_sum64(q_sum, red);
    if (threadIdx.x != 0) return;
    double inside = q_sum, outside = q_sum;
    if (a.ref) {
        const double q0 = 1.0 - q_sum;
        if (q0 > 0.0 && !(out <= 0.0)) {
            loss += q0 * (log1p(-q_sum) + log1p(in / out));
            inside = q_sum + q0;
            outside = inside - q0 * (sum / out);
        }
    }
    double* st = a.state + row * kState;
    const bool none = !(m > -INFINITY) && sum == 0.0;   // (a NaN logit leaves a NaN sum)
    st[0] = base;
    st[1] = none ? 0.0 : 1.0 / sum;
    st[2] = none ? 0.0 : inside;
    st[3] = none ? 0.0 : outside;
    st[4] = none ? INFINITY : ref;
    a.loss[row] = none ? 0.0f : (float)loss;
}

struct ChunkList {
    uint32_t bits[kDistWords];
    uint32_t before[kDistWords];               // marked items ahead of each word
    unsigned long long q[NCF_DISTILL_MAX_K];   // q of the chunk's marked items in 2^-51
    int scan[4];
};

// Gradient of one chunk of a row.
template <typename T>
__global__ __launch_bounds__(kDistThreads) void k_distill_grad(DistArgs a) {
    static_assert(kDistWords == kDistThreads, "one word of the bit map a thread");
    __shared__ ChunkList l;
    constexpr int V = Elem<T>::kVec;
    const int64_t row = blockIdx.x / a.chunks;
    const int chunk = (int)(blockIdx.x - row * a.chunks), first = chunk * kDistChunk;
    float x[kDistItems];
    load_chunk(static_cast<const T*>(a.x) + row * a.ld + first, a.v - first, x);
    const double* st = a.state + row * kState;
    const float base = (float)st[0];
    const double ref = st[4];
    const double g = (double)(a.gl ? a.gl[row] : a.gl_v) * a.inv_t;
    const float p_in = (float)(st[1] * st[2] * g), p_out = (float)(st[1] * st[3] * g);
    mark_list(a, row, first, l.bits);
    int total;
    l.before[threadIdx.x] = (uint32_t)block_exscan_256(__popc(l.bits[threadIdx.x]), l.scan, &total);
    for (int s = threadIdx.x; s < total; s += kDistThreads) l.q[s] = 0;
    __syncthreads();
    auto slot = [&](int o) { return l.before[o >> 5] + __popc(l.bits[o >> 5] & ((1u << (o & 31)) - 1u)); };
    for (int k = threadIdx.x; k < a.k; k += kDistThreads) {
        const int64_t i = list_item(a, row, k) - first;
        if (i < 0 || i >= kDistChunk || i + first >= a.v) continue;
        const double q = exp((double)a.y[row * a.y_ld + k] * a.inv_t - ref);
        // integers: the sum of an item's entries does not depend on their order.  (No q of a log-sum-exp
        // passes 1, up to its rounding; a NaN has made the row's p_in and p_out NaN.)
        atomicAdd(&l.q[slot((int)i)], (unsigned long long)rint(fmin(q, 2.0) * 0x1p51));
    }
    __syncthreads();
    T* out = static_cast<T*>(a.grad) + row * a.grad_ld + first;
    const int left = a.v - first;
#pragma unroll
    for (int j = 0; j < kDistItems / V; ++j) {
        const int o = vec_at<T>(j);
        const uint32_t b = l.bits[o >> 5] >> (o & 31);
        float r[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float w = exp2f((x[V * j + e] - base) * a.c2);
            r[e] = w * ((b >> e & 1u) ? p_in : p_out);
            if (b >> e & 1u) r[e] -= (float)((double)l.q[slot(o + e)] * 0x1p-51 * g);
        }
        if (o + V <= left) {
            typename Elem<T>::vec w;
#pragma unroll
            for (int e = 0; e < V; ++e) w[e] = (T)r[e];
            *reinterpret_cast<typename Elem<T>::vec*>(out + o) = w;
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (o + e < left) out[o + e] = (T)r[e];
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

template <typename T>
static hipError_t distill_t(const DistArgs& a, bool forward, bool backward, hipStream_t st) {
    const unsigned grid = (unsigned)(a.rows * a.chunks);
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

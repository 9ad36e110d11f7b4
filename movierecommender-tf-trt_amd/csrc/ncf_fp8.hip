// Block-scaled 8-bit operands: the quantiser and the product that scores users against a catalogue.
//
// An operand is held as e4m3 values q with one fp32 scale s per 128 consecutive values of a row (or
// per 128 x 128 tile): x ~ s q, s = max(max|x| / 448, 2^-126), q = e4m3(x / s), both roundings to
// nearest even.  The product is
//     y[m][n] = bias[n] + sum_j sa[m][j] sb[n][j] (sum over block j of qa[m][k] qb[n][k]),
// a block's sum on MFMA from a zero accumulator, then added, scaled, to the fp32 total, which is rounded
// once to the output's type.  The e4m3 values are widened to fp16 (exact) for v_mfma_f32_16x16x32_f16, whose
// products and sums are fp32 (relative error of a random 128-block 9e-9).  The 8-bit instruction
// v_mfma_f32_16x16x128_f8f6f4 has twice the rate, but it aligns the products of each 8 neighbouring k to the
// largest and drops what lies more than 13 binary places below its exponent (448 * 448 + 4 - 448 * 448 gives
// 0): where products cancel, 16-bit outputs see that too.  v_mfma_f32_16x16x32_fp8_fp8 drops the same.
//
// The reference scores one user against a list of items (movierec/trt_client.py:43-57).

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "ncf_common.h"
#include "ncf_internal.h"
#include "ncf_types.h"

namespace ncf {

constexpr int kScaleBlock = 128;
constexpr float kE4m3Max = 448.0f;
constexpr float kMinScale = 0x1p-126f;  // the smallest normal number: a block of zeros divides by it

// ----------------------------------------------------------------------------- quantiser

template <typename T>
__device__ __forceinline__ vf32x4 load4(const T* p, int valid) {
    vf32x4 r = {0.0f, 0.0f, 0.0f, 0.0f};
    if (valid >= 4) {
        typedef T v4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
        const v4 x = *reinterpret_cast<const v4*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = (float)x[e];
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (e < valid) r[e] = (float)p[e];
    }
    return r;
}

// the largest magnitude as bits: above every finite number stand infinity, then NaN, so both stay
__device__ __forceinline__ uint32_t mag4(vf32x4 x) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
    return m;
}

// a NaN among the values makes the scale NaN (fmaxf would drop it)
__device__ __forceinline__ float scale_of(uint32_t mag) {
    const float a = __uint_as_float(mag) / kE4m3Max;
    return a < kMinScale ? kMinScale : a;
}

__device__ __forceinline__ void store_q4(uint8_t* q, vf32x4 x, float s, int valid) {
    int w = 0;
    w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] / s, x[1] / s, w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] / s, x[3] / s, w, true);
    if (valid >= 4) {
        typedef int iu __attribute__((aligned(1)));
        *reinterpret_cast<iu*>(q) = w;
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (e < valid) q[e] = (uint8_t)(w >> (8 * e));
    }
}

// One scale per 128 values of a row: 32 lanes hold a block, four values each, and find its maximum by five
// exchanges; the values are read once.  Bound by memory: 1,000,000 x 128 fp32 133 us, 4.8 TB/s.
template <typename T>
__global__ __launch_bounds__(kBlock) void k_quantize_rows(const T* __restrict__ x, int64_t ld, int64_t blocks, int kb,
                                                          int cols, uint8_t* __restrict__ q, int64_t q_ld,
                                                          float* __restrict__ scale) {
    const int l = threadIdx.x & 31;
    const int64_t step = (int64_t)gridDim.x * (kBlock / 32);
    for (int64_t b = (int64_t)blockIdx.x * (kBlock / 32) + (threadIdx.x >> 5); b < blocks; b += step) {
        const int64_t row = b / kb;
        const int c = (int)(b - row * kb) * kScaleBlock + 4 * l;
        const vf32x4 v = load4(x + row * ld + c, cols - c);
        uint32_t m = mag4(v);
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d, 32));
        const float s = scale_of(m);
        if (l == 0) scale[b] = s;
        store_q4(q + row * q_ld + c, v, s, cols - c);
    }
}

// One scale per 128 x 128 tile: a workgroup holds the tile in registers, so that it too is read once.
template <typename T>
__global__ __launch_bounds__(kBlock) void k_quantize_tiles(const T* __restrict__ x, int64_t ld, int64_t rows, int kb,
                                                           int cols, uint8_t* __restrict__ q, int64_t q_ld,
                                                           float* __restrict__ scale) {
    __shared__ uint32_t red[kBlock / 64];
    const int64_t rb = blockIdx.x / kb;
    const int c = (int)(blockIdx.x - rb * kb) * kScaleBlock + 4 * (threadIdx.x & 31);
    const int64_t r0 = rb * kScaleBlock + (threadIdx.x >> 5);
    vf32x4 v[16];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int64_t row = r0 + 8 * i;
        v[i] = load4(x + (row < rows ? row : 0) * ld + c, row < rows ? cols - c : 0);
        m = max(m, mag4(v[i]));
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    const float s = scale_of(max(max(red[0], red[1]), max(red[2], red[3])));
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int64_t row = r0 + 8 * i;
        if (row < rows) store_q4(q + row * q_ld + c, v[i], s, cols - c);
    }
}

template <typename T>
static hipError_t quantize_t(const T* x, int64_t rows, int cols, int64_t ld, int tile, uint8_t* q, int64_t q_ld,
                             float* scale, hipStream_t st) {
    const int kb = (cols + kScaleBlock - 1) / kScaleBlock;
    if (tile) {
        const int64_t grid = (rows + kScaleBlock - 1) / kScaleBlock * kb;
        launch(k_quantize_tiles<T>, dim3((unsigned)grid), kBlock, 0, st, x, ld, rows, kb, cols, q, q_ld, scale);
    } else {
        const int64_t blocks = rows * kb;
        int64_t grid = (blocks + kBlock / 32 - 1) / (kBlock / 32);
        if (grid > 256 * 64) grid = 256 * 64;
        launch(k_quantize_rows<T>, dim3((unsigned)grid), kBlock, 0, st, x, ld, blocks, kb, cols, q, q_ld, scale);
    }
    return hipGetLastError();
}

hipError_t launch_quantize(const void* x, int dtype, int64_t rows, int cols, int64_t ld, int tile, uint8_t* q,
                           int64_t q_ld, float* scale, hipStream_t st) {
    if (rows <= 0) return hipSuccess;
    if (dtype == NCF_F32)
        return quantize_t(static_cast<const float*>(x), rows, cols, ld, tile, q, q_ld, scale, st);
    if (dtype == NCF_BF16)
        return quantize_t(static_cast<const __bf16*>(x), rows, cols, ld, tile, q, q_ld, scale, st);
    return quantize_t(static_cast<const _Float16*>(x), rows, cols, ld, tile, q, q_ld, scale, st);
}

// ----------------------------------------------------------------------------- product

typedef int mi32x8 __attribute__((ext_vector_type(8)));

typedef _Float16 mf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 mf16x2 __attribute__((ext_vector_type(2)));

// 8 of a fragment's 32 values in fp16
__device__ __forceinline__ mf16x8 widen(mi32x8 f, int e) {
    mf16x8 r;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const mf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(f[2 * e + w], 1.0f, false);
        const mf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(f[2 * e + w], 1.0f, true);
        r[4 * w + 0] = lo[0];
        r[4 * w + 1] = lo[1];
        r[4 * w + 2] = hi[0];
        r[4 * w + 3] = hi[1];
    }
    return r;
}

// One block of 128: both operands hold lane l's row l & 15 and 32 of its values, the same columns in both
// for the same l >> 4 (which of them share an instruction does not matter: a sum over k has no order).

// 16 values from column c on of a row of k values, zero past its end
__device__ __forceinline__ vu32x4 load_q16(const uint8_t* row, int c, int k) {
    if (c + 16 <= k) return load16(row + c);
    vu32x4 r = {0, 0, 0, 0};
    for (int e = 0; c + e < k; ++e) r[e >> 2] |= (uint32_t)row[c + e] << (8 * (e & 3));
    return r;
}

__device__ __forceinline__ mi32x8 load_frag(const uint8_t* row, int c, int k) {
    const vu32x4 lo = load_q16(row, c, k), hi = load_q16(row, c + 16, k);
    return mi32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

// a fragment as the MFMA takes it: widened once, for all the products it enters
struct Operand {
    mf16x8 v[4];
    __device__ __forceinline__ void set(mi32x8 f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = widen(f, e);
    }
    __device__ __forceinline__ static vf32x4 product(const Operand& a, const Operand& b) {
        vf32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < 4; ++e) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[e], b.v[e], d, 0, 0, 0);
        return d;
    }
};

struct MmArgs {
    const uint8_t* a;
    const uint8_t* b;
    const float* sa;    // [m][kb]
    const float* sb;    // [n][kb], or [ceil(n / 128)][kb] with b_tile
    const float* bias;  // [n], bias_step apart, or NULL
    void* y;
    int64_t lda, ldb, ldy;
    int64_t m, n;
    int k, kb, b_tile, bias_step;
    int64_t mt, nt;     // tiles along m and n
};

// y[m][n .. n + 4), the lane's four neighbouring columns
template <typename TO>
__device__ __forceinline__ void store_y4(TO* p, vf32x4 v, int valid) {
    typedef TO o4 __attribute__((ext_vector_type(4), aligned(sizeof(TO))));
    if (valid >= 4) {
        o4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (TO)v[e];
        *reinterpret_cast<o4*>(p) = o;
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (e < valid) p[e] = (TO)v[e];
    }
}

// Operands straight from memory to registers.  A wave computes 16 MI rows of y by 16 NI columns; the
// rows of b are the MFMA's A operand, so a lane ends with four neighbouring columns of one row of y.  Small
// products, bound by latency (1 x 27,278 x 64 fp32: 3.9 us), operands at any alignment.
template <int MI, int NI, typename TO>
__global__ __launch_bounds__(kBlock) void k_mm_direct(MmArgs p) {
    const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
    const int64_t wave = (int64_t)blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6);
    if (wave >= p.mt * p.nt) return;
    const int64_t m0 = wave / p.nt * (16 * MI), n0 = wave % p.nt * (16 * NI);
    vf32x4 acc[MI][NI];
#pragma unroll
    for (int x = 0; x < MI; ++x)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[x][j] = vf32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // rows past the end repeat the last one: what they give is not stored
    const uint8_t* ar[MI];
    const uint8_t* br[NI];
#pragma unroll
    for (int x = 0; x < MI; ++x) ar[x] = p.a + min(m0 + 16 * x + i, p.m - 1) * p.lda;
#pragma unroll
    for (int j = 0; j < NI; ++j) br[j] = p.b + min(n0 + 16 * j + i, p.n - 1) * p.ldb;
    for (int kb = 0; kb < p.kb; ++kb) {
        const int c = kb * kScaleBlock + 32 * g;
        Operand fb[NI];
        vf32x4 sb[NI];
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            fb[j].set(load_frag(br[j], c, p.k));
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t n = min(n0 + 16 * j + 4 * g + r, p.n - 1);
                sb[j][r] = p.sb[(p.b_tile ? n / kScaleBlock : n) * p.kb + kb];
            }
        }
#pragma unroll
        for (int x = 0; x < MI; ++x) {
            Operand fa;
            fa.set(load_frag(ar[x], c, p.k));
            const float sa = p.sa[min(m0 + 16 * x + i, p.m - 1) * p.kb + kb];
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const vf32x4 d = Operand::product(fb[j], fa);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[x][j][r] = fmaf(sa * sb[j][r], d[r], acc[x][j][r]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NI; ++j) {
        const int64_t n = n0 + 16 * j + 4 * g;
        const int valid = (int)min((int64_t)4, p.n - n);
        if (valid <= 0) continue;
        vf32x4 bias = {0.0f, 0.0f, 0.0f, 0.0f};
        if (p.bias)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (r < valid) bias[r] = p.bias[(n + r) * p.bias_step];
#pragma unroll
        for (int x = 0; x < MI; ++x) {
            const int64_t m = m0 + 16 * x + i;
            if (m < p.m) store_y4(static_cast<TO*>(p.y) + m * p.ldy + n, acc[x][j] + bias, valid);
        }
    }
}

// ----------------------------------------------------------------------------- large products
//
// 256 x 256 of y a workgroup of eight waves (64 rows by 128 columns each), 128 of k a step.  Both
// operands' steps go straight from memory to LDS (16 bytes a lane), the next while this one is multiplied.
// In LDS the 16-byte pieces of a row are permuted by the row (piece c at c ^ (row / 2 % 8)), so the 16
// lanes that read a fragment touch all 64 banks; a lane's fragment is pieces g and g + 4 of its row, in
// both operands alike.  8,192 x 4,096 x 4,096 with a scale per tile: bf16 out 238 us, 1.15 PFLOP/s, fp32 out 244
// (a library product of 8,192^3 in bf16 reaches 1.25); matrix instructions are busy 44 % of the time, widening and
// scaled additions beside them.

constexpr int kTile = 256, kTileThreads = 512, kTileWaves = kTileThreads / 64;
constexpr int kTileMI = 4, kTileNI = 8;   // 16-row, 16-column tiles of a wave

struct TileStage {
    uint8_t a[kTile * kScaleBlock];
    uint8_t b[kTile * kScaleBlock];
    float sa[kTile];
    float sb[kTile];
};

// Rows [r0, r0 + 256) of an operand, step j, into LDS; rows past the end repeat the last one.  A thread
// stages piece tid % 8 of rows tid / 8 + 64 i, in LDS order.
__device__ __forceinline__ void stage_rows(const uint8_t* q, int64_t ld, int64_t rows, int64_t r0, int j,
                                           uint8_t* lds) {
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t t = threadIdx.x >> 3, c = 16 * ((threadIdx.x & 7) ^ (t >> 1 & 7));
#pragma unroll
    for (int i = 0; i < kTile / 64; ++i) {
        const int64_t rb = min(r0 + 64 * i, rows - 1);               // (uniform: a scalar base, 32-bit offsets)
        const uint32_t off = min(t, (uint32_t)min(rows - 1 - rb, (int64_t)63)) * (uint32_t)ld + c;
        const uint8_t* src = q + rb * ld + (int64_t)j * kScaleBlock;
        uint8_t* dst = lds + 1024 * (8 * i + wave);                  // the wave's; a lane's 16 bytes follow
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + off),
                                         (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
    }
}
// the same for a last step that ends inside the block: zeros past column k
__device__ __forceinline__ void stage_tail(const uint8_t* q, int64_t ld, int64_t rows, int64_t r0, int j, int k,
                                           uint8_t* lds) {
    const int t = threadIdx.x >> 3, c = j * kScaleBlock + 16 * ((threadIdx.x & 7) ^ (t >> 1 & 7));
#pragma unroll 1
    for (int i = 0; i < kTile / 64; ++i)
        *reinterpret_cast<vu32x4*>(lds + 16 * (512 * i + (int)threadIdx.x)) =
            load_q16(q + min(r0 + 64 * i + t, rows - 1) * ld, c, k);
}

// A barrier behind which every wave may read what any wave has staged: a wave's loads to LDS are vector-memory
// operations in flight, which the barrier alone does not wait for.
__device__ __forceinline__ void staged_barrier() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// a fragment from its lane's two pieces, `rows` rows below the first
__device__ __forceinline__ mi32x8 tile_frag(const uint8_t* lo_piece, const uint8_t* hi_piece, int rows) {
    const vu32x4 lo = *reinterpret_cast<const vu32x4*>(lo_piece + rows * kScaleBlock);
    const vu32x4 hi = *reinterpret_cast<const vu32x4*>(hi_piece + rows * kScaleBlock);
    return mi32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

template <typename TO, bool B_TILE>
__global__ __launch_bounds__(kTileThreads, 2) void k_mm_tile(MmArgs p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t tile_lds[];
    TileStage* st = reinterpret_cast<TileStage*>(tile_lds);   // [2]
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, i = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // neighbouring tiles to one XCD (workgroups go round the eight); within it bands of four tile rows,
    // column by column
    const uint32_t mt = (uint32_t)p.mt, nt = (uint32_t)p.nt, total = mt * nt, per = (total + 7) / 8;
    const uint32_t tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (tile >= total) return;
    const uint32_t band = tile / (4 * nt), in_band = tile - band * 4 * nt, rows_in = min(4u, mt - 4 * band);
    const uint32_t col = in_band / rows_in, row = 4 * band + in_band - col * rows_in;
    const int64_t m0 = (int64_t)__builtin_amdgcn_readfirstlane((int)row) * kTile;
    const int64_t n0 = (int64_t)__builtin_amdgcn_readfirstlane((int)col) * kTile;
    const int wm = (wave & 3) * 16 * kTileMI, wn = (wave >> 2) * 16 * kTileNI;
    const int full = p.k / kScaleBlock;   // whole blocks
    // a lane's pieces g and g + 4 of row i of its wave (16 rows further the permutation is the same)
    const int piece = 16 * (g ^ (i >> 1)), at_a = (wm + i) * kScaleBlock, at_b = (wn + i) * kScaleBlock;

    vf32x4 acc[kTileMI][kTileNI];
#pragma unroll
    for (int x = 0; x < kTileMI; ++x)
#pragma unroll
        for (int j = 0; j < kTileNI; ++j) acc[x][j] = vf32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // a thread's scale of a step: rows of a, then rows (or tiles) of b
    const bool of_b = tid >= kTile;
    const int64_t srow = of_b ? min(n0 + tid - kTile, p.n - 1) : min(m0 + tid, p.m - 1);
    const float* sp = of_b ? p.sb + (B_TILE ? srow / kScaleBlock : srow) * p.kb : p.sa + srow * p.kb;
    // a block that k ends inside comes first, so every step of the loop stages a whole one
    const int tail = p.kb - full;
    if (tail) {
        stage_tail(p.a, p.lda, p.m, m0, full, p.k, st[0].a);
        stage_tail(p.b, p.ldb, p.n, n0, full, p.k, st[0].b);
    } else {
        stage_rows(p.a, p.lda, p.m, m0, 0, st[0].a);
        stage_rows(p.b, p.ldb, p.n, n0, 0, st[0].b);
    }
    (of_b ? st[0].sb : st[0].sa)[tid & (kTile - 1)] = sp[tail ? full : 0];
    staged_barrier();
    for (int step = 0; step < p.kb; ++step) {
        const TileStage& s = st[step & 1];
        TileStage& next = st[step & 1 ^ 1];
        const int kb = step + 1 - tail;   // the next block
        const float scale = sp[min(kb, p.kb - 1)];
        if (step + 1 < p.kb) {
            stage_rows(p.a, p.lda, p.m, m0, kb, next.a);
            stage_rows(p.b, p.ldb, p.n, n0, kb, next.b);
        }
        Operand fa[kTileMI];
        float sa[kTileMI];
#pragma unroll
        for (int x = 0; x < kTileMI; ++x) {
            fa[x].set(tile_frag(s.a + at_a + piece, s.a + at_a + (piece ^ 64), 16 * x));
            sa[x] = s.sa[wm + 16 * x + i];
            if constexpr (B_TILE) sa[x] *= s.sb[wn];   // (the wave's 128 columns are one tile of b)
        }
        // (a column tile at a time: widened fragments leave no registers for more)
#pragma unroll
        for (int j = 0; j < kTileNI; ++j) {
            Operand fb;
            fb.set(tile_frag(s.b + at_b + piece, s.b + at_b + (piece ^ 64), 16 * j));
            vf32x4 sb = {0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (!B_TILE) sb = *reinterpret_cast<const vf32x4*>(&s.sb[wn + 16 * j + 4 * g]);
#pragma unroll
            for (int x = 0; x < kTileMI; ++x) {
                const vf32x4 d = Operand::product(fb, fa[x]);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    acc[x][j][r] = fmaf(B_TILE ? sa[x] : sa[x] * sb[r], d[r], acc[x][j][r]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        // (also after the last step, where nobody reads it: a branch here would draw the sums behind it and
        // hold all 32 products in registers)
        (of_b ? next.sb : next.sa)[tid & (kTile - 1)] = scale;
        staged_barrier();
    }
#pragma unroll
    for (int j = 0; j < kTileNI; ++j) {
        const int64_t n = n0 + wn + 16 * j + 4 * g;
        const int valid = (int)min((int64_t)4, p.n - n);
        if (valid <= 0) continue;
        vf32x4 bias = {0.0f, 0.0f, 0.0f, 0.0f};
        if (p.bias)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (r < valid) bias[r] = p.bias[(n + r) * p.bias_step];
#pragma unroll
        for (int x = 0; x < kTileMI; ++x) {
            const int64_t m = m0 + wm + 16 * x + i;
            if (m < p.m) store_y4(static_cast<TO*>(p.y) + m * p.ldy + n, acc[x][j] + bias, valid);
        }
    }
}

// ----------------------------------------------------------------------------- rows of one block
//
// k <= 128, as the factors of the models here: the output's write is the work.  A wave keeps 32 rows of a in
// registers and goes along the columns, 128 bytes of each row of y at a time, the next columns' operand
// loaded meanwhile; the workgroup's four waves go along the same columns.  Products pass through a ring of
// two such pieces in LDS, placed by their address in y, so that every store writes whole, aligned lines of
// 128 bytes whatever the distance of the rows (8,192 x 27,278 fp32, rows 8 bytes off: 308 us with 16-byte stores
// at their own addresses, 215 so).
// Measured, 8,192 x 27,278 x 64: fp32 173 us (5.2 TB/s written), bf16 95-102; rows on their lines (27,264) 167 and 90.

constexpr int kShortRows = 32;
constexpr int kShortWaves = kBlock / 64;
constexpr int kLine = 128;

// A lane's part of a row of k <= 32 E values, 8 E of them: for E = 1 the 8 from column 8 g on, else 16 from
// column 16 g on of each 64.  Loads have no branch: a part that passes column k is read where the row's
// last values stand and shifted down when it is used (`past`: how many of its values the row has not).
template <int E>
struct ShortRaw {
    uint2 v[E];
    __device__ __forceinline__ static int past(int e, int g, int k) {
        return E == 1 ? 8 * g + 8 - max(k, 8) : 64 * (e / 2) + 16 * g + 16 - k;
    }
    __device__ __forceinline__ void load(const uint8_t* row, int g, int k) {
        if constexpr (E == 1) {
            typedef uint32_t u __attribute__((ext_vector_type(2), aligned(1)));
            if (k >= 8) {
                const u w = *reinterpret_cast<const u*>(row + min(8 * g, k - 8));
                v[0] = make_uint2(w[0], w[1]);
            } else {
                v[0] = make_uint2(0, 0);
                for (int c = 0; c < k; ++c) {
                    const uint32_t byte = (uint32_t)row[c] << (8 * (c & 3));
                    if (c < 4) v[0].x |= byte;
                    else v[0].y |= byte;
                }
            }
        } else {   // (k > 32)
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const vu32x4 w = load16(row + min(64 * (e / 2) + 16 * g, k - 16));
                v[e] = make_uint2(w[0], w[1]);
                v[e + 1] = make_uint2(w[2], w[3]);
            }
        }
    }
    // the part with zeros past column k
    __device__ __forceinline__ void settle(int g, int k) {
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const int n = max(past(e, g, k), 0);
            const uint64_t lo = (uint64_t)v[e].y << 32 | v[e].x;
            const uint64_t hi = E == 1 ? 0 : (uint64_t)v[E == 1 ? 0 : e + 1].y << 32 | v[E == 1 ? 0 : e + 1].x;
            const int bits = 8 * (n & 7);
            // whole halves first, then bytes
            const uint64_t l = n >= 16 ? 0 : n >= 8 ? hi : lo, h = n >= 8 ? 0 : hi;
            const uint64_t rl = bits ? l >> bits | h << (64 - bits) : l, rh = h >> bits;
            v[e] = make_uint2((uint32_t)rl, (uint32_t)(rl >> 32));
            if constexpr (E > 1) v[e + 1] = make_uint2((uint32_t)rh, (uint32_t)(rh >> 32));
        }
    }
};
template <int E>
struct ShortOperand {
    mf16x8 v[E];
    template <bool EXACT>
    __device__ __forceinline__ void set(ShortRaw<E> raw, int g, int k) {
        if constexpr (!EXACT) raw.settle(g, k);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const mi32x8 f = {(int)raw.v[e].x, (int)raw.v[e].y, 0, 0, 0, 0, 0, 0};
            v[e] = widen(f, 0);
        }
    }
    __device__ __forceinline__ static vf32x4 product(const ShortOperand& a, const ShortOperand& b) {
        vf32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < E; ++e) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[e], b.v[e], d, 0, 0, 0);
        return d;
    }
};

// four neighbouring outputs to their places in a row's ring, G of them at a time
template <typename TO, int G>
__device__ __forceinline__ void ring_put(uint8_t* ring, int col, vf32x4 y) {
    constexpr int S = (int)sizeof(TO), M = 2 * kLine - 1;
    typedef TO og __attribute__((ext_vector_type(G)));
#pragma unroll
    for (int e = 0; e < 4; e += G) {
        og v;
#pragma unroll
        for (int f = 0; f < G; ++f) v[f] = (TO)y[e + f];
        *reinterpret_cast<og*>(ring + ((col + e) * S & M)) = v;
    }
}

constexpr int kShortCols = 512;   // most columns of a workgroup (four workgroups a CU in LDS)

// EXACT: k = 32 E, no part passes a row's end
template <int E, typename TO, bool EXACT>
__global__ __launch_bounds__(kBlock, 4) void k_mm_short(MmArgs p, int cols, int unit) {
    constexpr bool OwnLoop = sizeof(TO) == 2 && E < 4;   // (below)
    constexpr int S = (int)sizeof(TO), C = kLine / S;      // columns of a line
    constexpr int NX = kShortRows / 16, NJ = 2, Step = 16 * NJ;   // columns of a step: a line takes C / Step
    constexpr int kPitch = 2 * kLine + 16;
    __shared__ __attribute__((aligned(16))) uint8_t rings[kShortWaves][kShortRows * kPitch];
    __shared__ __attribute__((aligned(16))) float col_scale[kShortCols + C], col_bias[kShortCols + C];
    const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    // Parts of the same rows follow each other on one XCD: its writes stay close to each other, and its L2 holds
    // the rows' operand (parts spread over the XCDs, rows first: 8,192 x 27,278 x 64 fp32 197 us)
    const uint32_t parts = (uint32_t)((p.n + cols - 1) / cols), total = parts * (uint32_t)p.mt;
    const uint32_t at = (blockIdx.x & 7) * ((total + 7) / 8) + (blockIdx.x >> 3);
    if (at >= total) return;
    const int64_t m0 = ((int64_t)(at / parts) * kShortWaves + wave) * kShortRows;
    const int64_t part = at % parts;
    const bool last = (part + 1) * cols >= p.n;
    // Columns of this workgroup, from c0 on.  Where rows do not start on a line it writes the lines that start
    // up to C columns ahead of its own part, and forms those columns too: only a row's ends are written in
    // parts of lines (8,192 x 27,278 fp32: a part's ends written so by both its sides took 215 us).
    const int lead = unit < kLine && part > 0 ? C : 0;
    const int64_t c0 = part * cols - lead;
    const int width = (int)min((int64_t)cols + lead, p.n - c0);
    for (int c = threadIdx.x; c < width; c += kBlock) {
        const int64_t n = c0 + c;
        col_scale[c] = p.sb[p.b_tile ? n / kScaleBlock : n];
        col_bias[c] = p.bias ? p.bias[n * p.bias_step] : 0.0f;
    }
    __syncthreads();
    if (m0 >= p.m) return;
    uint8_t* ring = rings[wave];
    // columns (of C) that y[m][c0] lies behind the start of its line
    auto off_of = [&](int64_t m) {
        return (int)(((uint64_t)(uintptr_t)p.y / S + (uint64_t)(m * p.ldy + c0)) & (C - 1));
    };
    ShortOperand<E> fa[NX];
    float sa[NX];
    int put[NX];        // the lane's place in a ring for its row and its columns
#pragma unroll
    for (int x = 0; x < NX; ++x) {
        const int64_t m = min(m0 + 16 * x + i, p.m - 1);
        ShortRaw<E> raw;
        raw.load(p.a + m * p.lda, g, p.k);
        fa[x].template set<EXACT>(raw, g, p.k);
        sa[x] = p.sa[m];
        put[x] = off_of(m) + 4 * g;
    }
    // the lane's stores: 16 bytes l % 8 of lines of rows l / 8 + 8 q
    constexpr int NQ = kShortRows / 8, P = 16 / S;
    const int piece = lane & 7;
    TO* to[NQ];         // where the lane's piece of the first line lies
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const int64_t m = min(m0 + 8 * q + (lane >> 3), p.m - 1);
        to[q] = static_cast<TO*>(p.y) + m * p.ldy + c0 + P * piece - off_of(m);
    }
    const uint8_t* b = p.b + c0 * p.ldb;
    ShortRaw<E> raw[NJ];
    auto load_b = [&](int n) {   // columns n .. n + Step
#pragma unroll
        for (int j = 0; j < NJ; ++j) raw[j].load(b + (int64_t)min(n + 16 * j + i, width - 1) * p.ldb, g, p.k);
    };
    load_b(0);
    // after the columns from n on are in the ring the line that starts n - off is whole
    auto form = [&](int n, auto ragged) {
#pragma unroll
        for (int h = n; h < n + C; h += Step) {
            if (decltype(ragged)::value && h >= width) continue;
            ShortOperand<E> fb[NJ];
            vf32x4 y[NJ][NX];
#pragma unroll
            for (int j = 0; j < NJ; ++j) fb[j].template set<EXACT>(raw[j], g, p.k);
            load_b(min(h + Step, width - 1));
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const vf32x4 sb = *reinterpret_cast<const vf32x4*>(&col_scale[h + 16 * j + 4 * g]);
                const vf32x4 bias = *reinterpret_cast<const vf32x4*>(&col_bias[h + 16 * j + 4 * g]);
#pragma unroll
                for (int x = 0; x < NX; ++x) {
                    const vf32x4 d = ShortOperand<E>::product(fb[j], fa[x]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[j][x][r] = fmaf(sa[x] * sb[r], d[r], bias[r]);
                }
            }
            auto put_all = [&](auto group) {
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int x = 0; x < NX; ++x)
                        ring_put<TO, decltype(group)::value>(ring + (16 * x + i) * kPitch, h + 16 * j + put[x],
                                                             y[j][x]);
            };
            if (unit >= 4 * S) put_all(std::integral_constant<int, 4>());
            else if (unit >= 2 * S) put_all(std::integral_constant<int, 2>());
            else put_all(std::integral_constant<int, 1>());
        }
        asm volatile("" ::: "memory");   // (the wave's own LDS, written and read in order)
    };
    auto store_lines = [&](int n) {
#pragma unroll
        for (int q = 0; q < NQ; ++q)
            *reinterpret_cast<vu32x4*>(to[q] + n) = *reinterpret_cast<const vu32x4*>(
                ring + (8 * q + (lane >> 3)) * kPitch + ((n * S + 16 * piece) & (2 * kLine - 1)));
        asm volatile("" ::: "memory");
    };
    // Turns from `whole` on to `rest` write whole lines of whole tiles of rows.  For 16-bit outputs and k <= 64 they
    // have a loop without a branch around its stores: those and the next columns' loads are then counted together,
    // and a turn does not wait for the stores of the one before (8,192 x 27,278 bf16, k = 64: 101 us, so 106; k = 32:
    // 92 and 97; fp16 97 and 100, 92 and 101).  With k = 128 its registers spill (151, so 143).  fp32 outputs write
    // twice as much, and waiting keeps the operands' loads from queueing behind their stores (in that loop
    // 8,192 x 27,278 x 128 took 206-212 us, so 202; with k = 64 180, so 182).
    const int whole = unit < kLine ? C : 0;
    const int rest = m0 + kShortRows <= p.m && width >= whole + C ? width / C * C : whole;
    const int end = width + (last ? C : 0);   // at a row's end a last turn without columns writes what is left
    for (int n = 0; n < end;) {
        if (OwnLoop && n == whole && rest > whole) {
            __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): nothing from before the loop counts in it
#pragma unroll 1
            for (; n < rest; n += C) {
                form(n, std::false_type());
                store_lines(n);
            }
            continue;
        }
        form(n, std::true_type());
        if (!OwnLoop && n >= whole && n < rest) {
            store_lines(n);
        } else if (n >= lead) {
#pragma unroll 1
            for (int q = 0; q < NQ; ++q) {
                const int row = 8 * q + (lane >> 3);
                if (m0 + row >= p.m) break;
                const int c = n + P * piece - off_of(m0 + row);
                TO* y = static_cast<TO*>(p.y) + (m0 + row) * p.ldy + c0;
                const TO* from = reinterpret_cast<const TO*>(ring + row * kPitch +
                                                             ((n * S + 16 * piece) & (2 * kLine - 1)));
                for (int e = 0; e < P; ++e)
                    if (c + e >= 0 && c + e < width) y[c + e] = from[e];
            }
        }
        asm volatile("" ::: "memory");
        n += C;
    }
}

template <int E, typename TO>
static void mm_short(MmArgs p, hipStream_t st) {
    constexpr int C = kLine / (int)sizeof(TO);
    constexpr int64_t rows = kShortWaves * kShortRows;
    p.mt = (p.m + rows - 1) / rows;
    // Columns of a workgroup: whole lines, about 2,048 workgroups together.  At least four lines (two and eight:
    // 2,000 x 3,706 x 128 bf16 15.8 and 21 us, so 13.6) and at most eight, or for k > 64 as many as LDS holds
    // scales for (8,192 x 27,278 fp32 at most eight and sixteen: k = 64 175 and 182 us, k = 128 210 and 202).
    const int64_t lines = (p.n + C - 1) / C;
    constexpr int64_t least = 4, most = E == 4 ? kShortCols / C : 8;
    const int64_t split = std::max<int64_t>(1, std::min<int64_t>((lines + least - 1) / least, 2048 / p.mt));
    const int64_t cols = std::min<int64_t>((lines + split - 1) / split, most) * C;
    const int64_t grid = (p.mt * ((p.n + cols - 1) / cols) + 7) / 8 * 8;
    // the largest power of two, up to a line, that divides every row's distance from a line's start
    const uint64_t bytes = (uint64_t)(uintptr_t)p.y | (p.m > 1 ? (uint64_t)p.ldy * sizeof(TO) : 0);
    const int unit = (int)std::min<uint64_t>(bytes & (0 - bytes), kLine);
    if (p.k == 32 * E) launch(k_mm_short<E, TO, true>, dim3((unsigned)grid), kBlock, 0, st, p, (int)cols, unit);
    else launch(k_mm_short<E, TO, false>, dim3((unsigned)grid), kBlock, 0, st, p, (int)cols, unit);
}

template <int MI, int NI, typename TO>
static void mm_direct(MmArgs p, hipStream_t st) {
    p.mt = (p.m + 16 * MI - 1) / (16 * MI);
    p.nt = (p.n + 16 * NI - 1) / (16 * NI);
    launch(k_mm_direct<MI, NI, TO>, dim3((unsigned)((p.mt * p.nt + 3) / 4)), kBlock, 0, st, p);
}

template <typename TO, bool B_TILE>
static hipError_t mm_tile(MmArgs p, hipStream_t st) {
    constexpr size_t lds = 2 * sizeof(TileStage);
    static std::atomic<uint64_t> allowed{0};   // devices on which the kernel may use this much LDS
    int dev = 0;
    if (hipError_t e = hipGetDevice(&dev)) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(allowed.load(std::memory_order_relaxed) & bit)) {
        if (hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k_mm_tile<TO, B_TILE>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds))
            return e;
        allowed.fetch_or(bit, std::memory_order_relaxed);
    }
    p.mt = (p.m + kTile - 1) / kTile;
    p.nt = (p.n + kTile - 1) / kTile;
    const int64_t per = (p.mt * p.nt + 7) / 8;
    launch(k_mm_tile<TO, B_TILE>, dim3((unsigned)(8 * per)), kTileThreads, lds, st, p);
    return hipGetLastError();
}

// Which kernel, and both sides of each choice (us); k_mm_tile also needs rows that start at multiples of 16 bytes (as
// quantize_blocks lays them out; 4,096 x 4,096 x 1,000 fp32 61, at 1,000 bytes a row 132 by k_mm_direct, 8,192 x 4,096 x
// 4,095 309 and 2,065):
//   more than 64 tiles of 256 x 256, k > 128: k_mm_tile (2,304 x 2,304 x 1,024, 81 tiles: fp32 45, so 58 by k_mm_direct;
//     2,048 x 2,048, 64 tiles: 44, so 29; 4,096 x 4,096 x 144: 22, so 24)
//   k <= 128 and 1,024 waves of 64 x 64: k_mm_short (4,096 x 4,096 x 64 fp32 15, so 36; 2,048 x 1,682: both 10.5)
//   up to 16 rows: a tile a wave (8 x 4,096 x 4,096: 18, with 2 x 2 tiles 34, 4 x 4 70)
//   1,024 waves of 64 x 64: 4 x 4 tiles a wave, else 2 x 2 (2,000 x 2,000 x 256 fp32 14 and 16.5;
//     333 x 1,682 x 200 19 and 10.5)
template <typename TO>
static hipError_t mm_t(const MmArgs& p, hipStream_t st) {
    const bool aligned = ((uintptr_t)p.a | (uintptr_t)p.b | (uint64_t)p.lda | (uint64_t)p.ldb) % 16 == 0;
    // (rows up to 16 MB apart: a thread's offsets in 32 bits)
    const bool near = p.lda <= 1 << 24 && p.ldb <= 1 << 24;
    if (aligned && near && p.k > kScaleBlock && ((p.m + kTile - 1) / kTile) * ((p.n + kTile - 1) / kTile) > 64)
        return p.b_tile ? mm_tile<TO, true>(p, st) : mm_tile<TO, false>(p, st);
    const int64_t waves = ((p.m + 63) / 64) * ((p.n + 63) / 64);   // of 64 x 64
    if (p.k <= kScaleBlock && waves >= 1024) {
        if (p.k > 64) mm_short<4, TO>(p, st);
        else if (p.k > 32) mm_short<2, TO>(p, st);
        else mm_short<1, TO>(p, st);
    } else if (p.m <= 16) mm_direct<1, 1, TO>(p, st);
    else if (waves >= 1024) mm_direct<4, 4, TO>(p, st);
    else mm_direct<2, 2, TO>(p, st);
    return hipGetLastError();
}

hipError_t launch_matmul_blocks(const uint8_t* a, int64_t lda, const float* sa, const uint8_t* b, int64_t ldb,
                                const float* sb, int b_tile, const float* bias, int bias_step, int64_t m, int64_t n,
                                int k, int out_dtype, void* y, int64_t ldy, hipStream_t st) {
    if (m <= 0 || n <= 0) return hipSuccess;
    const int kb = (k + kScaleBlock - 1) / kScaleBlock, size = out_dtype == NCF_F32 ? 4 : 2;
    // (HIP counts a launch's threads in 32 bits: 2^29 columns by tiles of 16 a wave are 2^31)
    constexpr int64_t most = (int64_t)1 << 29;
    for (int64_t c = 0; c < n; c += most) {
        MmArgs p{a, b + c * ldb, sa, sb + (b_tile ? c / kScaleBlock : c) * kb, bias ? bias + c * bias_step : nullptr,
                 static_cast<char*>(y) + c * size, lda, ldb, ldy, m, std::min(n - c, most), k, kb, b_tile, bias_step, 0, 0};
        hipError_t e = out_dtype == NCF_F32 ? mm_t<float>(p, st)
                       : out_dtype == NCF_BF16 ? mm_t<__bf16>(p, st) : mm_t<_Float16>(p, st);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// ----------------------------------------------------------------------------- GMF-only models
//
// z(u, i) = sum_f w_f e_u,f e_i,f + b (movierec/model.py:184-188 without hidden layers): the factors of the
// users, times w, against the table's item rows.

__global__ __launch_bounds__(kBlock) void k_gmf_users(const float* __restrict__ emb, const float* __restrict__ w,
                                                      const int32_t* __restrict__ users, int64_t n, int num_users,
                                                      int width, int dim, float* __restrict__ out) {
    const int64_t x = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (x >= n * dim) return;
    const int64_t q = x / dim;
    const int f = (int)(x - q * dim), u = users[q];
    out[x] = u >= 0 && u < num_users ? w[f] * emb[(int64_t)u * width + f] : __int_as_float(0x7fc00000);
}

GmfLayout gmf_layout(const ncf_shape_t& s, int64_t n) {
    GmfLayout l{};
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t at = off;
        off = (off + bytes + 255) / 256 * 256;
        return at;
    };
    const int64_t kb = (s.gmf_dim + kScaleBlock - 1) / kScaleBlock;
    l.q_ld = (s.gmf_dim + 15) / 16 * 16;
    l.uf = take((size_t)n * s.gmf_dim * 4);
    l.uq = take((size_t)n * l.q_ld);
    l.us = take((size_t)n * kb * 4);
    l.iq = take((size_t)s.num_items * l.q_ld);
    l.is = take((size_t)s.num_items * kb * 4);
    l.total = off;
    return l;
}

hipError_t launch_gmf_logits(const ncf_shape_t& s, void* ws, const float* emb, const float* mlp, const int32_t* users,
                             int64_t n, float* logits, hipStream_t st) {
    const GmfLayout l = gmf_layout(s, n);
    const int dim = s.gmf_dim;
    float* uf = at<float>(ws, l.uf);
    const float* w = mlp + s.layer_off[0];
    launch(k_gmf_users, dim3((unsigned)((n * dim + kBlock - 1) / kBlock)), kBlock, 0, st, emb, w, users, n, s.num_users,
           s.row_width, dim, uf);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess)
        e = launch_quantize(uf, NCF_F32, n, dim, dim, 0, at<uint8_t>(ws, l.uq), l.q_ld, at<float>(ws, l.us), st);
    if (e == hipSuccess)
        e = launch_quantize(emb + (int64_t)s.num_users * s.row_width, NCF_F32, s.num_items, dim, s.row_width, 0,
                            at<uint8_t>(ws, l.iq), l.q_ld, at<float>(ws, l.is), st);
    if (e == hipSuccess)
        e = launch_matmul_blocks(at<uint8_t>(ws, l.uq), l.q_ld, at<float>(ws, l.us), at<uint8_t>(ws, l.iq), l.q_ld,
                                 at<float>(ws, l.is), 0, w + s.out_features, 0, n, s.num_items, dim, NCF_F32, logits,
                                 s.num_items, st);
    return e;
}

// The same in fp32, z = sum_f (e_u,f e_i,f) w_f + b with the fp32 forward's roundings in its order: the same bits as a
// pair's.  A workgroup forms 64 users by 64 items, a thread 4 by 4; both sides go through LDS 16
// values of a row at a time.  2,048 users x 27,278 items, 64 values: 300 us (a pair a thread: 54.7 ms, each
// with its factors from memory and its products written to the activations).
constexpr int kGmfTile = 64, kGmfStep = 16;

__global__ __launch_bounds__(kBlock) void k_gmf_logits(const float* __restrict__ emb, const float* __restrict__ wo,
                                                       const int32_t* __restrict__ users, int64_t n, int num_users,
                                                       int num_items, int width, int dim, int item_tiles,
                                                       float* __restrict__ logits) {
    __shared__ __attribute__((aligned(16))) float su[kGmfStep][kGmfTile + 4], si[kGmfStep][kGmfTile + 4];
    __shared__ float sw[kGmfStep];
    const int64_t q0 = (int64_t)(blockIdx.x / item_tiles) * kGmfTile;
    const int i0 = (int)(blockIdx.x % item_tiles) * kGmfTile;
    const int tu = 4 * ((int)threadIdx.x >> 4), ti = 4 * ((int)threadIdx.x & 15);
    // a thread's part of the staging: four values of one user's row and of one item's
    const int sr = (int)threadIdx.x >> 2, sf = 4 * ((int)threadIdx.x & 3);
    const int u = users[min(q0 + sr, n - 1)];
    const float* pu = emb + (int64_t)(u >= 0 && u < num_users ? u : 0) * width;
    const float* pi = emb + ((int64_t)num_users + min(i0 + sr, num_items - 1)) * width;
    float z[4][4] = {};
    for (int f0 = 0; f0 < dim; f0 += kGmfStep) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool in = f0 + sf + e < dim;
            su[sf + e][sr] = in ? pu[f0 + sf + e] : 0.0f;
            si[sf + e][sr] = in ? pi[f0 + sf + e] : 0.0f;
        }
        if (threadIdx.x < kGmfStep) sw[threadIdx.x] = f0 + (int)threadIdx.x < dim ? wo[f0 + threadIdx.x] : 0.0f;
        __syncthreads();
        const int steps = min(kGmfStep, dim - f0);   // (a sum of zeros beyond dim would turn -0 into 0)
        for (int f = 0; f < steps; ++f) {
            const float4 a = *reinterpret_cast<const float4*>(&su[f][tu]);
            const float4 b = *reinterpret_cast<const float4*>(&si[f][ti]);
            const float x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w}, w = sw[f];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < 4; ++c) z[r][c] = fmaf(x[r] * y[c], w, z[r][c]);
        }
    }
    const float bias = wo[dim];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int64_t q = q0 + tu + r;
        if (q >= n) break;
        const int id = users[q];
        const bool known = id >= 0 && id < num_users;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (i0 + ti + c < num_items)
                logits[q * num_items + i0 + ti + c] = known ? z[r][c] + bias : __int_as_float(0x7fc00000);
    }
}

hipError_t launch_gmf_logits_fp32(const ncf_shape_t& s, const float* emb, const float* mlp, const int32_t* users,
                                  int64_t n, float* logits, hipStream_t st) {
    const int item_tiles = (s.num_items + kGmfTile - 1) / kGmfTile;
    const int64_t grid = (n + kGmfTile - 1) / kGmfTile * item_tiles;
    launch(k_gmf_logits, dim3((unsigned)grid), kBlock, 0, st, emb, mlp + s.layer_off[0], users, n, s.num_users,
           s.num_items, s.row_width, s.gmf_dim, item_tiles, logits);
    return hipGetLastError();
}

}  // namespace ncf

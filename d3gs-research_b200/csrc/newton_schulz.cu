// Orthogonalised updates of weight matrices by Newton-Schulz products, and the optimizer step around them.
//
//   U = the update (given, or momentum buffer and gradient joined), X = U / max(|U|_F, eps), the short side first
//   each step: A = X X^T,  B = a I + b A + c A A,  X <- B X
//   result X, or param <- decay param - rate X
//
// B - a I is one product: with V = A + b/c I it is c A V, so that nothing but products and a shifted diagonal is needed.
// V is A but for the blocks on its diagonal, which are kept twice.  (c = 0: B = a I + b A, and no second product.)
// Shifting both factors, c S S with S = A + b/(2c) I, would need no second blocks, but its sums are of size one where
// b A + c A A is small, and lost twice the accuracy of 32-bit matrices up to 256 x 256.
//
// All matrices of a call go through the same launches: a table in the kernel arguments maps CTAs to matrices.
//
// The products run on the tensor cores (tcgen05, 32-bit sums in TMEM).  Their operands are fp16 with a power-of-two
// scale: X, A and B have bounded spectra (the bounds follow from the coefficients), so the 2^29 of fp16's normal range
// hold every entry that matters.  One fp16 value keeps 11 bits, two of them, v = hi + lo, keep 22.
//  * 32-bit matrices: all operands hi + lo, three products hi hi + hi lo + lo hi; the dropped lo lo is of the size of
//    the last bit.  (Two bf16 values would hold 16 bits only, and three of them need six products.)
//  * 16-bit matrices (large ones, see Batch): A, B and V one value, X two of which A sees the first: A = Xhi Xhi^T, B X =
//    B Xhi + B Xlo.  What A and B lose turns X's singular directions by that much and no more.  What X loses is noise in all
//    directions alike, and the next steps amplify it where X is small: with one value a result is 2.8e-3 off at 512 x 512
//    and 5.1e-3 at 4096 x 4096 before its own rounding to bfloat16, which is 1.65e-3; with two, measured, 0.7e-3 at 2048 x
//    512, 0.8e-3 at 512 x 512, 1.2e-3 at 2048 x 2048, 1.4e-3 at 4096 x 4096 (gradients with a few strong directions) and up
//    to 1.5e-3 (a quarter of full rank).  The same roundings done in 64 bits give these figures within 7 %; a third is that
//    of V's diagonal, a value near b / c, behind which A V is no longer symmetric though one triangle stands for both.
//    (Operands like those of 32-bit matrices would leave the output's rounding alone, for three products where there are
//    now one or two.)  The last step amplifies little: there X is one value.  So it is in the first one, where U times a
//    power of two is exact (8 bits) and what is left of 1 / |U| goes into the scales.
//
// Working matrices are stored as the products read them: blocks of 128 rows x 64 columns, each the image of one shared
// memory tile (128-byte rows, 16-byte pieces exchanged within groups of eight rows), hi and lo one after the other, zero
// where the matrix ends.  A tile is then one contiguous bulk copy, odd sizes need no care outside the first and the last
// pass, and no tensor maps are made.  X serves both as rows of the Gram matrix (its columns are summed over) and as the
// right factor of B X (its rows are summed over) from this one layout.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "common.cuh"

namespace d3gs {
namespace {

constexpr int kMaxMatrices = 32;   // per launch, a table of less than 4 KB; longer lists are cut
constexpr int kThreads = 256;
constexpr int kPieces = 1024;       // pieces of eight neighbouring columns that a CTA of the norm pass takes at a time
constexpr int kMaxNorms = 4096;     // sums of squares of a matrix: every CTA of the first pass adds them up
constexpr int kMaxShort = 16384, kMaxLong = 1 << 24;
constexpr int kRows = 128, kCols = 64;                 // one block
constexpr uint32_t kPlane = kRows * kCols * 2;         // bytes of one fp16 plane of a block
constexpr int kTickets = 148;                          // of shared tiles: one for every CTA at most
constexpr size_t kSumBytes = 128 * 256 * 4;            // of a CTA of a shared tile
constexpr float kMaxSpectrum = 1024.0f;                // largest singular value the scales leave room for

struct Matrix {
    const void* src;
    float* momentum;
    void* dst;
    int64_t src_stride;   // values between rows
    char *x[2], *a, *b;   // blocks of X (two buffers), A, B
    char* v;              // V's blocks on the diagonal: two for each block of rows
    double* norms;        // sums of squares of the norm pass; before them, as a float, the factor that `exact` leaves out
    int32_t rows, cols;
    int32_t m;            // short side
    int32_t mb, mk, nk;   // blocks: rows of all three, columns of A and B, columns of X
    int32_t rounds, sums; // of the norm pass: how many times kPieces a CTA takes; sums of squares that gives
    float rate;
};
struct Table {
    Matrix mat[kMaxMatrices];
    int32_t first_block[kMaxMatrices + 1];
    int32_t count;
    int32_t bf16;         // src and dst type (momentum and parameters are always 32 bits)
    float eps, decay;
    float mu, fresh;      // weights of the old buffer and of the gradient; fresh is 1 - mu, rounded once
    int32_t nesterov;
    int32_t from;         // which of x[] holds X
    float out_scale;      // of a product's result; of X in the first and the last pass
    float shift;          // added on the diagonal of V or B
    int32_t cubic;        // c = 0: the first product gives B
    int32_t exact;        // X is U times a power of two, as one value (first pass and first step of large 16-bit matrices)
    uint32_t* fail;       // set when a bounded wait ran out: the last pass then writes NaN
    int32_t parts;        // how many pairs of CTAs share the sum of a tile
    uint32_t* tickets;    // how many of them have put their sums down: for both halves of every tile, zero between products
    float4* sums;         // those sums
    TestHooks hooks;
};

// Launches follow one another closely: a kernel may start while its predecessor's last CTAs run, and waits here before
// it touches memory.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// the matrix a CTA belongs to, and its number within it
__device__ __forceinline__ int find_matrix(const Table& t, int id, int& block) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (id >= t.first_block[mid]) lo = mid;
        else hi = mid - 1;
    }
    block = id - t.first_block[lo];
    return lo;
}

// the update from gradient and NEW momentum
__device__ __forceinline__ float update_of(const Table& t, float g, float buf) {
    return t.nesterov ? fmaf(t.mu, buf, t.fresh * g) : buf;
}

// Eight neighbouring columns of a row of U, of which `n` exist; where rows are so aligned, as vectors.
struct Access {
    bool src, state;   // gradient or update; momentum and parameter
};
__device__ __forceinline__ Access access_of(const Table& t, const Matrix& m) {
    Access a;
    a.src = ((uintptr_t)m.src & 15) == 0 && m.src_stride % (t.bf16 ? 8 : 4) == 0;
    a.state = (((uintptr_t)m.momentum | (uintptr_t)m.dst) & 15) == 0 && m.cols % (t.bf16 ? 8 : 4) == 0;
    return a;
}
__device__ __forceinline__ void load8(const float* p, bool vector, int n, float (&v)[8]) {
    if (vector && n == 8) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.0f;
    }
}
__device__ __forceinline__ void store8(float* p, bool vector, int n, const float (&v)[8]) {
    if (vector && n == 8) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = v[i];
    }
}
__device__ __forceinline__ void load_src8(const Table& t, const Matrix& m, int64_t at, bool vector, int n, float (&v)[8]) {
    if (!t.bf16) return load8(static_cast<const float*>(m.src) + at, vector, n, v);
    const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(m.src) + at;
    if (vector && n == 8) {
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(q[i] << 16);
            v[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? __bfloat162float(p[i]) : 0.0f;
    }
}

// ---- new momentum, and the sum of squares of the update (in 64 bits: no value of a float overflows it) -----------
// TURNS: a CTA may take several times kPieces.  (An instance of its own: the loop makes 8 x 2048 x 512 in 16 bits 17 us, not 13.)
template <bool TURNS> __global__ void __launch_bounds__(kThreads) ns_norm_kernel(const __grid_constant__ Table t) {
    __shared__ double s[kThreads / 32];
    int block;
    const Matrix& m = t.mat[find_matrix(t, (int)blockIdx.x, block)];
    const unsigned per_row = (m.cols + 7) / 8, pieces = m.rows * per_row;
    const Access access = access_of(t, m);
    let_next_start();
    wait_for_previous();
    if (blockIdx.x == 0 && threadIdx.x == 0) *t.fail = 0;
    if (blockIdx.x == 0 && threadIdx.x < kTickets) t.tickets[threadIdx.x] = 0;
    double sum = 0.0;
    const int rounds = TURNS ? m.rounds : 1;
    for (int round = 0; round < rounds; ++round) {
        const unsigned first = ((unsigned)block * rounds + round) * kPieces;
        float u[kPieces / kThreads][8], buf[kPieces / kThreads][8];
#pragma unroll
        for (int k = 0; k < kPieces / kThreads; ++k) {
            const unsigned i = first + k * kThreads + threadIdx.x;
            const int r = i / per_row, c = (i - r * per_row) * 8, n = i < pieces ? min(8, m.cols - c) : 0;
            load_src8(t, m, n ? r * m.src_stride + c : 0, access.src, n, u[k]);
            if (m.momentum) load8(m.momentum + (n ? (int64_t)r * m.cols + c : 0), access.state, n, buf[k]);
        }
#pragma unroll
        for (int k = 0; k < kPieces / kThreads; ++k) {
            if (m.momentum) {
                const unsigned i = first + k * kThreads + threadIdx.x;
                const int r = i / per_row, c = (i - r * per_row) * 8, n = i < pieces ? min(8, m.cols - c) : 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    buf[k][j] = fmaf(t.mu, buf[k][j], t.fresh * u[k][j]);
                    u[k][j] = update_of(t, u[k][j], buf[k][j]);
                }
                store8(m.momentum + (n ? (int64_t)r * m.cols + c : 0), access.state, n, buf[k]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += (double)u[k][j] * (double)u[k][j];
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < kThreads / 32; ++k) sum += s[k];
        m.norms[block] = sum;
    }
}

// What turns U into X: first / max(|U|, eps) as the product of two floats, since one alone does not hold it at the ends of
// the range (a norm above 2^126, or one below 2^-114 with an eps as small).  A power of two goes onto U first; it is one
// in between.  With both finite, zeros stay zeros whatever eps is.
struct Factor {
    float power, rest;
    __device__ __forceinline__ float operator()(float u) const { return u * power * rest; }
};
__device__ __forceinline__ Factor factor_of(double sum_of_squares, float eps, float first) {
    const double norm = sqrt(sum_of_squares), f = 1.0 / (norm < (double)eps ? (double)eps : norm) * first;   // a NaN stays one
    Factor r;
    r.power = f > 0x1p100 ? 0x1p100f : f < 0x1p-100 ? 0x1p-100f : 1.0f;
    r.rest = (float)(f / (double)r.power);
    return r;
}

// every CTA adds the sums up itself, in the same order
__device__ __forceinline__ double sum_of_squares(const Matrix& m) {
    __shared__ double s[kThreads / 32];
    double sum = 0.0;
    for (int i = threadIdx.x; i < m.sums; i += kThreads) sum += m.norms[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = 0.0;
    for (int k = 0; k < kThreads / 32; ++k) sum += s[k];
    return sum;
}

// byte of value (r, c) in a plane of a block
__device__ __forceinline__ uint32_t block_offset(uint32_t r, uint32_t c) {
    return r * 128u + (((c >> 3) ^ (r & 7u)) << 4) + (c & 7u) * 2u;
}
// A pair of values v = hi + lo with 22 bits each, as pairs of fp16: hi, and what its rounding left.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// ---- first pass: blocks of X = U / norm, transposed when the matrix is tall; one CTA per block --------------------
// Pieces of eight columns of U.  As rows of X they go straight to their block, eight threads to a 128-byte line; as
// columns by way of shared memory.
__global__ void __launch_bounds__(kThreads) ns_load_kernel(const __grid_constant__ Table t) {
    __shared__ __align__(16) char s[2 * kPlane];
    int block;
    const Matrix& m = t.mat[find_matrix(t, (int)blockIdx.x, block)];
    const bool tall = m.rows > m.cols;
    const int r0 = block / m.nk * kRows, c0 = block % m.nk * kCols;
    const Access access = access_of(t, m);
    char* const out = m.x[0] + (int64_t)block * 2 * kPlane;
    let_next_start();
    wait_for_previous();
    Factor scale = factor_of(sum_of_squares(m), t.eps, t.out_scale);
    if (t.exact) {
        const uint32_t exponent = __float_as_uint(scale.rest) & 0x7f800000u;
        float rest = 1.0f;   // in [1, 2); factors without a power of two (zero, not finite) stay whole
        if (exponent != 0 && exponent != 0x7f800000u) {
            rest = scale.rest / __uint_as_float(exponent);
            scale.rest = __uint_as_float(exponent);
        }
        if (block == 0 && threadIdx.x == 0) *reinterpret_cast<float*>(m.norms - 1) = rest;
    }
#pragma unroll 2
    for (int i = threadIdx.x; i < kRows * kCols / 8; i += kThreads) {
        // row and column within the block's part of U
        const int r = tall ? i % kCols : i / (kCols / 8), c = (tall ? i / kCols : i % (kCols / 8)) * 8;
        const int ur = (tall ? c0 : r0) + r, uc = (tall ? r0 : c0) + c, n = ur < m.rows ? max(0, min(8, m.cols - uc)) : 0;
        float u[8], buf[8];
        load_src8(t, m, n ? ur * m.src_stride + uc : 0, access.src, n, u);
        if (m.momentum) {
            load8(m.momentum + (n ? (int64_t)ur * m.cols + uc : 0), access.state, n, buf);
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] = update_of(t, u[j], buf[j]);
        }
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) split2(scale(u[2 * j]), scale(u[2 * j + 1]), hi[j], lo[j]);
        if (!tall) {
            const uint32_t o = block_offset(r, c);
            *reinterpret_cast<uint4*>(out + o) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if (!t.exact) *reinterpret_cast<uint4*>(out + kPlane + o) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t o = block_offset(c + j, r);
                *reinterpret_cast<uint16_t*>(s + o) = (uint16_t)(hi[j / 2] >> (16 * (j & 1)));
                *reinterpret_cast<uint16_t*>(s + kPlane + o) = (uint16_t)(lo[j / 2] >> (16 * (j & 1)));
            }
        }
    }
    if (!tall) return;
    __syncthreads();
    for (int i = threadIdx.x; i < (t.exact ? 1 : 2) * (int)kPlane / 16; i += kThreads)
        reinterpret_cast<uint4*>(out)[i] = reinterpret_cast<const uint4*>(s)[i];
}

// Eight neighbouring values of the result: stored, or taken from the parameter.
__device__ __forceinline__ void write_result8(const Table& t, const Matrix& m, int64_t at, bool vector, int n, float (&v)[8], float scale,
                                              bool failed) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = failed ? __int_as_float(0x7fffffff) : v[j] * scale;
    if (m.momentum) {
        float p[8];
        load8(static_cast<const float*>(m.dst) + at, vector, n, p);
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = fmaf(-m.rate, v[j], t.decay * p[j]);
        store8(static_cast<float*>(m.dst) + at, vector, n, p);
    } else if (!t.bf16) {
        store8(static_cast<float*>(m.dst) + at, vector, n, v);
    } else if (vector && n == 8) {
        uint4 w;
        __nv_bfloat162* const q = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(m.dst) + at) = w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) static_cast<__nv_bfloat16*>(m.dst)[at + j] = __float2bfloat16_rn(v[j]);
    }
}

// ---- last pass: result or parameter from the blocks of X; one CTA per block ---------------------------------------
__global__ void __launch_bounds__(kThreads) ns_store_kernel(const __grid_constant__ Table t) {
    int block;
    const Matrix& m = t.mat[find_matrix(t, (int)blockIdx.x, block)];
    const bool tall = m.rows > m.cols;
    const int r0 = block / m.nk * kRows, c0 = block % m.nk * kCols;
    const Access access = access_of(t, m);
    const char* const x = m.x[t.from] + (int64_t)block * 2 * kPlane;
    wait_for_previous();
    const bool failed = *t.fail != 0;
#pragma unroll 2
    for (int i = threadIdx.x; i < kRows * kCols / 8; i += kThreads) {
        const int r = tall ? i % kCols : i / (kCols / 8), c = (tall ? i / kCols : i % (kCols / 8)) * 8;
        const int ur = (tall ? c0 : r0) + r, uc = (tall ? r0 : c0) + c, n = ur < m.rows ? max(0, min(8, m.cols - uc)) : 0;
        if (n == 0) continue;
        float v[8];
        if (!tall) {
            const uint32_t o = block_offset(r, c);
            const uint4 h = *reinterpret_cast<const uint4*>(x + o), l = *reinterpret_cast<const uint4*>(x + kPlane + o);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 a = __half22float2(reinterpret_cast<const __half2*>(&h)[j]), b = __half22float2(reinterpret_cast<const __half2*>(&l)[j]);
                v[2 * j] = a.x + b.x;
                v[2 * j + 1] = a.y + b.y;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {   // (neighbouring threads read neighbouring columns of X)
                const uint32_t o = block_offset(c + j, r);
                v[j] = __half2float(*reinterpret_cast<const __half*>(x + o)) + __half2float(*reinterpret_cast<const __half*>(x + kPlane + o));
            }
        }
        write_result8(t, m, (int64_t)ur * m.cols + uc, access.state, n, v, t.out_scale, failed);
    }
}

// ---- tcgen05 ------------------------------------------------------------------------------------------------------
// CG: 1, or 2 where a pair of CTAs works on one tile
template <int CG> __device__ __forceinline__ void tmem_alloc(uint32_t* out, uint32_t cols) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(out)), "r"(cols) : "memory");
    else
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(out)), "r"(cols) : "memory");
}
template <int CG> __device__ __forceinline__ void tmem_free(uint32_t at, uint32_t cols) {
    if constexpr (CG == 2) {
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(cols));
    } else {
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(cols));
    }
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// arrives at the barrier (of both CTAs of a pair) when the products issued so far are done
template <int CG> __device__ __forceinline__ void tc_commit(uint64_t* bar) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                         smem_u32(bar)),
                     "h"((uint16_t)3)
                     : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
template <int CG> __device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    if constexpr (CG == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.u32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.u32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
            : "memory");
}
// 32 columns of this thread's TMEM lane
__device__ __forceinline__ void tmem_load32(uint32_t at, float (&v)[32]) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const float* v) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%"
        "17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// The same barrier in CTA `rank` of the cluster.  What it orders are tensor-core and bulk-copy accesses, never plain
// ones, so no cluster-wide release is asked for (the fence that it costs held the products of a pair up by a factor of
// two: 1.6 k cycles a column block of 512 cycles of products).
__device__ __forceinline__ void mbar_arrive_at(uint64_t* bar, uint32_t rank) {
    asm volatile(
        "{\n\t.reg .b32 a;\n\t"
        "mapa.shared::cluster.u32 a, %0, %1;\n\t"
        "mbarrier.arrive.shared::cluster.b64 _, [a];\n\t}" ::"r"(smem_u32(bar)),
        "r"(rank)
        : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
// four floats at the same place in CTA `rank` of the cluster
__device__ __forceinline__ float4 load_shared_of(uint32_t at, uint32_t rank) {
    float4 v;
    asm volatile(
        "{\n\t.reg .b32 a;\n\t"
        "mapa.shared::cluster.u32 a, %4, %5;\n\t"
        "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
        : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
        : "r"(at), "r"(rank)
        : "memory");
    return v;
}
// mbar_wait_bounded without its sleep: a wait here is a link of the chain that every column block goes through.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, uint32_t limit = 0) {
    const uint32_t polls = limit != 0 ? limit : (1u << 24);
    for (uint32_t it = 0; it < polls; ++it)
        if (mbar_try_wait(bar, parity)) return true;
    return false;
}

// A loading thread that has given up waits here until the copies number `from` to `to` - 1 have landed (number j in stage
// j % count of `full`): the CTA must not end, nor its shared memory become another's, before.  The limit is this wait's
// own, some 7 ms where a copy takes microseconds, and not the one that has just run out, which a test may have made short.
// (It can run out itself where a stage's barrier also counts the other CTA's word, and that one has given up as well: by
// then every copy has landed.)
__device__ __forceinline__ void drain(uint64_t* full, int count, int from, int to) {
    uint32_t left = 1u << 17;
    for (int j = from; j < to; ++j) {
        uint32_t landed = 0;
        while (landed == 0 && left-- != 0)
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                "selp.u32 %0, 1, 0, p;\n\t}"
                : "=r"(landed)
                : "r"(smem_u32(full + j % count)), "r"((uint32_t)(j / count) & 1u)
                : "memory");
        if (landed == 0) return;
    }
}
// What a test makes a CTA's loading thread withhold: everything (hold = the CTA's number), so that nothing of it is in
// flight when waits run out, or the first copy alone (hold = -2 - number), so that the others are.
__device__ __forceinline__ bool withholds_all(const Table& t) { return t.hooks.hold == (int)blockIdx.x; }
__device__ __forceinline__ bool withholds_first(const Table& t) { return t.hooks.hold == -2 - (int)blockIdx.x; }

// Shared-memory operand in 128-byte rows with the 16-byte pieces exchanged (swizzle mode 2).  Summed along the rows:
// eight rows are 1024 bytes apart, `next` is not used.  Summed across the rows: the next eight summed rows are 1024
// bytes apart, the next 64 columns `next`.  The low word holds the address: moving by n bytes adds n / 16 to it.
// In a cluster a CTA's own shared addresses carry its rank from bit 24 on (0x01000400 is 0x400 of CTA 1).  The address field
// has no place for it: shifted in as it is, it would add 256 bytes a rank to `next`, and products that sum across the rows
// would read past the end of shared memory.
constexpr uint32_t kSharedOffset = 0x3ffffu;
__host__ __device__ constexpr uint32_t operand_low(uint32_t at, uint32_t next) {
    return ((at & kSharedOffset) >> 4) | ((next >> 4) << 16);
}
static_assert(operand_low(0x07000400u, 8192) == operand_low(0x400u, 8192) && operand_low(0x400u, 8192) == (0x40u | 512u << 16),
              "an operand is addressed within its CTA, whatever the CTA's rank");
__device__ __forceinline__ uint64_t operand(uint32_t low) {
    return ((uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29)) << 32) | low;
}
// D 32 bits, A and B fp16; B X sums its right factor across the rows (bit 16)
__device__ __forceinline__ uint32_t instruction(bool across, uint32_t rows, uint32_t cols) {
    return (1u << 4) | ((across ? 1u : 0u) << 16) | ((cols / 8u) << 17) | ((rows / 16u) << 24);
}

// ---- products -----------------------------------------------------------------------------------------------------
// Roles of a CTA: one warp brings in operand tiles by bulk copies, one issues the products, the others take the sums
// out of TMEM and write the result's blocks.
//
// The tensor cores cut the last bits of a running sum at every addition (towards zero, so that the losses add up: 2e-5
// of the result at 1025 x 515 when nothing is done about it).  For 32-bit matrices the sums of hi hi are therefore taken
// out after every column block and added in registers (rounded).  That costs no time: hi lo + lo hi, 2^-11 of their
// size, go to a sum of their own, taken out once, and the tensor cores work on those meanwhile.
//
// A and B are symmetric: only tiles on and above the diagonal are computed, and written twice.  Rows behind the last
// column block of A and B hold anything: nothing sums over them, and no valid row or column reads them.
enum { kGram = 0, kSquare = 1, kApply = 2 };

// What the products of a mode of large matrices read: planes of the left and the right factor and of the result, and how
// many planes lie between blocks of A and B.  RIGHT is 1 in the first and the last step of 16-bit matrices.
template <bool F32, int MODE, int RIGHT> struct Planes {
    static constexpr int kLeft = F32 ? 2 : 1;
    static constexpr int kRight = RIGHT;
    static constexpr int kOut = F32 || MODE == kApply ? 2 : 1;
    static constexpr uint32_t kAB = (F32 ? 2 : 1) * kPlane, kX = 2 * kPlane;   // bytes of one block
};

// One 16-byte piece of a result: eight columns of a row, from sums to planes; `diagonal`: which of them takes the shift.
__device__ __forceinline__ void finish(const float* v, float scale, float shift, int diagonal, uint32_t* hi, uint32_t* lo) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = fmaf(v[i], scale, i == diagonal ? shift : 0.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) split2(f[2 * i], f[2 * i + 1], hi[i], lo[i]);
}
template <bool TWO> __device__ __forceinline__ void put(char* at, const uint32_t* hi, const uint32_t* lo) {
    *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if (TWO) *reinterpret_cast<uint4*>(at + kPlane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}
// Eight columns of this thread's row into the mirrored tile, where they are eight rows.  Neighbouring threads hold
// neighbouring columns there: they exchange values and write two at a time.  row0: the first of the eight rows, even.
template <bool TWO> __device__ __forceinline__ void write_mirrored(char* block, uint32_t row0, uint32_t col, const uint32_t* hi,
                                                                   const uint32_t* lo) {
    const bool odd = col & 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // rows row0 + 2 i and the next one
        const uint32_t o = block_offset(row0 + 2 * i + (odd ? 1 : 0), col & ~1u);
        // an even thread keeps its first value and takes the neighbour's first, an odd one the second ones
        const uint32_t h = __shfl_xor_sync(~0u, hi[i], 1);
        *reinterpret_cast<uint32_t*>(block + o) = odd ? __byte_perm(h, hi[i], 0x7632) : __byte_perm(hi[i], h, 0x5410);
        if (TWO) {
            const uint32_t l = __shfl_xor_sync(~0u, lo[i], 1);
            *reinterpret_cast<uint32_t*>(block + kPlane + o) = odd ? __byte_perm(l, lo[i], 0x7632) : __byte_perm(lo[i], l, 0x5410);
        }
    }
}

// ---- tiny matrices: the whole chain in one CTA --------------------------------------------------------------------
// Where X, A and V fit into shared memory together (sides of at most 128 and 256, seven blocks in all) they stay there from
// the first step to the last, and a matrix costs one launch instead of eighteen.  What takes time is the way from a
// product to its epilogue and back, three of each a step: 64 x 64 takes 25 us, 1.6 us a product (the launches of larger
// matrices 82 us); 128 x 128 48 us (110), thirty of 128 x 192 64 us (121).  Sums of hi hi are taken out after every block (after every
// second one the result of a 128 x 128 matrix was 2.4e-6 off instead of 1.6e-6).
constexpr int kTinyThreads = 256, kTinyBlocks = 7, kTinyCols = 256;

// the scalars of every step, in the products' scales (see scales_of)
struct Steps {
    float gram[D3GS_NS_MAX_STEPS], gram_shift[D3GS_NS_MAX_STEPS], square[D3GS_NS_MAX_STEPS], square_shift[D3GS_NS_MAX_STEPS],
        apply[D3GS_NS_MAX_STEPS];
    float first, last;    // scale of X at the start, one over that at the end
    uint32_t cubic;       // a bit for each step with c = 0
    int32_t count;
};

__global__ void __launch_bounds__(kTinyThreads, 1) ns_tiny_kernel(const __grid_constant__ Table t, const __grid_constant__ Steps sp) {
    constexpr uint32_t kBlock = 2 * kPlane;
    extern __shared__ char raw[];
    __shared__ uint64_t s_done, s_end;
    __shared__ uint32_t s_tmem;
    __shared__ int s_failed;
    __shared__ double s_norm[kTinyThreads / 32];
    char* const smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Matrix& m = t.mat[blockIdx.x];
    const int nk = m.nk, mk = m.mk;
    char* const x = smem;                        // nk blocks
    char* const ab = x + nk * (int)kBlock;       // mk blocks: A, then B
    char* const v = ab + mk * (int)kBlock;       // mk blocks
    constexpr uint32_t columns = 512;            // hi hi of two blocks, and the rest (and 128 that a power of two brings)
    if (tid == 0) {
        mbar_init(&s_done, 1);
        mbar_init(&s_end, 1);
        s_failed = 0;
        fence_mbar_init();
    }
    if (warp == 0) tmem_alloc<1>(&s_tmem, columns);
    for (int i = tid; i < nk * (int)kBlock / 16; i += kTinyThreads) reinterpret_cast<uint4*>(x)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();   // no CTA of the next kernel takes an SM before this one has its TMEM
    let_next_start();
    wait_for_previous();

    // ---- momentum, norm, X: pieces of eight columns of U ----
    const bool tall = m.rows > m.cols;
    const int per_row = (m.cols + 7) / 8, pieces = m.rows * per_row;
    const Access access = access_of(t, m);
    auto load_piece = [&](int i, int& r, int& c, float (&u)[8], bool update) {
        r = i / per_row;
        c = (i - r * per_row) * 8;
        const int n = min(8, m.cols - c);
        load_src8(t, m, r * m.src_stride + c, access.src, n, u);
        if (m.momentum) {
            float buf[8];
            load8(m.momentum + r * m.cols + c, access.state, n, buf);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (update) buf[e] = fmaf(t.mu, buf[e], t.fresh * u[e]);
                u[e] = update_of(t, u[e], buf[e]);
            }
            if (update) store8(m.momentum + r * m.cols + c, access.state, n, buf);
        }
    };
    double sum = 0.0;
#pragma unroll 2
    for (int i = tid; i < pieces; i += kTinyThreads) {
        int r, c;
        float u[8];
        load_piece(i, r, c, u, true);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += (double)u[e] * (double)u[e];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) s_norm[warp] = sum;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    sum = 0.0;
    for (int k = 0; k < kTinyThreads / 32; ++k) sum += s_norm[k];
    const Factor scale = factor_of(sum, t.eps, sp.first);
#pragma unroll 2
    for (int i = tid; i < pieces; i += kTinyThreads) {   // (a thread reads the momentum that it wrote)
        int r, c;
        float u[8];
        load_piece(i, r, c, u, false);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split2(scale(u[2 * e]), scale(u[2 * e + 1]), hi[e], lo[e]);
        if (!tall) {   // (a piece's columns behind the matrix' end are zeros, as all that is not written)
            put<true>(x + (c / kCols) * (int)kBlock + block_offset(r, c % kCols), hi, lo);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                char* const to = x + (r / kCols) * (int)kBlock + block_offset(c + e, r % kCols);
                *reinterpret_cast<uint16_t*>(to) = (uint16_t)(hi[e / 2] >> (16 * (e & 1)));
                *reinterpret_cast<uint16_t*>(to + kPlane) = (uint16_t)(lo[e / 2] >> (16 * (e & 1)));
            }
        }
    }

    // ---- products ----
    const uint32_t tmem = s_tmem, polls = t.hooks.poll_limit;
    const int half = warp >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const int tiles = (nk + 1) / 2;              // of B X: 128 columns each
    bool ok = true;
    uint32_t phase = 0;
    auto next_phase = [&]() {   // what was written to shared memory is there for the products, TMEM is free
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
    };
    // one round of products: `blocks` (at most two) column blocks, hi hi of each to a sum of its own, the rest together
    auto issue = [&](int blocks, uint32_t a, uint32_t a_next, uint32_t b, uint32_t b_next, uint32_t step, uint32_t idesc, bool new_rest) {
        for (int k = 0; k < blocks; ++k, a += a_next, b += b_next)
#pragma unroll
            for (int q = 0; q < kCols / 16; ++q) {
                const uint64_t ah = operand(a + q * 2), al = operand(a + kPlane / 16 + q * 2);
                const uint64_t bh = operand(b + q * step), bl = operand(b + kPlane / 16 + q * step);
                tc_mma<1>(tmem + k * 128, ah, bh, idesc, q != 0);
                tc_mma<1>(tmem + 256, ah, bl, idesc, !new_rest || k != 0 || q != 0);
                tc_mma<1>(tmem + 256, al, bh, idesc, true);
            }
        tc_commit<1>(&s_done);
    };
    auto wait_done = [&]() {
        __syncwarp();
        if (ok) ok = __all_sync(~0u, wait_for(&s_done, phase & 1, polls));
        if (!ok) s_failed = 1;
        tc_fence_after();
    };
    auto take = [&](float* to, uint32_t at) {   // adds 32 columns
        float w[32];
        tmem_load32(tmem + at + lanes, w);
#pragma unroll
        for (int i = 0; i < 32; ++i) to[i] += w[i];
    };
    constexpr uint32_t kNext = kBlock / 16;
    const uint32_t x0 = operand_low(smem_u32(x), 16), x0_across = operand_low(smem_u32(x), kBlock), ab0 = operand_low(smem_u32(ab), 16),
                   v0 = operand_low(smem_u32(v), 16), square = instruction(false, 128, mk * kCols);
    const int share = mk * 32, col = half * share;       // columns of A and B that each half of the warps finishes
    char* const at_ab = ab + (col / kCols) * (int)kBlock;
    const int on = row < m.m ? row - col : -256;         // the diagonal among them
    for (int step = 0; step < sp.count; ++step) {
        const bool cubic = sp.cubic >> step & 1;
        float f[128];   // of A or B, or of X
#pragma unroll
        for (int c = 0; c < 64; ++c) f[c] = 0.0f;
        for (int k = 0; k < nk; k += 2, ++phase) {   // A = X X^T, two blocks a round
            next_phase();
            const int blocks = min(2, nk - k);
            if (tid == 0 && !(withholds_all(t) && phase == 0))   // (a test: the first products never come)
                issue(blocks, x0 + k * kNext, kNext, x0 + k * kNext, kNext, 2, square, k == 0);
            wait_done();
#pragma unroll
            for (int c = 0; c < 64; c += 32) {
                if (c >= share) continue;
                take(f + c, col + c);
                if (blocks > 1) take(f + c, 128 + col + c);
                if (k + 2 >= nk) take(f + c, 256 + col + c);
            }
        }
#pragma unroll
        for (int c = 0; c < 64; c += 8) {
            if (c >= share) continue;
            uint32_t hi[4], lo[4];
            const uint32_t at = block_offset(row, col % kCols + c);
            finish(f + c, sp.gram[step], sp.gram_shift[step], cubic ? on - c : -1, hi, lo);
            put<true>(at_ab + at, hi, lo);
            if (cubic) continue;
            if ((unsigned)(on - c) < 8u) finish(f + c, sp.gram[step], sp.gram_shift[step], on - c, hi, lo);
            put<true>(at_ab + mk * (int)kBlock + at, hi, lo);   // V
        }
        if (!cubic) {
            next_phase();   // B = a I + c A V
            if (tid == 0) issue(mk, ab0, kNext, v0, kNext, 2, square, true);
            wait_done();
#pragma unroll
            for (int c = 0; c < 64; ++c) f[c] = 0.0f;
#pragma unroll
            for (int c = 0; c < 64; c += 32) {
                if (c >= share) continue;
                take(f + c, col + c);
                if (mk > 1) take(f + c, 128 + col + c);
                take(f + c, 256 + col + c);
            }
#pragma unroll
            for (int c = 0; c < 64; c += 8) {
                if (c >= share) continue;
                uint32_t hi[4], lo[4];
                finish(f + c, sp.square[step], sp.square_shift[step], on - c, hi, lo);
                put<true>(at_ab + block_offset(row, col % kCols + c), hi, lo);
            }
            ++phase;
        }
#pragma unroll
        for (int c = 0; c < 128; ++c) f[c] = 0.0f;
#pragma unroll
        for (int w = 0; w < 2; ++w) {   // X <- B X, two blocks a round, one for each half of the warps
            if (w >= tiles) continue;
            next_phase();
            if (tid == 0)
                issue(mk, ab0, kNext, x0_across + w * 2 * kNext, (kPlane / 2) / 16, 2048 / 16, instruction(true, 128, min(2, nk - 2 * w) * kCols), true);
            wait_done();
            if (2 * w + half < nk) {
#pragma unroll
                for (int c = 0; c < 64; c += 32) {
                    take(f + w * 64 + c, half * 64 + c);
                    if (mk > 1) take(f + w * 64 + c, 128 + half * 64 + c);
                    take(f + w * 64 + c, 256 + half * 64 + c);
                }
            }
            ++phase;
        }
#pragma unroll
        for (int c = 0; c < 128; c += 8) {   // every product has read X by now
            const int block = c / 64 * 2 + half;
            if (block >= nk) continue;
            uint32_t hi[4], lo[4];
            finish(f + c, sp.apply[step], 0.0f, -1, hi, lo);
            put<true>(x + block * (int)kBlock + block_offset(row, c % kCols), hi, lo);
        }
    }
    if (tid == 0) {   // whatever was issued has ended before TMEM is handed back
        tc_commit<1>(&s_end);
        wait_for(&s_end, 0);
    }
    next_phase();
    if (warp == 0) tmem_free<1>(tmem, columns);

    // ---- result ----
    const bool failed = s_failed != 0;
    for (int i = tid; i < pieces; i += kTinyThreads) {
        const int r = i / per_row, c = (i - r * per_row) * 8, n = min(8, m.cols - c);
        float u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int xr = tall ? c + e : r, xc = tall ? r : c + e;
            const char* const at = x + (xc / kCols) * (int)kBlock + block_offset(xr, xc % kCols);   // (in X, up to its last block's end)
            u[e] = __half2float(*reinterpret_cast<const __half*>(at)) + __half2float(*reinterpret_cast<const __half*>(at + kPlane));
        }
        write_result8(t, m, r * m.cols + c, access.state, n, u, sp.last, failed);
    }
}

// ---- small matrices: one 128 x 128 tile a cluster, its CTAs share the summed axis ---------------------------------
// With few tiles the summed axis is what takes time, the long one of X X^T: there the CTAs of a cluster (1, 2, 4 or 8)
// each sum a part of it, put their sums into shared memory and each finish a part of the columns, adding the parts in the
// order of their ranks.  The other products sum over at most kPairFrom / 64 = 6 blocks, in one CTA.
//
// What orders the accesses of such a cluster, one by one: a stage is written by bulk copies and read by products, ordered by
// s_full; the next copy into it by s_empty (a commit: the products have read it).  The sums are plain stores into the same
// memory: behind s_last, the commit of all products, whose copies had landed before.  Other CTAs read them behind the first
// cluster barrier (its arrival releases, its wait acquires for the cluster), and no CTA leaves before the second.  All ten
// warps arrive at both, the two that load and issue after __syncwarp.  Results are plain stores to memory; bulk copies read
// them in the next kernel, behind griddepcontrol.wait, which returns when this grid has ended and its stores are visible.
// Nine convolution layers of 3 to 256 rows take 165 us, eighteen launches of 9 us with the tensor cores busy for 5 to 7 %:
// what bounds them is one launch after another, each a wait for the last one's memory, a fill of the stages, the way out
// through TMEM and shared memory.
constexpr int kSmallThreads = 320, kTile = 128;
struct SmallStages {
    static constexpr uint32_t kLeft = 2 * kPlane, kRight = 2 * kPlane, kStage = kLeft + kRight;
    static constexpr int kCount = 3;
    static constexpr uint32_t kBytes = kCount * kStage + 1024;   // alignment to 1024
};

template <int MODE>
__global__ void __launch_bounds__(kSmallThreads, 1) ns_small_kernel(const __grid_constant__ Table t) {
    using S = SmallStages;
    constexpr uint32_t kBlock = 2 * kPlane;   // every operand has two planes
    constexpr uint32_t kTmem = 512;           // columns: hi hi twice, and the rest
    extern __shared__ char raw[];
    __shared__ uint64_t s_full[S::kCount], s_empty[S::kCount], s_sum[2], s_taken[2], s_last;
    __shared__ uint32_t s_tmem;
    char* const smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int parts = MODE == kGram ? (int)cluster_size() : 1, part = MODE == kGram ? (int)cluster_rank() : 0;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kCount; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_sum[i], 1);
            mbar_init(&s_taken[i], 256);
        }
        mbar_init(&s_last, 1);
        fence_mbar_init();
    }
    if (warp == 9) tmem_alloc<1>(&s_tmem, kTmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem, polls = t.hooks.poll_limit;
    int block;
    const Matrix& m = t.mat[find_matrix(t, (int)blockIdx.x / parts, block)];
    int ti, tj;
    if (MODE == kApply) {
        const int across = (m.nk + 1) / 2;
        ti = block / across;
        tj = block % across;
    } else {   // column tj of the upper triangle holds tj + 1 tiles
        tj = (int)((sqrtf(8.0f * (float)block + 1.0f) - 1.0f) * 0.5f);
        while ((tj + 1) * (tj + 2) / 2 <= block) ++tj;
        while (tj * (tj + 1) / 2 > block) --tj;
        ti = block - tj * (tj + 1) / 2;
    }
    const bool same = MODE != kApply && ti == tj;      // both operands are one tile
    const char* const left = MODE == kGram ? m.x[t.from] : MODE == kSquare ? m.a : m.b;
    const char* const right = MODE == kSquare ? m.a : m.x[t.from];
    const int all = MODE == kGram ? m.nk : m.mk;       // column blocks summed over, this CTA's share of them
    const int first = all * part / parts, blocks = all * (part + 1) / parts - first;
    bool ok = true;
    let_next_start();
    wait_for_previous();

    if (warp == 8) {
        if (lane == 0) {
            const int landing = withholds_first(t) ? 1 : 0;
            int k = 0;
            for (; k < blocks && !withholds_all(t); ++k) {
                const int st = k % S::kCount;
                if (k >= S::kCount) ok = wait_for(&s_empty[st], (k / S::kCount - 1) & 1, polls);
                if (!ok) break;
                char* const a = smem + st * S::kStage;
                char* const b = a + S::kLeft;
                if (k < landing) continue;   // a test: this copy never comes
                const int kb = first + k;
                if (MODE == kApply) {
                    const int wide = 2 * tj + 1 < m.nk ? 2 : 1;            // the last tile may be one block wide
                    mbar_arrive_expect_tx(&s_full[st], S::kLeft + 2 * wide * (kPlane / 2));
                    bulk_copy_g2s(a, left + ((int64_t)ti * m.mk + kb) * kBlock, S::kLeft, &s_full[st]);
                    for (int p = 0; p < 2; ++p)
                        for (int w = 0; w < wide; ++w)                     // 64 rows of a block: one half of a plane
                            bulk_copy_g2s(b + (p * 2 + w) * (kPlane / 2),
                                          right + ((int64_t)(kb >> 1) * m.nk + 2 * tj + w) * kBlock + p * kPlane +
                                              (kb & 1) * (kPlane / 2),
                                          kPlane / 2, &s_full[st]);
                } else {
                    const bool v = MODE == kSquare && kb >> 1 == tj, shared = same && !v;
                    mbar_arrive_expect_tx(&s_full[st], shared ? S::kLeft : S::kStage);
                    bulk_copy_g2s(a, left + ((int64_t)ti * all + kb) * kBlock, S::kLeft, &s_full[st]);
                    if (!shared)
                        bulk_copy_g2s(b, v ? m.v + (int64_t)kb * kBlock : right + ((int64_t)tj * all + kb) * kBlock, S::kRight,
                                      &s_full[st]);
                }
            }
            if (!ok) drain(s_full, S::kCount, max(k - S::kCount, landing), k);
        }
    } else if (warp == 9) {
        if (lane == 0) {
            const uint32_t idesc = instruction(MODE == kApply, 128, kTile);
            constexpr uint32_t kStep = (MODE == kApply ? 2048 : 32) / 16, kNext = MODE == kApply ? kPlane / 2 : 16;
            const uint32_t a0 = operand_low(smem_u32(smem), 16), b0 = operand_low(smem_u32(smem) + S::kLeft, kNext);
            int st = 0, phase = 0;
            for (int k = 0; k < blocks; ++k) {
                const int buf = k & 1;
                ok = wait_for(&s_full[st], phase, polls);
                if (ok && k > 1) ok = wait_for(&s_taken[buf], ((k >> 1) - 1) & 1, polls);
                if (!ok) break;
                tc_fence_after();
                const bool shared = same && !(MODE == kSquare && (first + k) >> 1 == tj);
                const uint32_t a = a0 + st * (S::kStage / 16), b = shared ? a : b0 + st * (S::kStage / 16);
                const uint32_t d = tmem + buf * kTile;
#pragma unroll
                for (int q = 0; q < kCols / 16; ++q) tc_mma<1>(d, operand(a + q * 2), operand(b + q * kStep), idesc, q != 0);
                tc_commit<1>(&s_sum[buf]);
#pragma unroll
                for (int q = 0; q < kCols / 16; ++q) {
                    tc_mma<1>(tmem + 2 * kTile, operand(a + q * 2), operand(b + kPlane / 16 + q * kStep), idesc, k != 0 || q != 0);
                    tc_mma<1>(tmem + 2 * kTile, operand(a + kPlane / 16 + q * 2), operand(b + q * kStep), idesc, true);
                }
                tc_commit<1>(&s_empty[st]);
                if (++st == S::kCount) st = 0, phase ^= 1;
            }
            // everything issued so far, in the good case the whole sum
            tc_commit<1>(&s_last);
            if (!ok) wait_for(&s_last, 0);
        }
    } else {
        constexpr int kPart = kTile / 2;                 // columns of a thread; the warps' upper half takes the right ones
        const int half = warp >> 2;
        float v[kPart];
#pragma unroll
        for (int c = 0; c < kPart; ++c) v[c] = 0.0f;
        auto take = [&](uint32_t from) {
#pragma unroll
            for (int c = 0; c < kPart; c += 32) {
                float w[32];
                tmem_load32(tmem + from + half * kPart + c + ((uint32_t)(warp & 3) << 21), w);
#pragma unroll
                for (int i = 0; i < 32; ++i) v[c + i] += w[i];
            }
        };
        for (int k = 0; k < blocks; ++k) {
            ok = __all_sync(~0u, wait_for(&s_sum[k & 1], (k >> 1) & 1, polls));
            if (!ok) break;
            tc_fence_after();
            take((k & 1) * kTile);
            tc_fence_before();
            mbar_arrive(&s_taken[k & 1]);
        }
        if (ok) ok = __all_sync(~0u, wait_for(&s_last, 0, polls));
        tc_fence_after();
        if (ok && blocks > 0) take(2 * kTile);
        // every product has read its operands by now: their shared memory is free
        const uint32_t r = threadIdx.x & 127;
        const int wide = MODE == kApply ? m.nk : m.mk;   // blocks across the result
        char* const out = MODE == kGram && !t.cubic ? m.a : MODE != kApply ? m.b : m.x[t.from ^ 1];
        // The sums go through shared memory, four columns of 128 rows after one another, so that what follows is a loop: code
        // that every CTA runs once is bound by fetching it, and unrolled over the registers it took twice the time.
        float4* const sums = reinterpret_cast<float4*>(smem) + r;
#pragma unroll
        for (int c = 0; c < kPart; c += 4) sums[(half * kPart + c) * 32] = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
        if (!ok) *t.fail = 1;
        if (parts > 1) cluster_sync();
        const int valid = min(2, wide - 2 * tj);         // of the tile's two blocks across
        const bool mirrored = MODE != kApply && !same, keeps_v = MODE == kGram && same && !t.cubic;
        // This tile's blocks; the mirrored tile's, where this thread's row is a column, or V's, of tiles on the diagonal.
        // With one CTA they are put together in shared memory and leave as whole blocks.
        char* const to_direct = out + ((int64_t)ti * wide + 2 * tj) * kBlock;
        char* const to_other = mirrored ? out + ((int64_t)tj * wide + 2 * ti) * kBlock : m.v + (int64_t)2 * ti * kBlock;
        char* const direct = parts == 1 ? smem + 2 * kBlock : to_direct;
        char* const other = parts == 1 ? smem + 4 * kBlock : to_other;
        const int share = kPart / parts, begin = (2 * part + half) * share;   // columns this CTA finishes, half of them here
        const int end = min(begin + share, valid * kCols);
        const int diagonal = same && ti * kRows + (int)r < m.m ? (int)r : -256;
#pragma unroll 1
        for (int c = begin; c < end; c += 8) {
            float w[8];
            if (parts == 1) {
                const float4 a = sums[c * 32], b = sums[(c + 4) * 32];
                w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
            } else {
                float4 a[8], b[8];   // all parts on their way before the first is added
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (q < parts) {
                        a[q] = load_shared_of(smem_u32(sums + c * 32), q);
                        b[q] = load_shared_of(smem_u32(sums + (c + 4) * 32), q);
                    }
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = 0.0f;
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (q < parts) {
                        w[0] += a[q].x, w[1] += a[q].y, w[2] += a[q].z, w[3] += a[q].w;
                        w[4] += b[q].x, w[5] += b[q].y, w[6] += b[q].z, w[7] += b[q].w;
                    }
            }
            const uint32_t o = (c / kCols) * kBlock + block_offset(r, c % kCols);
            uint32_t hi[4], lo[4];
            finish(w, t.out_scale, t.shift, MODE == kSquare || (MODE == kGram && t.cubic) ? diagonal - c : -1, hi, lo);
            put<true>(direct + o, hi, lo);
            if (mirrored) write_mirrored<true>(other + (r / kCols) * kBlock, c, r % kCols, hi, lo);
            if (keeps_v) {
                finish(w, t.out_scale, t.shift, diagonal - c, hi, lo);
                put<true>(other + o, hi, lo);
            }
        }
        if (parts == 1) {
            fence_proxy_async_smem();
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (threadIdx.x == 0 && ok) {
                bulk_copy_s2g(to_direct, direct, valid * kBlock);
                if (mirrored || keeps_v) bulk_copy_s2g(to_other, other, (mirrored ? 2 : valid) * kBlock);
                bulk_commit_group();
                bulk_wait_group_read0();   // (what leaves is in memory when the grid has ended)
            }
        } else {
            cluster_sync();   // no CTA leaves while another reads its sums
        }
    }
    if (warp >= 8) {
        if (!ok) *t.fail = 1;
        __syncwarp();
        if (parts > 1) {
            cluster_sync();
            cluster_sync();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 9) tmem_free<1>(tmem, kTmem);
}

// ---- large matrices: one 256 x N tile a pair of CTAs --------------------------------------------------------------
// A 128 x 128 tile reads 8 KB of shared memory for every 64 cycles of products and takes 64 KB in for every 768, more
// than its 128 bytes a cycle.  In a pair each CTA holds 128 rows of the left and N / 2 columns of the right factor, and
// both are read by the products of both: at N = 256, 8 KB in 128 cycles.  CTA 0 issues; CTA 1's second warp passes on
// that its tiles have arrived.
//
// Measured: 4096 x 4096 in 16 bits 1.65 ms a call of five steps, 0.83 PFLOP/s, with X's second plane counted 1.08, where
// the power limit leaves a plain product 1.40; tensor cores busy for 69 % of B X, 56 % of the others
// (1.84 rounds of tiles on 74 pairs).  2048 x 2048 in 32 bits 0.51 to 0.58 ms: busy for 58 % of B X in 256-wide tiles, 38 %
// of the others in 128-wide ones, which an SM takes 48 KB in for every 768 cycles of products.
constexpr int kPairThreads = 320;
template <int L, int R, int N> struct PairStages {
    static constexpr uint32_t kLeft = L * kPlane, kRight = R * (uint32_t)N / 2 * 128, kStage = kLeft + kRight;
    // A commit takes the issuing thread about 400 cycles.  Where a column block is 256 or 512 cycles of products one
    // commit hands back two stages (one -> two: 2048 x 2048 305 -> 300 us, 4096 x 4096 1715 -> 1698).
    static constexpr int kGroup = L == 1 && R == 1 ? 2 : 1;
    static constexpr int kCount = (int)(196608u / kStage) / kGroup * kGroup;
    static constexpr uint32_t kBytes = kCount * kStage + 1024;
};

// SHARED: several pairs share the sum of a tile.
template <bool F32, int MODE, int RIGHT, int N, bool SHARED = false>
__global__ void __launch_bounds__(kPairThreads, 1) ns_pair_kernel(const __grid_constant__ Table t) {
    using P = Planes<F32, MODE, RIGHT>;
    constexpr int L = P::kLeft, R = P::kRight, kWide = N / kCols;   // column blocks of the tile
    using S = PairStages<L, R, N>;
    constexpr int kSums = N == 128 ? 2 : 1;              // sums of hi hi in TMEM: as many as it has room for
    // With two of them a commit says both that a block's hi hi is there and that the stage of the block before is free.
    // The loading thread may look at it late: one barrier a stage, so that none completes twice before it has looked.
    constexpr bool kOneCommit = F32 && kSums == 2;
    constexpr int kSumBars = kOneCommit ? S::kCount : 1;
    constexpr uint32_t kTmem = F32 ? 512 : N;
    extern __shared__ char raw[];
    __shared__ uint64_t s_full[S::kCount], s_empty[S::kCount], s_sum[kSumBars], s_taken[kSums], s_last;
    __shared__ uint32_t s_tmem;
    char* const smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)cluster_rank();
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kCount; ++i) {
            mbar_init(&s_full[i], rank == 0 ? 2 : 1);   // CTA 0: its own tiles, and word from CTA 1
            mbar_init(&s_empty[i], 1);
        }
        for (int i = 0; i < kSumBars; ++i) mbar_init(&s_sum[i], 1);
        for (int i = 0; i < kSums; ++i) mbar_init(&s_taken[i], 16);   // the eight warps of both CTAs
        mbar_init(&s_last, 1);
        fence_mbar_init();
    }
    if (warp == 9) tmem_alloc<2>(&s_tmem, kTmem);
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = s_tmem, polls = t.hooks.poll_limit;
    int block;
    const int parts = SHARED ? t.parts : 1, tile = (int)blockIdx.x / 2 / parts, part = (int)blockIdx.x / 2 - tile * parts;
    const Matrix& m = t.mat[find_matrix(t, tile, block)];
    const int pairs = (m.mb + 1) / 2;                   // 256-row tiles
    int ti, tj;
    if (MODE == kApply) {
        ti = block % pairs;                             // neighbours share the columns of X, the larger factor
        tj = block / pairs;
    } else if (N == 256) {                              // column tj of the upper triangle holds tj + 1 tiles
        tj = (int)((sqrtf(8.0f * (float)block + 1.0f) - 1.0f) * 0.5f);
        while ((tj + 1) * (tj + 2) / 2 <= block) ++tj;
        while (tj * (tj + 1) / 2 > block) --tj;
        ti = block - tj * (tj + 1) / 2;
    } else {                                            // columns 2 h and 2 h + 1 hold h + 1 tiles each
        int h = (int)(sqrtf((float)block + 0.25f) - 0.5f);
        while ((h + 1) * (h + 2) <= block) ++h;
        while (h * (h + 1) > block) --h;
        const int in = block - h * (h + 1);
        tj = 2 * h + in / (h + 1);
        ti = in % (h + 1);
    }
    const bool same = MODE != kApply && N == 256 && ti == tj;   // both operands are one tile
    const int row = 2 * ti + rank;                              // this CTA's block of rows
    const char* const left = MODE == kGram ? m.x[t.from] : MODE == kSquare ? m.a : m.b;
    const char* const right = MODE == kSquare ? m.a : m.x[t.from];
    constexpr uint32_t kLeftBlock = MODE == kGram ? P::kX : P::kAB, kRightBlock = MODE == kSquare ? P::kAB : P::kX;
    const int all = MODE == kGram ? m.nk : m.mk;         // column blocks summed over, this pair's share of them
    const int first = all * part / parts, blocks = all * (part + 1) / parts - first;
    bool ok = true;
    let_next_start();
    wait_for_previous();

    if (warp == 8) {
        if (lane == 0) {
            // blocks behind the matrix's end are taken from its last ones; what they give is not written
            const int lrow = min(row, m.mb - 1), landing = withholds_first(t) ? 1 : 0;
            int k = 0;
            for (; k < blocks && !withholds_all(t); ++k) {
                const int st = k % S::kCount;
                if (k >= S::kCount) {
                    if (kOneCommit) {   // block k - kCount is done with when the block after it has been committed
                        const int j = k - S::kCount + 1;
                        ok = wait_for(&s_sum[j % kSumBars], (j / kSumBars) & 1, polls);
                    } else if (st % S::kGroup == 0) {
                        ok = wait_for(&s_empty[st / S::kGroup], (k / S::kCount - 1) & 1, polls);
                    }
                }
                if (!ok) break;
                char* const a = smem + st * S::kStage;
                char* const b = a + S::kLeft;
                if (k < landing) continue;   // a test: this copy never comes
                const int kb = first + k;
                const bool shared = same && !(MODE == kSquare && kb >> 2 == tj);
                mbar_arrive_expect_tx(&s_full[st], shared ? S::kLeft : S::kStage);
                bulk_copy_g2s(a, left + ((int64_t)lrow * all + kb) * kLeftBlock, S::kLeft, &s_full[st]);
                if (MODE == kApply) {
                    for (int p = 0; p < R; ++p)
                        for (int w = 0; w < kWide / 2; ++w)                // 64 rows of a block: one half of a plane
                            bulk_copy_g2s(b + (p * (kWide / 2) + w) * (kPlane / 2),
                                          right + ((int64_t)(kb >> 1) * m.nk + min(kWide * tj + kWide / 2 * rank + w, m.nk - 1)) * kRightBlock +
                                              p * kPlane + (kb & 1) * (kPlane / 2),
                                          kPlane / 2, &s_full[st]);
                } else if (N == 256) {
                    const int j = min(2 * tj + rank, m.mb - 1);
                    const bool v = MODE == kSquare && kb >> 1 == j;
                    if (!shared)
                        bulk_copy_g2s(b, v ? m.v + (int64_t)kb * kRightBlock : right + ((int64_t)j * all + kb) * kRightBlock, S::kRight,
                                      &s_full[st]);
                } else {
                    const int j = min(tj, m.mb - 1);
                    const bool v = MODE == kSquare && kb >> 1 == j;
                    const char* from = v ? m.v + (int64_t)kb * kRightBlock : right + ((int64_t)j * all + kb) * kRightBlock;
                    for (int p = 0; p < R; ++p)
                        bulk_copy_g2s(b + p * (kPlane / 2), from + p * kPlane + rank * (kPlane / 2), kPlane / 2, &s_full[st]);
                }
            }
            if (!ok) drain(s_full, S::kCount, max(k - S::kCount, landing), k);
        }
    } else if (warp == 9) {
        if (lane == 0 && rank == 1) {
            for (int k = 0; k < blocks && ok; ++k) {
                ok = wait_for(&s_full[k % S::kCount], (k / S::kCount) & 1, polls);
                if (ok) mbar_arrive_at(&s_full[k % S::kCount], 0);
            }
        } else if (lane == 0) {
            const uint32_t idesc = instruction(MODE == kApply, 256, N);
            constexpr uint32_t kStep = (MODE == kApply ? 2048 : 32) / 16, kNext = MODE == kApply ? kPlane / 2 : 16;
            constexpr uint32_t kLowB = (uint32_t)N / 2 * 128 / 16;   // from hi to lo of the right factor
            const uint32_t a0 = operand_low(smem_u32(smem), 16), b0 = operand_low(smem_u32(smem) + S::kLeft, kNext);
            auto left_of = [&](int st) { return a0 + st * (S::kStage / 16); };
            auto right_of = [&](int k, int st) {
                const bool shared = same && !(MODE == kSquare && (first + k) >> 2 == tj);
                return shared ? left_of(st) : b0 + st * (S::kStage / 16);
            };
            auto rest = [&](int k, int st) {   // hi lo + lo hi
                const uint32_t a = left_of(st), b = right_of(k, st);
#pragma unroll
                for (int q = 0; q < kCols / 16; ++q) {
                    tc_mma<2>(tmem + kSums * N, operand(a + q * 2), operand(b + kLowB + q * kStep), idesc, k != 0 || q != 0);
                    tc_mma<2>(tmem + kSums * N, operand(a + kPlane / 16 + q * 2), operand(b + q * kStep), idesc, true);
                }
            };
            int st = 0, phase = 0, before = 0;
            for (int k = 0; k < blocks; ++k) {
                const int buf = k % kSums;
                ok = wait_for(&s_full[st], phase, polls);
                if (F32 && ok && k >= kSums) ok = wait_for(&s_taken[buf], (k / kSums - 1) & 1, polls);
                if (!ok) break;
                tc_fence_after();
                const uint32_t a = left_of(st), b = right_of(k, st);
                const uint32_t d = F32 ? tmem + buf * N : tmem;
#pragma unroll
                for (int q = 0; q < kCols / 16; ++q) tc_mma<2>(d, operand(a + q * 2), operand(b + q * kStep), idesc, (!F32 && k != 0) || q != 0);
                if (kOneCommit) {
                    if (k > 0) rest(k - 1, before);
                    tc_commit<2>(&s_sum[k % kSumBars]);
                    before = st;
                } else if (F32) {
                    tc_commit<2>(&s_sum[0]);
                    rest(k, st);
                    tc_commit<2>(&s_empty[st]);
                } else {
                    if (R == 2) {
#pragma unroll
                        for (int q = 0; q < kCols / 16; ++q) tc_mma<2>(d, operand(a + q * 2), operand(b + kLowB + q * kStep), idesc, true);
                    }
                    if (st % S::kGroup == S::kGroup - 1) tc_commit<2>(&s_empty[st / S::kGroup]);
                }
                if (++st == S::kCount) st = 0, phase ^= 1;
            }
            if (kOneCommit && ok) rest(blocks - 1, before);
            tc_commit<2>(&s_last);
            if (!ok) wait_for(&s_last, 0, 0);
        }
    } else {
        constexpr int kPart = N / 2;                     // columns of a thread; the warps' upper half takes the right ones
        const int half = warp >> 2;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21, r = threadIdx.x & 127;
        float scale = t.out_scale;
        if (!F32 && MODE != kSquare && t.exact) {   // what X leaves out of 1 / |U|
            const float rest = *reinterpret_cast<const float*>(m.norms - 1);
            scale *= MODE == kGram ? rest * rest : rest;
        }
        float v[F32 ? kPart : 1];
#pragma unroll
        for (int c = 0; c < kPart && F32; ++c) v[c] = 0.0f;
        auto take = [&](uint32_t from) {
#pragma unroll
            for (int c = 0; c < kPart; c += 32) {
                float w[32];
                tmem_load32(tmem + from + half * kPart + c + lanes, w);
#pragma unroll
                for (int i = 0; i < 32; ++i) v[c + i] += w[i];
            }
        };
        if constexpr (F32)
            for (int k = 0; k < blocks; ++k) {
                ok = __all_sync(~0u, wait_for(&s_sum[k % kSumBars], (k / kSumBars) & 1, polls));
                if (!ok) break;
                tc_fence_after();
                take(k % kSums * N);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_at(&s_taken[k % kSums], 0);
            }
        if (ok) ok = __all_sync(~0u, wait_for(&s_last, 0, polls));
        tc_fence_after();
        if (!ok) *t.fail = 1;
        // What follows are loops over TMEM: code that every CTA runs once is bound by fetching it.
        const uint32_t sums_at = tmem + half * kPart + lanes;
        if constexpr (F32) {
            if (ok && (!SHARED || blocks > 0)) take(kSums * N);
#pragma unroll
            for (int c = 0; c < kPart; c += 32) tmem_store32(sums_at + c, v + c);
            tmem_wait_stored();
        }
        // A tile that several pairs share: everyone puts its sums down, four columns of 128 rows after one another, the last
        // one to do so adds them up in the order of the parts and goes on.
        bool finishes = true;
        if constexpr (SHARED) {
            __shared__ uint32_t s_ticket;
            constexpr int kNext = (int)(kSumBytes / 16);
            float4* const sums = t.sums + (int64_t)(tile * 2 + rank) * parts * kNext + half * kPart * 32 + r;
#pragma unroll 1
            for (int c = 0; c < kPart; c += 32) {
                float w[32];
                tmem_load32(sums_at + c, w);
                const bool some = F32 || blocks > 0;
#pragma unroll
                for (int i = 0; i < 32; i += 4)
                    __stcg(sums + part * kNext + (c + i) * 32, some ? make_float4(w[i], w[i + 1], w[i + 2], w[i + 3]) : make_float4(0, 0, 0, 0));
            }
            __threadfence();
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (threadIdx.x == 0) {
                uint32_t* const ticket = t.tickets + tile * 2 + rank;
                s_ticket = atomicAdd(ticket, 1u);
                if (s_ticket == (uint32_t)parts - 1) *ticket = 0;   // for the next product
                __threadfence();
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            finishes = s_ticket == (uint32_t)parts - 1;
#pragma unroll 1
            for (int c = 0; c < kPart && finishes; c += 32) {
                float w[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) w[i] = 0.0f;
#pragma unroll 1
                for (int q = 0; q < parts; q += 4) {   // (four or eight parts)
                    float4 f[4][8];
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int i = 0; i < 8; ++i) f[k][i] = __ldcg(sums + (q + k) * kNext + (c + 4 * i) * 32);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            w[4 * i] += f[k][i].x, w[4 * i + 1] += f[k][i].y, w[4 * i + 2] += f[k][i].z, w[4 * i + 3] += f[k][i].w;
                }
                tmem_store32(sums_at + c, w);
            }
            tmem_wait_stored();
        }
        // Every product has read its operands by now: their shared memory takes the finished blocks, from where they
        // leave as whole blocks.
        const int wide = MODE == kApply ? m.nk : m.mk;   // blocks across the result
        char* const out = MODE == kGram && !t.cubic ? m.a : MODE != kApply ? m.b : m.x[t.from ^ 1];
        constexpr uint32_t kOutBlock = MODE == kApply ? P::kX : P::kAB, kOutBytes = P::kOut * kPlane;
        const int col = kWide * tj + half * (kPart / kCols);   // first block column of this thread
        const bool mirrored = MODE != kApply && (N == 256 ? tj > ti : tj > 2 * ti + 1);
        // V's blocks take the place of mirrored ones, which tiles on the diagonal do not have
        const bool keeps_v = MODE == kGram && !t.cubic && (N == 256 ? col == 2 * row : tj == row);
        // space: kPart / 64 blocks and as many mirrored ones for each half; what does not fit side by side takes turns
        constexpr uint32_t kMine = kPart / kCols * kOutBytes, kSpace = MODE == kApply ? kMine : 2 * kMine;
        constexpr bool kTurns = 2 * kSpace > 196608u;
        char* const space = smem + (kTurns ? 0 : half * (N == 256 ? kSpace : kMine));
        auto write = [&]() {
#pragma unroll 1
            for (int c0 = 0; c0 < kPart; c0 += 32) {
                if (col + c0 / kCols >= wide || row >= m.mb) continue;
                float w[32];
                tmem_load32(sums_at + c0, w);
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    const int c = c0 + i;
                    const uint32_t o = block_offset(r, c % kCols);
                    uint32_t hi[4], lo[4];
                    const int in = row * kRows + (int)r, on = in < m.m ? in - (col * kCols + c) : -1;   // diagonal
                    finish(w + i, scale, t.shift, MODE == kSquare || (MODE == kGram && t.cubic) ? on : -1, hi, lo);
                    put<P::kOut == 2>(space + (c / kCols) * kOutBytes + o, hi, lo);
                    if (MODE == kGram && keeps_v) {
                        finish(w + i, scale, t.shift, on, hi, lo);
                        put<P::kOut == 2>((N == 256 ? space + kMine : smem + (2 + half) * kMine) + (c / kCols) * kOutBytes + o, hi, lo);
                    }
                    if (MODE != kApply && mirrored) {
                        // N 256: rows of one block, columns of the two blocks that the rows r belong to.  N 128: a half's 64
                        // columns are 64 rows of a block, the two halves' rows follow one another.
                        char* const to = N == 256 ? space + kMine + (r / kCols) * kOutBytes : smem + 2 * kMine + (r / kCols) * kOutBytes;
                        write_mirrored<P::kOut == 2>(to, (N == 256 ? 0 : half * kCols) + c, r % kCols, hi, lo);
                    }
                }
            }
            fence_proxy_async_smem();
        };
        // one thread of each half sends its blocks
        auto send = [&]() {
            for (int c = 0; c < kPart / kCols; ++c)
                if (col + c < wide) bulk_copy_s2g(out + ((int64_t)row * wide + col + c) * kOutBlock, space + c * kOutBytes, kOutBytes);
            if (MODE != kApply && mirrored) {
                if (N == 256) {
                    const int to = 2 * tj + half;
                    for (int c = 0; c < 2; ++c)
                        if (to < m.mb)
                            bulk_copy_s2g(out + ((int64_t)to * wide + 2 * row + c) * kOutBlock, space + kMine + c * kOutBytes, kOutBytes);
                } else if (tj < m.mb) {   // this half's block column of the mirrored tile
                    bulk_copy_s2g(out + ((int64_t)tj * wide + 2 * row + half) * kOutBlock, smem + 2 * kMine + half * kOutBytes, kOutBytes);
                }
            }
            if (MODE == kGram && keeps_v)
                for (int c = 0; c < kPart / kCols; ++c)
                    if (col + c < wide)
                        bulk_copy_s2g(m.v + (int64_t)(col + c) * kOutBlock,
                                      (N == 256 ? space + kMine : smem + (2 + half) * kMine) + c * kOutBytes, kOutBytes);
            bulk_commit_group();
            bulk_wait_group_read0();   // (what leaves is in memory when the grid has ended)
        };
        auto all_warps = []() { asm volatile("bar.sync 1, 256;" ::: "memory"); };
        const bool sender = ok && (threadIdx.x & 127) == 0 && row < m.mb;
        if (SHARED && !finishes) {
        } else if (kTurns) {
            for (int turn = 0; turn < 2; ++turn) {
                if (half == turn) write();
                all_warps();
                if (half == turn && sender) send();
                all_warps();
            }
        } else {
            write();
            all_warps();
            if (sender) send();
        }
    }
    if (warp >= 8) {
        if (!ok) *t.fail = 1;
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();   // neither CTA leaves, or frees TMEM, while the other may still use it
    tc_fence_after();
    if (warp == 9) tmem_free<2>(tmem, kTmem);
}

// ---- host ---------------------------------------------------------------------------------------------------------
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

struct Parts {
    int m, n, mb, mk, nk, rounds, sums;
    size_t x, a, v, norms, total;   // bytes
};
Parts parts_of(const D3gsOrthoMatrix& d, int planes) {
    Parts p;
    p.m = (int)(d.rows < d.cols ? d.rows : d.cols);
    p.n = (int)(d.rows < d.cols ? d.cols : d.rows);
    p.mb = (p.m + kRows - 1) / kRows;
    p.mk = (p.m + kCols - 1) / kCols;
    p.nk = (p.n + kCols - 1) / kCols;
    p.x = (size_t)p.mb * p.nk * 2 * kPlane;
    p.a = (size_t)p.mb * p.mk * planes * kPlane;
    // Every CTA of the first pass adds up all sums of squares of its matrix: at most kMaxNorms of them, since the work would be
    // quadratic in the number of values.  (One each kPieces -> this, 64 x 16777216 in 32 bits: 155 -> 137 ms.)
    const int64_t pieces = d.rows * ((d.cols + 7) / 8);
    p.rounds = (int)div_up64(pieces, (int64_t)kPieces * kMaxNorms);
    p.sums = p.rounds == 0 ? 0 : (int)div_up64(pieces, (int64_t)kPieces * p.rounds);
    p.norms = up256((size_t)p.sums * 8 + 8);
    p.v = (size_t)p.mb * 2 * planes * kPlane;
    p.total = p.m == 0 ? 0 : 2 * p.x + 2 * p.a + p.v + p.norms;
    return p;
}
// The ways through the products.  kLarge, pairs of CTAs: short sides above kPairFrom.  (Pairs from 257 on instead: 320 x
// 320 155 us either way, 384 x 384 171 instead of 167, 384 x 3456 335 instead of 176.)  kTiny, a CTA a matrix: what fits
// shared memory.  kSmall, tiles: the others.
constexpr int kPairFrom = 384;
enum { kNone = -1, kTiny = 0, kSmall = 1, kLarge = 2 };
int way_of(const D3gsOrthoMatrix& d) {
    const int64_t m = min(d.rows, d.cols), n = max(d.rows, d.cols);
    if (m == 0) return kNone;
    if (m > kPairFrom) return kLarge;
    return m > kRows || n > kTinyCols || div_up64(n, kCols) + 2 * div_up64(m, kCols) > kTinyBlocks ? kSmall : kTiny;
}
// A list of matrices, cut into batches that share launches.  The largest come first, and a batch goes the way of its largest:
// smaller ones run beside that and cost nothing.  (What is left of them when a batch is full goes its own way.)
struct List {
    const D3gsOrthoMatrix* mats;
    int32_t count, dtype;
    int32_t at = 0;
    int way = kLarge;
    const D3gsOrthoMatrix* next() {
        for (; way > kNone; --way, at = 0)
            while (at < count)
                if (way_of(mats[at++]) == way) return &mats[at - 1];
        return nullptr;
    }
};
constexpr size_t kHead = 256 + 1024;   // the failure word, the tickets
// Column blocks of a long axis that each of the pairs sharing a tile should have at least; twice that in 16 bits.
constexpr int kShare = 8;
struct Batch {
    const D3gsOrthoMatrix* mat[kMaxMatrices];
    int count = 0, way = kNone;
    // Planes of A and B.  Small matrices take two for 16-bit types too: with them it is not the products that take time, and
    // one plane would cost an 8 x 8 matrix up to twice the error of its own rounding.
    int planes = 2;
    size_t sums = 0, bytes = 0;   // room for shared sums; all of the workspace
};
bool next_batch(List& list, Batch& b) {
    b = Batch{};
    int64_t longest = 0;
    while (b.count < kMaxMatrices) {
        const D3gsOrthoMatrix* const d = list.next();
        if (!d) break;
        if (b.count == 0) {
            b.way = way_of(*d);
            b.planes = list.dtype != D3GS_DTYPE_F32 && b.way == kLarge ? 1 : 2;
        }
        b.mat[b.count++] = d;
        longest = max(longest, max(d->rows, d->cols));
        b.bytes += parts_of(*d, b.planes).total;
    }
    if (b.way == kTiny) b.bytes = 0;   // (all in shared memory)
    else {
        if (b.way == kLarge && div_up64(longest, kCols) >= 4 * kShare) b.sums = kTickets * kSumBytes;
        b.bytes += kHead + b.sums;
    }
    return b.count > 0;
}
// Batches run one after another, each in the same workspace.
size_t workspace_of(const D3gsOrthoMatrix* mats, int32_t count, const D3gsOrthoConfig& cfg) {
    List list{mats, count, cfg.dtype};
    Batch b;
    size_t most = 0;
    while (next_batch(list, b)) most = max(most, b.bytes);
    return 256 + most;   // (alignment)
}

// Scales of the operands.  The singular values of X lie in [0, x]: x = 1 at the start, and after a step the largest
// |a s + b s^3 + c s^5| over [0, x], found at x or where the derivative a + 3 b s^2 + 5 c s^4 vanishes.  No entry of X
// exceeds x, none of A and V = A + b/c I the largest of x^2, |b/c| and |x^2 + b/c|, none of B the largest
// |a + b y + c y^2| over y in [0, x^2].  Each is scaled to at most 2^15 by a power of two, so that scaling loses nothing.
struct Scales {
    float x[D3GS_NS_MAX_STEPS + 1], v[D3GS_NS_MAX_STEPS], b[D3GS_NS_MAX_STEPS];
};
float scale_for(double most) {
    int e;
    std::frexp(std::fmax(most, 1.0 / kMaxSpectrum) * 1.001, &e);   // at most 2^e; zeros are held by any scale
    return std::ldexp(1.0f, 15 - e);
}
// Fails when singular values would pass kMaxSpectrum, or where b / c would: A shares V's scale.
bool scales_of(const D3gsOrthoConfig& cfg, Scales& out) {
    double x = 1.0;
    out.x[0] = scale_for(x);
    for (int k = 0; k < cfg.steps; ++k) {
        const double a = cfg.coefficients[k][0], b = cfg.coefficients[k][1], c = cfg.coefficients[k][2], top = x * x;
        if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c) || (c != 0.0 && std::fabs(b) > kMaxSpectrum * std::fabs(c))) return false;
        auto f = [&](double y) { return std::fabs(std::sqrt(y) * (a + y * (b + y * c))); };
        double next = f(top), poly = std::fmax(std::fabs(a), std::fabs(a + top * (b + top * c)));
        auto inside = [&](double y) {
            if (y > 0.0 && y < top) next = std::fmax(next, f(y));
        };
        double shift = 0.0;
        if (c != 0.0) {
            const double d = 9.0 * b * b - 20.0 * a * c;
            if (d >= 0.0) {
                inside((-3.0 * b + std::sqrt(d)) / (10.0 * c));
                inside((-3.0 * b - std::sqrt(d)) / (10.0 * c));
            }
            shift = b / c;
            if (-0.5 * shift > 0.0 && -0.5 * shift < top) poly = std::fmax(poly, std::fabs(a - b * b / (4.0 * c)));
        } else if (b != 0.0) {
            inside(-a / (3.0 * b));
        }
        out.v[k] = scale_for(std::fmax(top, std::fmax(std::fabs(shift), std::fabs(top + shift))));
        out.b[k] = scale_for(poly);
        x = std::fmax(next, 1.0 / kMaxSpectrum);
        if (!(x <= kMaxSpectrum) || !(poly <= kMaxSpectrum * kMaxSpectrum)) return false;
        out.x[k + 1] = scale_for(x);
    }
    return true;
}

int32_t check(const D3gsOrthoMatrix* mats, int32_t count, const D3gsOrthoConfig* cfg, bool muon, Scales& scales, const char* what) {
    D3GS_REQUIRE(cfg != nullptr, "%s: cfg is NULL", what);
    D3GS_REQUIRE(count >= 0 && (count == 0 || mats != nullptr), "%s: %d matrices", what, count);
    D3GS_REQUIRE(cfg->dtype == D3GS_DTYPE_F32 || (cfg->dtype == D3GS_DTYPE_BF16 && !muon), "%s: dtype %d", what, cfg->dtype);
    D3GS_REQUIRE(cfg->steps >= 1 && cfg->steps <= D3GS_NS_MAX_STEPS, "%s: %d steps (1 to %d)", what, cfg->steps,
                 D3GS_NS_MAX_STEPS);
    D3GS_REQUIRE(cfg->eps > 0.0f, "%s: eps must be positive", what);
    D3GS_REQUIRE(scales_of(*cfg, scales), "%s: with these coefficients singular values grow past %g, or b / c does", what, kMaxSpectrum);
    for (int32_t i = 0; i < count; ++i) {
        const D3gsOrthoMatrix& m = mats[i];
        const int64_t small = m.rows < m.cols ? m.rows : m.cols, large = m.rows < m.cols ? m.cols : m.rows;
        D3GS_REQUIRE(small >= 0 && small <= kMaxShort && large <= kMaxLong && small * large < (int64_t)1 << 31,
                     "%s: matrix %d is %lld x %lld (short side at most %d, long side at most %d, below 2^31 values)", what, i,
                     (long long)m.rows, (long long)m.cols, kMaxShort, kMaxLong);
        if (small == 0) continue;
        D3GS_REQUIRE(m.src && m.dst && (!muon || m.momentum), "%s: matrix %d has a NULL pointer", what, i);
        D3GS_REQUIRE(m.rows <= 1 || m.src_row_stride >= 0, "%s: matrix %d has a negative stride", what, i);
    }
    return D3GS_OK;
}

// most: the most dynamic shared memory that any call of this kernel asks for (0: all ask for the same).  The attribute
// belongs to the kernel, not to the call: set to what a call needs, another thread's smaller call could lower it between
// this one's two steps.
template <typename K, typename... A>
int32_t launch(K kernel, const char* name, unsigned grid, unsigned threads, size_t smem, unsigned cluster, cudaStream_t st, size_t most,
               const A&... args) {
    if (smem > 48 * 1024) D3GS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(most ? most : smem)));
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(grid);
    c.blockDim = dim3(threads);
    c.dynamicSmemBytes = smem;
    c.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    c.attrs = attr;
    c.numAttrs = 2;
    D3GS_CUDA(cudaLaunchKernelEx(&c, kernel, args...));
    D3GS_LAUNCH_CHECK(name);
    return D3GS_OK;
}

template <int MODE, typename B> int32_t small_product(const Table& t, B& blocks, cudaStream_t st) {
    const unsigned tiles = blocks([](const Matrix& m) {
        return MODE == kApply ? (int64_t)m.mb * ((m.nk + 1) / 2) : (int64_t)m.mb * (m.mb + 1) / 2;
    });
    // X X^T: as many CTAs a tile as the machine has room for, none without four blocks to sum (one CTA a tile -> this:
    // 256 x 2304 250 -> 146 us, 64 x 1152 143 -> 104, 384 x 512 170 -> 156)
    unsigned parts = 1;
    if (MODE == kGram) {
        int longest = 0;
        for (int k = 0; k < t.count; ++k) longest = max(longest, t.mat[k].nk);
        while (parts < 8 && tiles * parts * 2 <= 148 && longest >= (int)parts * 2 * 4) parts *= 2;
    }
    return launch(ns_small_kernel<MODE>, "ns_small_kernel", tiles * parts, kSmallThreads, SmallStages::kBytes, parts, st, 0, t);
}
template <bool F32, int MODE, int RIGHT, typename B> int32_t pair_product(const Table& t, B& blocks, cudaStream_t st) {
    constexpr int L = Planes<F32, MODE, RIGHT>::kLeft;
    // 256 x 256 tiles move the least; 256 x 128 ones when those would leave SMs idle.  (256-wide from 40 CTAs on -> 100:
    // 2048 x 2048 719 -> 522 us, 8 x 2048 x 512 in 16 bits 314 -> 275; from 160 on -> 100: 2560 x 2560 1188 -> 1063 us,
    // 2048 x 2048 600 -> 522.)
    const unsigned tiles = blocks([](const Matrix& m) {
        const int64_t pairs = (m.mb + 1) / 2;
        return MODE == kApply ? pairs * ((m.nk + 3) / 4) : pairs * (pairs + 1) / 2;
    });
    if constexpr (MODE == kGram) {
        // Few tiles and a long axis: four or eight pairs a tile, with enough of the axis for each; two do not make up for
        // the way of the sums through memory.  One pair a tile -> this: 500 x 2600 302 -> 283 us, 1024 x 2304 350 -> 346,
        // 512 x 8192 610 -> 355, 512 x 32768 2126 -> 833; in 16 bits 1024 x 4096 259 -> 253, 512 x 8192 309 -> 227.  (From
        // twelve blocks a pair on, 24 in 16 bits, instead: 512 x 4608 317 instead of 297 us, in 16 bits 215 instead of 193.)
        Table u = t;
        int longest = 0;
        for (int k = 0; k < t.count; ++k) longest = max(longest, t.mat[k].nk);
        u.parts = 8;
        while (u.parts > 1 && ((int)tiles * 2 * u.parts > kTickets || longest < u.parts * (F32 ? kShare : 2 * kShare))) u.parts /= 2;
        if (u.parts >= 4)
            return launch(ns_pair_kernel<F32, MODE, RIGHT, 256, true>, "ns_pair_kernel", tiles * u.parts * 2, kPairThreads,
                          PairStages<L, RIGHT, 256>::kBytes, 2, st, 0, u);
    }
    if (tiles * 2 > 100)
        return launch(ns_pair_kernel<F32, MODE, RIGHT, 256>, "ns_pair_kernel", tiles * 2, kPairThreads,
                      PairStages<L, RIGHT, 256>::kBytes, 2, st, 0, t);
    const unsigned narrow = blocks([](const Matrix& m) {
        const int64_t pairs = (m.mb + 1) / 2;
        return MODE == kApply ? pairs * ((m.nk + 1) / 2) : pairs * (pairs + 1);
    });
    return launch(ns_pair_kernel<F32, MODE, RIGHT, 128>, "ns_pair_kernel", narrow * 2, kPairThreads,
                  PairStages<L, RIGHT, 128>::kBytes, 2, st, 0, t);
}
// one product of every matrix of the table; `blocks` writes its first_block; one: X is one value
template <bool F32, bool PAIR, int MODE, typename B> int32_t product(const Table& t, bool one, B& blocks, cudaStream_t st) {
    if constexpr (!PAIR) return small_product<MODE>(t, blocks, st);
    else if constexpr (F32) return pair_product<true, MODE, 2>(t, blocks, st);
    else if constexpr (MODE == kApply)
        return one ? pair_product<false, MODE, 1>(t, blocks, st) : pair_product<false, MODE, 2>(t, blocks, st);
    else return pair_product<false, MODE, 1>(t, blocks, st);
}

// The table of a batch, whose workspace begins at `at`.
void fill_table(Table& t, const Batch& b, bool muon, char* at) {
    t.fail = reinterpret_cast<uint32_t*>(at);
    t.tickets = reinterpret_cast<uint32_t*>(at + 256);
    t.sums = reinterpret_cast<float4*>(at + kHead);
    at += kHead + b.sums;
    for (t.count = 0; t.count < b.count;) {
        const D3gsOrthoMatrix& d = *b.mat[t.count];
        const Parts p = parts_of(d, b.planes);
        Matrix& m = t.mat[t.count++];
        m.src = d.src;
        m.momentum = muon ? d.momentum : nullptr;
        m.dst = d.dst;
        m.src_stride = d.src_row_stride;
        m.rows = (int32_t)d.rows;
        m.cols = (int32_t)d.cols;
        m.m = p.m;
        m.mb = p.mb;
        m.mk = p.mk;
        m.nk = p.nk;
        m.rounds = p.rounds;
        m.sums = p.sums;
        m.rate = d.rate;
        m.x[0] = at;
        m.x[1] = at + p.x;
        m.a = at + 2 * p.x;
        m.b = at + 2 * p.x + p.a;
        m.v = at + 2 * p.x + 2 * p.a;
        m.norms = reinterpret_cast<double*>(at + 2 * p.x + 2 * p.a + p.v) + 1;
        at += p.total;
    }
}

Steps steps_of(const D3gsOrthoConfig& cfg, const Scales& sc) {
    Steps sp{};
    sp.count = cfg.steps;
    sp.first = sc.x[0];
    sp.last = 1.0f / sc.x[cfg.steps];
    for (int s = 0; s < cfg.steps; ++s) {
        const double a = cfg.coefficients[s][0], b = cfg.coefficients[s][1], c = cfg.coefficients[s][2];
        const double sx = sc.x[s], sv = sc.v[s], sb = sc.b[s];
        if (c == 0.0) {   // the Gram product gives B
            sp.cubic |= 1u << s;
            sp.gram[s] = (float)(b * (sb / (sx * sx)));
            sp.gram_shift[s] = (float)(a * sb);
        } else {
            sp.gram[s] = (float)(sv / (sx * sx));
            sp.gram_shift[s] = (float)(b / c * sv);
            sp.square[s] = (float)(c * (sb / (sv * sv)));
            sp.square_shift[s] = (float)(a * sb);
        }
        sp.apply[s] = sc.x[s + 1] / sc.b[s] / sc.x[s];
    }
    return sp;
}

// Tiny matrices: one launch, a CTA each.
int32_t run_tiny(Table& t, const Steps& sp, cudaStream_t st) {
    int blocks = 0;
    for (int k = 0; k < t.count; ++k) blocks = max(blocks, t.mat[k].nk + 2 * t.mat[k].mk);
    return launch(ns_tiny_kernel, "ns_tiny_kernel", t.count, kTinyThreads, blocks * 2 * kPlane + 1024, 1, st,
                  kTinyBlocks * 2 * kPlane + 1024, t, sp);
}

template <bool F32, bool PAIR>
int32_t run_products(Table& t, const Steps& sp, cudaStream_t st) {
    auto blocks = [&](auto per) {
        int64_t b = 0;
        for (int k = 0; k < t.count; ++k) {
            t.first_block[k] = (int32_t)b;
            b += per(t.mat[k]);
        }
        t.first_block[t.count] = (int32_t)b;
        return (unsigned)b;
    };
    auto every_block = [](const Matrix& m) { return (int64_t)m.mb * m.nk; };
    t.from = 0;
    unsigned grid = blocks([](const Matrix& m) { return (int64_t)m.sums; });
    int rounds = 1;
    for (int k = 0; k < t.count; ++k) rounds = max(rounds, t.mat[k].rounds);
    if (int32_t rc = launch(rounds > 1 ? ns_norm_kernel<true> : ns_norm_kernel<false>, "ns_norm_kernel", grid, kThreads, 0, 1, st, 0, t)) return rc;
    t.out_scale = sp.first;
    t.exact = !F32;
    grid = blocks(every_block);
    if (int32_t rc = launch(ns_load_kernel, "ns_load_kernel", grid, kThreads, 0, 1, st, 0, t)) return rc;
    for (int s = 0; s < sp.count; ++s) {
        const bool one = s == 0 || s == sp.count - 1;
        t.exact = !F32 && s == 0;
        t.cubic = sp.cubic >> s & 1;
        t.out_scale = sp.gram[s];
        t.shift = sp.gram_shift[s];
        if (int32_t rc = product<F32, PAIR, kGram>(t, one, blocks, st)) return rc;
        if (!t.cubic) {
            t.out_scale = sp.square[s];
            t.shift = sp.square_shift[s];
            if (int32_t rc = product<F32, PAIR, kSquare>(t, one, blocks, st)) return rc;
        }
        t.out_scale = sp.apply[s];
        if (int32_t rc = product<F32, PAIR, kApply>(t, one, blocks, st)) return rc;
        t.from ^= 1;
    }
    t.out_scale = sp.last;
    grid = blocks(every_block);
    if (int32_t rc = launch(ns_store_kernel, "ns_store_kernel", grid, kThreads, 0, 1, st, 0, t)) return rc;
    return D3GS_OK;
}

int32_t entry(const D3gsOrthoMatrix* mats, int32_t count, const D3gsOrthoConfig* cfg, bool muon, void* ws, size_t ws_bytes,
              void* stream, const char* what) {
    Scales sc;
    if (int32_t rc = check(mats, count, cfg, muon, sc, what)) return rc;
    bool any = false;
    for (int32_t i = 0; i < count; ++i) any |= mats[i].rows > 0 && mats[i].cols > 0;
    if (!any) return D3GS_OK;
    D3GS_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= workspace_of(mats, count, *cfg),
                 "%s: workspace missing, unaligned or smaller than d3gs_orthogonalize_workspace_bytes", what);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const Steps sp = steps_of(*cfg, sc);
    char* const at = reinterpret_cast<char*>(up256((size_t)(uintptr_t)ws));
    Table t{};
    t.bf16 = cfg->dtype == D3GS_DTYPE_BF16;
    t.eps = cfg->eps;
    t.mu = (float)cfg->momentum;
    t.fresh = (float)(1.0 - cfg->momentum);
    t.nesterov = cfg->nesterov;
    t.decay = cfg->decay;
    t.hooks = test_hooks();
    List list{mats, count, cfg->dtype};
    Batch b;
    while (next_batch(list, b)) {
        fill_table(t, b, muon, at);
        const int32_t rc = b.way == kTiny                  ? run_tiny(t, sp, st)
                           : b.way == kSmall               ? run_products<true, false>(t, sp, st)
                           : cfg->dtype == D3GS_DTYPE_F32 ? run_products<true, true>(t, sp, st)
                                                           : run_products<false, true>(t, sp, st);
        if (rc) return rc;
    }
    return D3GS_OK;
}

}  // namespace
}  // namespace d3gs

using namespace d3gs;

extern "C" size_t d3gs_orthogonalize_workspace_bytes(const D3gsOrthoMatrix* matrices, int32_t count,
                                                     const D3gsOrthoConfig* cfg) {
    Scales sc;
    if (check(matrices, count, cfg, false, sc, "d3gs_orthogonalize_workspace_bytes") != D3GS_OK) return 0;
    return workspace_of(matrices, count, *cfg);
}

extern "C" int32_t d3gs_orthogonalize(const D3gsOrthoMatrix* matrices, int32_t count, const D3gsOrthoConfig* cfg,
                                      void* workspace, size_t workspace_bytes, void* stream) {
    return entry(matrices, count, cfg, false, workspace, workspace_bytes, stream, "d3gs_orthogonalize");
}

extern "C" int32_t d3gs_muon_step(const D3gsOrthoMatrix* matrices, int32_t count, const D3gsOrthoConfig* cfg,
                                  void* workspace, size_t workspace_bytes, void* stream) {
    return entry(matrices, count, cfg, true, workspace, workspace_bytes, stream, "d3gs_muon_step");
}

// Orthogonalised updates of weight matrices by Newton-Schulz products, and the optimizer step around them.
//
//   U = the update (given, or momentum buffer and gradient joined), X = U / max(|U|_F, eps), the short side first
//   each step: A = X X^T,  B = a I + b A + c A A,  X <- B X
//   result X, or param <- decay param - rate X
//
// All matrices of a call go through the same launches: a table in the kernel arguments maps CTAs to matrices.
//
// The products run on the tensor cores (tcgen05, 32-bit sums in TMEM).  Their operands are fp16 with a power-of-two
// scale: X, A and B have bounded spectra (the bounds follow from the coefficients), so the 2^29 of fp16's normal range
// hold every entry that matters.  16-bit matrices use one fp16 value per entry (11 bits: their result is rounded to 8).
// 32-bit matrices use two, v = hi + lo (22 bits), and three products hi hi + hi lo + lo hi; the dropped lo lo is of the
// size of the last bit.  (Two bf16 values would hold 16 bits only, and three of them need six products.)
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

constexpr int kMaxMatrices = 64;   // per launch; longer lists are cut
constexpr int kThreads = 256;
constexpr int kNormChunk = 8192;   // values per CTA of the norm pass
constexpr int kMaxShort = 16384, kMaxLong = 1 << 24;
constexpr int kRows = 128, kCols = 64;                 // one block
constexpr uint32_t kPlane = kRows * kCols * 2;         // bytes of one fp16 plane of a block
constexpr float kMaxSpectrum = 1024.0f;                // largest singular value the scales leave room for

struct Matrix {
    const void* src;
    float* momentum;
    void* dst;
    int64_t src_stride;   // values between rows
    char *x[2], *a, *b;   // blocks of X (two buffers), A, B
    double* norms;        // sums of squares of the norm pass
    int32_t rows, cols;
    int32_t m, n;         // short and long side
    int32_t mb, mk, nk;   // blocks: rows of all three, columns of A and B, columns of X
    float rate;
};
struct Table {
    Matrix mat[kMaxMatrices];
    int32_t first_block[kMaxMatrices + 1];
    int32_t count;
    int32_t bf16;         // src and dst type (momentum and parameters are always 32 bits)
    float eps, mu, decay;
    int32_t nesterov;
    int32_t from;         // which of x[] holds X
    float ca, cb, cc;     // this step's coefficients, by the scales of what they multiply (see scales_of)
    float out_scale;      // of a product's result; of X in the first and the last pass
    uint32_t* fail;       // set when a bounded wait ran out: the last pass then writes NaN
    TestHooks hooks;
};

// the matrix a CTA belongs to, and its number within it
__device__ __forceinline__ int find_matrix(const Table& t, int& block) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((int)blockIdx.x >= t.first_block[mid]) lo = mid;
        else hi = mid - 1;
    }
    block = (int)blockIdx.x - t.first_block[lo];
    return lo;
}

__device__ __forceinline__ float load_src(const Table& t, const Matrix& m, int64_t r, int64_t c) {
    const int64_t i = r * m.src_stride + c;
    return t.bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(m.src)[i]) : static_cast<const float*>(m.src)[i];
}
// the update from gradient and NEW momentum
__device__ __forceinline__ float update_of(const Table& t, float g, float buf) {
    return t.nesterov ? fmaf(t.mu, buf, (1.0f - t.mu) * g) : buf;
}

// ---- new momentum, and the sum of squares of the update (in 64 bits: no value of a float overflows it) -----------
__global__ void __launch_bounds__(kThreads) ns_norm_kernel(const __grid_constant__ Table t) {
    __shared__ double s[kThreads / 32];
    if (blockIdx.x == 0 && threadIdx.x == 0) *t.fail = 0;
    int block;
    const Matrix& m = t.mat[find_matrix(t, block)];
    const int64_t count = (int64_t)m.rows * m.cols, i0 = (int64_t)block * kNormChunk, i1 = min(count, i0 + kNormChunk);
    double sum = 0.0;
    for (int64_t i = i0 + threadIdx.x; i < i1; i += kThreads) {
        float u = load_src(t, m, i / m.cols, i % m.cols);
        if (m.momentum) {
            const float buf = fmaf(t.mu, m.momentum[i], (1.0f - t.mu) * u);
            m.momentum[i] = buf;
            u = update_of(t, u, buf);
        }
        sum += (double)u * (double)u;
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

// every CTA adds the sums up itself, in the same order
__device__ __forceinline__ float inverse_norm(const Table& t, const Matrix& m) {
    __shared__ double s[kThreads / 32];
    const int n = (int)(((int64_t)m.rows * m.cols + kNormChunk - 1) / kNormChunk);
    double sum = 0.0;
    for (int i = threadIdx.x; i < n; i += kThreads) sum += m.norms[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = 0.0;
    for (int k = 0; k < kThreads / 32; ++k) sum += s[k];
    const double norm = sqrt(sum);
    return (float)(1.0 / (norm < (double)t.eps ? (double)t.eps : norm));   // a NaN stays one
}

// byte of value (r, c) in a plane of a block
__device__ __forceinline__ uint32_t block_offset(uint32_t r, uint32_t c) {
    return r * 128u + (((c >> 3) ^ (r & 7u)) << 4) + (c & 7u) * 2u;
}
// v = hi + lo with 22 bits; lo takes what hi's rounding left
__device__ __forceinline__ void split(float v, __half& hi, __half& lo) {
    hi = __float2half_rn(v);
    lo = __float2half_rn(v - __half2float(hi));
}
__device__ __forceinline__ uint32_t pack(__half a, __half b) {
    return (uint32_t)__half_as_ushort(a) | ((uint32_t)__half_as_ushort(b) << 16);
}

// ---- first pass: blocks of X = U / norm, transposed when the matrix is tall; one CTA per block --------------------
template <int PLANES> __global__ void __launch_bounds__(kThreads) ns_load_kernel(const __grid_constant__ Table t) {
    __shared__ __align__(16) uint32_t s[PLANES * kPlane / 4];
    int block;
    const Matrix& m = t.mat[find_matrix(t, block)];
    const float inv = inverse_norm(t, m);
    const bool tall = m.rows > m.cols;
    const int r0 = block / m.nk * kRows, c0 = block % m.nk * kCols;
    // two neighbouring columns of X a thread; neighbouring threads along the rows of U
    for (int i = threadIdx.x; i < kRows * kCols / 2; i += kThreads) {
        const int r = tall ? i % kRows : i / (kCols / 2), c = (tall ? i / kRows : i % (kCols / 2)) * 2;
        float v[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int64_t xr = r0 + r, xc = c0 + c + k;
            v[k] = 0.0f;
            if (xr < m.m && xc < m.n) {
                const int64_t ur = tall ? xc : xr, uc = tall ? xr : xc;
                float u = load_src(t, m, ur, uc);
                if (m.momentum) u = update_of(t, u, m.momentum[ur * m.cols + uc]);
                v[k] = u * inv * t.out_scale;
            }
        }
        __half h[2], l[2];
        split(v[0], h[0], l[0]);
        split(v[1], h[1], l[1]);
        const uint32_t o = block_offset(r, c) / 4;
        s[o] = pack(h[0], h[1]);
        if (PLANES == 2) s[kPlane / 4 + o] = pack(l[0], l[1]);
    }
    __syncthreads();
    uint4* out = reinterpret_cast<uint4*>(m.x[0] + (int64_t)block * PLANES * kPlane);
    for (int i = threadIdx.x; i < PLANES * (int)kPlane / 16; i += kThreads) out[i] = reinterpret_cast<const uint4*>(s)[i];
}

// ---- last pass: result or parameter from the blocks of X; one CTA per block ---------------------------------------
template <int PLANES> __global__ void __launch_bounds__(kThreads) ns_store_kernel(const __grid_constant__ Table t) {
    int block;
    const Matrix& m = t.mat[find_matrix(t, block)];
    const bool tall = m.rows > m.cols, failed = *t.fail != 0;
    const int r0 = block / m.nk * kRows, c0 = block % m.nk * kCols;
    const char* x = m.x[t.from] + (int64_t)block * PLANES * kPlane;
    for (int i = threadIdx.x; i < kRows * kCols / 2; i += kThreads) {
        const int r = tall ? i % kRows : i / (kCols / 2), c = (tall ? i / kRows : i % (kCols / 2)) * 2;
        const uint32_t o = block_offset(r, c);
        const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(x + o));
        const float2 lo = PLANES == 2 ? __half22float2(*reinterpret_cast<const __half2*>(x + kPlane + o)) : make_float2(0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int64_t xr = r0 + r, xc = c0 + c + k;
            if (xr >= m.m || xc >= m.n) continue;
            const int64_t j = tall ? xc * m.cols + xr : xr * m.cols + xc;
            float v = (k ? hi.y + lo.y : hi.x + lo.x) * t.out_scale;
            if (failed) v = __int_as_float(0x7fffffff);
            if (m.momentum) {
                float* p = static_cast<float*>(m.dst) + j;
                *p = fmaf(-m.rate, v, t.decay * *p);
            } else if (t.bf16) {
                static_cast<__nv_bfloat16*>(m.dst)[j] = __float2bfloat16_rn(v);
            } else {
                static_cast<float*>(m.dst)[j] = v;
            }
        }
    }
}

// ---- tcgen05 ------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t* out, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(out)), "r"(cols) : "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t cols) {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(cols));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
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
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void bulk_wait_group0() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Shared-memory operand in 128-byte rows with the 16-byte pieces exchanged (swizzle mode 2).  Summed along the rows:
// eight rows are 1024 bytes apart (`group`), `next` is not used.  Summed across the rows: `group` is the distance of
// the next eight summed rows, `next` that of the next 64 columns.
__device__ __forceinline__ uint64_t operand(uint32_t at, uint32_t next, uint32_t group) {
    return (uint64_t)((at >> 4) & 0x3fffu) | ((uint64_t)(next >> 4) << 16) | ((uint64_t)(group >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}

// ---- products: one 128 x 128 tile a CTA ---------------------------------------------------------------------------
// Warp 4 brings in operand tiles by bulk copies, warp 5 issues the products, warps 0-3 (one TMEM quarter each) take the
// sums out.  The tensor cores cut the last bits of a running sum at every step (towards zero, so that the losses add
// up; 2e-5 of the result at 1025 x 515 when nothing is done about it).  With PLANES == 2 the sums of hi hi are therefore
// taken out every kRunBlocks column blocks and added in registers (rounded), the products going to another part of TMEM
// meanwhile; hi lo + lo hi, 2^-11 of their size, have a sum of their own that is taken out once.
// A and B are symmetric: only tiles on and above the diagonal are computed, and written twice.  Rows behind the last
// column block of A and B hold anything: nothing sums over them, and no valid row or column reads them.
enum { kGram = 0, kSquare = 1, kApply = 2 };
constexpr int kGemmThreads = 192, kTile = 128, kRunBlocks = 2;
template <int PLANES> struct Stages {
    static constexpr uint32_t kOperand = PLANES * kPlane, kStage = 2 * kOperand;
    static constexpr int kCount = PLANES == 2 ? 3 : 6;
    static constexpr uint32_t kBytes = kCount * kStage + 1024;   // alignment to 1024
    static constexpr uint32_t kTmem = PLANES == 2 ? 512 : 128;   // columns: two sums of hi hi, one of the rest; one sum
};

template <int PLANES, int MODE>
__global__ void __launch_bounds__(kGemmThreads, 1) ns_gemm_kernel(const __grid_constant__ Table t) {
    using S = Stages<PLANES>;
    extern __shared__ char raw[];
    __shared__ uint64_t s_full[S::kCount], s_empty[S::kCount], s_sum[2], s_taken[2], s_drain;
    __shared__ uint32_t s_tmem;
    char* const smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int block;
    const Matrix& m = t.mat[find_matrix(t, block)];
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
    const int blocks = MODE == kGram ? m.nk : m.mk;    // summed over
    const int run = PLANES == 2 ? kRunBlocks : blocks, runs = (blocks + run - 1) / run;
    const uint32_t polls = t.hooks.poll_limit;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kCount; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_sum[i], 1);
            mbar_init(&s_taken[i], 128);
        }
        mbar_init(&s_drain, 1);
        fence_mbar_init();
    }
    if (warp == 5) tmem_alloc(&s_tmem, S::kTmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    bool ok = true;

    if (warp == 4) {
        if (lane == 0) {
            int k = 0;
            for (; k < blocks && ok; ++k) {
                const int st = k % S::kCount;
                if (k >= S::kCount) ok = mbar_wait_bounded(&s_empty[st], (k / S::kCount - 1) & 1, polls);
                if (!ok) break;
                char* const a = smem + st * S::kStage;
                char* const b = a + S::kOperand;
                if (t.hooks.hold == (int)blockIdx.x && k == 0) continue;   // a test: this copy never comes
                if (MODE == kApply) {
                    const int wide = 2 * tj + 1 < m.nk ? 2 : 1;            // the last tile may be one block wide
                    mbar_arrive_expect_tx(&s_full[st], S::kOperand + PLANES * wide * (kPlane / 2));
                    bulk_copy_g2s(a, left + ((int64_t)ti * m.mk + k) * S::kOperand, S::kOperand, &s_full[st]);
                    for (int p = 0; p < PLANES; ++p)
                        for (int w = 0; w < wide; ++w)                     // 64 rows of a block: one half of a plane
                            bulk_copy_g2s(b + (p * 2 + w) * (kPlane / 2),
                                          right + ((int64_t)(k >> 1) * m.nk + 2 * tj + w) * S::kOperand + p * kPlane +
                                              (k & 1) * (kPlane / 2),
                                          kPlane / 2, &s_full[st]);
                } else {
                    mbar_arrive_expect_tx(&s_full[st], same ? S::kOperand : S::kStage);
                    bulk_copy_g2s(a, left + ((int64_t)ti * blocks + k) * S::kOperand, S::kOperand, &s_full[st]);
                    if (!same) bulk_copy_g2s(b, right + ((int64_t)tj * blocks + k) * S::kOperand, S::kOperand, &s_full[st]);
                }
            }
            if (!ok)   // given up: what is on its way has to land before the CTA ends
                for (int j = k > S::kCount ? k - S::kCount : 0; j < k; ++j)
                    mbar_wait_bounded(&s_full[j % S::kCount], (j / S::kCount) & 1, polls);
        }
    } else if (warp == 5) {
        if (lane == 0) {
            // D 32 bits, A and B fp16; in B X the right factor is summed across its rows (bit 16)
            const uint32_t idesc = (1u << 4) | ((MODE == kApply ? 1u : 0u) << 16) | ((kTile / 8u) << 17) | ((128u / 16u) << 24);
            for (int k = 0; k < blocks && ok; ++k) {
                const int st = k % S::kCount, r = k / run, half = r & 1;
                if (k % run == 0 && r >= 2) ok = mbar_wait_bounded(&s_taken[half], (r / 2 - 1) & 1, polls);
                if (ok) ok = mbar_wait_bounded(&s_full[st], (k / S::kCount) & 1, polls);
                if (!ok) break;
                tc_fence_after();
                const uint32_t a = smem_u32(smem + st * S::kStage), b = same ? a : a + S::kOperand;
                const uint32_t d = tmem + half * kTile;
#pragma unroll
                for (int q = 0; q < kCols / 16; ++q) {
                    const bool add = k % run != 0 || q != 0;
                    uint64_t da[PLANES], db[PLANES];
#pragma unroll
                    for (int p = 0; p < PLANES; ++p) {
                        da[p] = operand(a + p * kPlane + q * 32, 16, 1024);
                        db[p] = MODE == kApply ? operand(b + p * kPlane + q * 2048, kPlane / 2, 1024)
                                               : operand(b + p * kPlane + q * 32, 16, 1024);
                    }
                    tc_mma(d, da[0], db[0], idesc, add);
                    if (PLANES == 2) {
                        tc_mma(tmem + 2 * kTile, da[0], db[PLANES - 1], idesc, k != 0 || q != 0);
                        tc_mma(tmem + 2 * kTile, da[PLANES - 1], db[0], idesc, true);
                    }
                }
                tc_commit(&s_empty[st]);
                if (k % run == run - 1 || k == blocks - 1) tc_commit(&s_sum[half]);
            }
            if (!ok) {   // given up: the products that were issued end before TMEM is handed back
                tc_commit(&s_drain);
                mbar_wait_bounded(&s_drain, 0, polls);
            }
        }
    } else {
        float v[kTile];
#pragma unroll
        for (int c = 0; c < kTile; ++c) v[c] = 0.0f;
        for (int r = 0; r < runs && ok; ++r) {
            ok = __all_sync(~0u, mbar_wait_bounded(&s_sum[r & 1], (r / 2) & 1, polls));
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < kTile; c += 32) {
                float w[32];
                tmem_load32(tmem + (r & 1) * kTile + c + ((uint32_t)warp << 21), w);
#pragma unroll
                for (int i = 0; i < 32; ++i) v[c + i] += w[i];
            }
            if (PLANES == 2 && r == runs - 1) {
#pragma unroll
                for (int c = 0; c < kTile; c += 32) {
                    float w[32];
                    tmem_load32(tmem + 2 * kTile + c + ((uint32_t)warp << 21), w);
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[c + i] += w[i];
                }
            }
            tc_fence_before();
            mbar_arrive(&s_taken[r & 1]);
        }
        // every product has read its operands by now: their shared memory takes the finished tile
        const uint32_t r = threadIdx.x;
        const int wide = MODE == kApply ? m.nk : m.mk;   // blocks across the result
        char* const out = MODE == kGram ? m.a : MODE == kSquare ? m.b : m.x[t.from ^ 1];
        if (ok) {
#pragma unroll
            for (int c = 0; c < kTile; c += 8) {
                if (2 * tj + c / kCols >= wide) continue;
                const uint32_t o = (c / kCols) * S::kOperand + block_offset(r, c % kCols);
                float old[8];
                if (MODE == kSquare) {
                    const char* a = m.a + ((int64_t)ti * m.mk + 2 * tj) * S::kOperand + o;
                    const uint4 h = *reinterpret_cast<const uint4*>(a);
                    const uint4 l = PLANES == 2 ? *reinterpret_cast<const uint4*>(a + kPlane) : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 f = __half22float2(reinterpret_cast<const __half2*>(&h)[i]);
                        const float2 g = __half22float2(reinterpret_cast<const __half2*>(&l)[i]);
                        old[2 * i] = f.x + g.x;
                        old[2 * i + 1] = f.y + g.y;
                    }
                }
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    __half h[2], l[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float f = v[c + i + j];
                        if (MODE == kSquare) {
                            f = fmaf(t.cc, f, t.cb * old[i + j]);
                            if (same && (int)r == c + i + j && ti * kRows + (int)r < m.m) f += t.ca;
                        } else {
                            f *= t.out_scale;
                        }
                        split(f, h[j], l[j]);
                        if (MODE != kApply && !same) {   // the mirrored tile: this thread's row is a column
                            const uint32_t w = 2 * S::kOperand + (r / kCols) * S::kOperand + block_offset(c + i + j, r % kCols);
                            *reinterpret_cast<__half*>(smem + w) = h[j];
                            if (PLANES == 2) *reinterpret_cast<__half*>(smem + w + kPlane) = l[j];
                        }
                    }
                    hi[i / 2] = pack(h[0], h[1]);
                    lo[i / 2] = pack(l[0], l[1]);
                }
                *reinterpret_cast<uint4*>(smem + o) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if (PLANES == 2) *reinterpret_cast<uint4*>(smem + o + kPlane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
            fence_proxy_async_smem();
        } else {
            *t.fail = 1;
        }
        const bool all = __syncthreads_and(ok);   // (the other two warps join below)
        if (all && threadIdx.x == 0) {
            for (int c = 0; c < 2; ++c) {
                if (2 * tj + c < wide)
                    bulk_copy_s2g(out + ((int64_t)ti * wide + 2 * tj + c) * S::kOperand, smem + c * S::kOperand, S::kOperand);
                if (MODE != kApply && !same && 2 * ti + c < wide)
                    bulk_copy_s2g(out + ((int64_t)tj * wide + 2 * ti + c) * S::kOperand, smem + (2 + c) * S::kOperand, S::kOperand);
            }
            bulk_commit_group();
            bulk_wait_group0();
        }
    }
    if (warp >= 4) {
        if (!ok) *t.fail = 1;
        __syncwarp();
        (void)__syncthreads_and(ok);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 5) tmem_free(tmem, S::kTmem);
}

// ---- host ---------------------------------------------------------------------------------------------------------
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

struct Parts {
    int m, n, mb, mk, nk;
    size_t x, a, norms, total;   // bytes
};
Parts parts_of(const D3gsOrthoMatrix& d, int planes) {
    Parts p;
    p.m = (int)(d.rows < d.cols ? d.rows : d.cols);
    p.n = (int)(d.rows < d.cols ? d.cols : d.rows);
    p.mb = (p.m + kRows - 1) / kRows;
    p.mk = (p.m + kCols - 1) / kCols;
    p.nk = (p.n + kCols - 1) / kCols;
    p.x = (size_t)p.mb * p.nk * planes * kPlane;
    p.a = (size_t)p.mb * p.mk * planes * kPlane;
    p.norms = up256((size_t)div_up64(d.rows * d.cols, kNormChunk) * 8);
    p.total = p.m == 0 ? 0 : 2 * p.x + 2 * p.a + p.norms;
    return p;
}
int planes_of(const D3gsOrthoConfig& cfg) { return cfg.dtype == D3GS_DTYPE_F32 ? 2 : 1; }
size_t workspace_of(const D3gsOrthoMatrix* mats, int32_t count, const D3gsOrthoConfig& cfg) {
    size_t need = 512;   // alignment, the failure word
    for (int32_t i = 0; i < count; ++i) need += parts_of(mats[i], planes_of(cfg)).total;
    return need;
}

// Scales of the operands.  The singular values of X lie in [0, s]: s = 1 at the start, and after a step the largest
// |a x + b x^3 + c x^5| over [0, s], found at s or where the derivative a + 3 b x^2 + 5 c x^4 vanishes.  No entry of X
// exceeds s, none of A s^2, none of B the largest |a + b y + c y^2| over y in [0, s^2].  Each is scaled to at most 2^15
// by a power of two, so that scaling loses nothing.
struct Scales {
    float x[D3GS_NS_MAX_STEPS + 1], a[D3GS_NS_MAX_STEPS], b[D3GS_NS_MAX_STEPS];
};
float scale_for(double most) {
    int e;
    std::frexp(most * 1.001, &e);   // most * 1.001 <= 2^e
    return std::ldexp(1.0f, 15 - e);
}
bool scales_of(const D3gsOrthoConfig& cfg, Scales& out) {
    double s = 1.0;
    out.x[0] = scale_for(s);
    for (int k = 0; k < cfg.steps; ++k) {
        const double a = cfg.coefficients[k][0], b = cfg.coefficients[k][1], c = cfg.coefficients[k][2], top = s * s;
        auto f = [&](double y) { return std::fabs(std::sqrt(y) * (a + y * (b + y * c))); };
        double next = f(top), poly = std::fmax(std::fabs(a), std::fabs(a + top * (b + top * c)));
        auto inside = [&](double y) {
            if (y > 0.0 && y < top) next = std::fmax(next, f(y));
        };
        if (c != 0.0) {
            const double d = 9.0 * b * b - 20.0 * a * c;
            if (d >= 0.0) {
                inside((-3.0 * b + std::sqrt(d)) / (10.0 * c));
                inside((-3.0 * b - std::sqrt(d)) / (10.0 * c));
            }
            const double v = -b / (2.0 * c);
            if (v > 0.0 && v < top) poly = std::fmax(poly, std::fabs(a + v * (b + v * c)));
        } else if (b != 0.0) {
            inside(-a / (3.0 * b));
        }
        out.a[k] = scale_for(top);
        out.b[k] = scale_for(std::fmax(poly, 1.0 / kMaxSpectrum));
        s = std::fmax(next, 1.0 / kMaxSpectrum);   // coefficients of zeros: any scale holds a zero
        if (!(s <= kMaxSpectrum) || !(poly <= kMaxSpectrum * kMaxSpectrum)) return false;
        out.x[k + 1] = scale_for(s);
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
    D3GS_REQUIRE(scales_of(*cfg, scales), "%s: with these coefficients singular values grow past %g", what, kMaxSpectrum);
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

template <int PLANES, int MODE> int32_t launch_product(const Table& t, unsigned grid, cudaStream_t st) {
    D3GS_CUDA(cudaFuncSetAttribute(ns_gemm_kernel<PLANES, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)Stages<PLANES>::kBytes));
    ns_gemm_kernel<PLANES, MODE><<<grid, kGemmThreads, Stages<PLANES>::kBytes, st>>>(t);
    D3GS_LAUNCH_CHECK("ns_gemm_kernel");
    return D3GS_OK;
}

template <int PLANES>
int32_t run(const D3gsOrthoMatrix* mats, int32_t count, const D3gsOrthoConfig& cfg, bool muon, const Scales& sc, void* ws,
            cudaStream_t st) {
    char* at = reinterpret_cast<char*>(up256((size_t)(uintptr_t)ws));
    Table t{};
    t.fail = reinterpret_cast<uint32_t*>(at);
    at += 256;
    t.bf16 = cfg.dtype == D3GS_DTYPE_BF16;
    t.eps = cfg.eps;
    t.mu = cfg.momentum;
    t.nesterov = cfg.nesterov;
    t.decay = cfg.decay;
    t.hooks = test_hooks();
    int32_t i = 0;
    while (i < count) {
        t.count = 0;
        for (; i < count && t.count < kMaxMatrices; ++i) {
            const D3gsOrthoMatrix& d = mats[i];
            if (d.rows == 0 || d.cols == 0) continue;
            const Parts p = parts_of(d, PLANES);
            Matrix& m = t.mat[t.count++];
            m.src = d.src;
            m.momentum = muon ? d.momentum : nullptr;
            m.dst = d.dst;
            m.src_stride = d.src_row_stride;
            m.rows = (int32_t)d.rows;
            m.cols = (int32_t)d.cols;
            m.m = p.m;
            m.n = p.n;
            m.mb = p.mb;
            m.mk = p.mk;
            m.nk = p.nk;
            m.rate = d.rate;
            m.x[0] = at;
            m.x[1] = at + p.x;
            m.a = at + 2 * p.x;
            m.b = at + 2 * p.x + p.a;
            m.norms = reinterpret_cast<double*>(at + 2 * p.x + 2 * p.a);
            at += p.total;
        }
        if (t.count == 0) break;
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
        unsigned grid = blocks([](const Matrix& m) { return div_up64((int64_t)m.rows * m.cols, kNormChunk); });
        ns_norm_kernel<<<grid, kThreads, 0, st>>>(t);
        D3GS_LAUNCH_CHECK("ns_norm_kernel");
        t.out_scale = sc.x[0];
        grid = blocks(every_block);
        ns_load_kernel<PLANES><<<grid, kThreads, 0, st>>>(t);
        D3GS_LAUNCH_CHECK("ns_load_kernel");
        for (int s = 0; s < cfg.steps; ++s) {
            grid = blocks([](const Matrix& m) { return (int64_t)m.mb * (m.mb + 1) / 2; });
            t.out_scale = sc.a[s] / (sc.x[s] * sc.x[s]);
            if (int32_t rc = launch_product<PLANES, kGram>(t, grid, st)) return rc;
            t.ca = cfg.coefficients[s][0] * sc.b[s];
            t.cb = cfg.coefficients[s][1] * (sc.b[s] / sc.a[s]);
            t.cc = cfg.coefficients[s][2] * (sc.b[s] / sc.a[s] / sc.a[s]);
            if (int32_t rc = launch_product<PLANES, kSquare>(t, grid, st)) return rc;
            t.out_scale = sc.x[s + 1] / sc.b[s] / sc.x[s];
            grid = blocks([](const Matrix& m) { return (int64_t)m.mb * ((m.nk + 1) / 2); });
            if (int32_t rc = launch_product<PLANES, kApply>(t, grid, st)) return rc;
            t.from ^= 1;
        }
        t.out_scale = 1.0f / sc.x[cfg.steps];
        grid = blocks(every_block);
        ns_store_kernel<PLANES><<<grid, kThreads, 0, st>>>(t);
        D3GS_LAUNCH_CHECK("ns_store_kernel");
    }
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
    return planes_of(*cfg) == 2 ? run<2>(mats, count, *cfg, muon, sc, ws, st) : run<1>(mats, count, *cfg, muon, sc, ws, st);
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

// Orthogonalised updates of weight matrices by Newton-Schulz products, and the optimizer step around them.
//
//   U = the update (given, or momentum buffer and gradient joined), X = U / max(|U|_F, eps), the short side first
//   each step: A = X X^T,  B = b A + c A A,  X <- a X + B X
//   result X, or param <- decay param - rate X
//
// All matrices of a call go through the same launches: a table in the kernel arguments maps CTAs to matrices.
#include <cuda_bf16.h>

#include "common.cuh"

namespace d3gs {
namespace {

constexpr int kMaxMatrices = 64;   // per launch; longer lists are cut
constexpr int kThreads = 256;
constexpr int kNormChunk = 8192;   // values per CTA of the norm pass
constexpr int kTile = 64;
constexpr int kMaxShort = 16384, kMaxLong = 1 << 24;

struct Matrix {
    const void* src;
    float* momentum;
    void* dst;
    int64_t src_stride;   // values between rows
    float *x[2], *a, *b;  // X (two buffers), A, B
    double* norms;        // sums of squares of the norm pass
    int32_t rows, cols;
    int32_t m, n;         // short and long side
    float rate;
};
struct Table {
    Matrix mat[kMaxMatrices];
    int32_t first_block[kMaxMatrices + 1];
    int32_t count;
    int32_t bf16;         // src and dst type (momentum and parameters are always 32 bits)
    float eps, mu, decay;
    int32_t nesterov;
    float ca, cb, cc;     // this step's coefficients
    int32_t from;         // which of x[] holds X
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

// ---- X = U / norm, transposed when the matrix is tall -------------------------------------------------------------
__global__ void __launch_bounds__(kThreads) ns_load_kernel(const __grid_constant__ Table t) {
    int block;
    const Matrix& m = t.mat[find_matrix(t, block)];
    const float inv = inverse_norm(t, m);
    const int64_t count = (int64_t)m.rows * m.cols, i0 = (int64_t)block * kNormChunk, i1 = min(count, i0 + kNormChunk);
    for (int64_t i = i0 + threadIdx.x; i < i1; i += kThreads) {
        const int64_t r = i / m.cols, c = i % m.cols;
        float u = load_src(t, m, r, c);
        if (m.momentum) u = update_of(t, u, m.momentum[i]);
        m.x[0][m.rows > m.cols ? c * m.n + r : i] = u * inv;
    }
}

// ---- result -------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(kThreads) ns_store_kernel(const __grid_constant__ Table t) {
    int block;
    const Matrix& m = t.mat[find_matrix(t, block)];
    const int64_t count = (int64_t)m.rows * m.cols, i0 = (int64_t)block * kNormChunk, i1 = min(count, i0 + kNormChunk);
    for (int64_t i = i0 + threadIdx.x; i < i1; i += kThreads) {
        const int64_t r = i / m.cols, c = i % m.cols;
        const float x = m.x[t.from][m.rows > m.cols ? c * m.n + r : i];
        if (m.momentum) {
            float* p = static_cast<float*>(m.dst) + i;
            *p = fmaf(-m.rate, x, t.decay * *p);
        } else if (t.bf16) {
            static_cast<__nv_bfloat16*>(m.dst)[i] = __float2bfloat16_rn(x);
        } else {
            static_cast<float*>(m.dst)[i] = x;
        }
    }
}

// ---- products: out = P Q (or P Q^T) with an epilogue, 64 x 64 tiles, 4 x 4 values a thread ------------------------
enum { kGram = 0, kSquare = 1, kApply = 2 };
template <int MODE> __global__ void __launch_bounds__(kThreads) ns_gemm_kernel(const __grid_constant__ Table t) {
    __shared__ float sp[16][kTile + 1], sq[16][kTile + 1];
    int block;
    const Matrix& m = t.mat[find_matrix(t, block)];
    const int nn = MODE == kApply ? m.n : m.m, kk = MODE == kGram ? m.n : m.m;
    const int tiles_n = (nn + kTile - 1) / kTile;
    const int r0 = block / tiles_n * kTile, c0 = block % tiles_n * kTile;
    const float* x = m.x[t.from];
    const float* P = MODE == kGram ? x : MODE == kSquare ? m.a : m.b;
    const float* Q = MODE == kGram ? x : MODE == kSquare ? m.a : x;
    const int ldp = MODE == kGram ? m.n : m.m, ldq = MODE == kSquare ? m.m : m.n;
    const int tr = threadIdx.x / 16 * 4, tc = threadIdx.x % 16 * 4;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < kk; k0 += 16) {
        for (int i = threadIdx.x; i < 16 * kTile; i += kThreads) {
            const int k = i % 16, r = i / 16;
            sp[k][r] = r0 + r < m.m && k0 + k < kk ? P[(int64_t)(r0 + r) * ldp + k0 + k] : 0.0f;
            if (MODE != kApply) sq[k][r] = c0 + r < nn && k0 + k < kk ? Q[(int64_t)(c0 + r) * ldq + k0 + k] : 0.0f;
        }
        if (MODE == kApply)
            for (int i = threadIdx.x; i < 16 * kTile; i += kThreads) {
                const int c = i % kTile, k = i / kTile;
                sq[k][c] = c0 + c < nn && k0 + k < kk ? Q[(int64_t)(k0 + k) * ldq + c0 + c] : 0.0f;
            }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sp[k][tr + i], sq[k][tc + j], acc[i][j]);
        __syncthreads();
    }
    float* out = MODE == kGram ? m.a : MODE == kSquare ? m.b : m.x[t.from ^ 1];
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int r = r0 + tr + i, c = c0 + tc + j;
            if (r >= m.m || c >= nn) continue;
            const int64_t o = (int64_t)r * nn + c;
            float v = acc[i][j];
            if (MODE == kSquare) v = fmaf(t.cc, v, t.cb * m.a[o]);
            if (MODE == kApply) v = fmaf(t.ca, x[o], v);
            out[o] = v;
        }
}

// ---- host ---------------------------------------------------------------------------------------------------------
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

struct Parts {
    size_t x, a, norms, total;   // bytes
};
Parts parts_of(const D3gsOrthoMatrix& d) {
    const size_t m = d.rows < d.cols ? d.rows : d.cols, n = d.rows < d.cols ? d.cols : d.rows;
    Parts p;
    p.x = up256(m * n * 4);
    p.a = up256(m * m * 4);
    p.norms = up256((size_t)div_up64(d.rows * d.cols, kNormChunk) * 8);
    p.total = 2 * p.x + 2 * p.a + p.norms;
    return p;
}

int32_t check(const D3gsOrthoMatrix* mats, int32_t count, const D3gsOrthoConfig* cfg, bool muon, const char* what) {
    D3GS_REQUIRE(cfg != nullptr, "%s: cfg is NULL", what);
    D3GS_REQUIRE(count >= 0 && (count == 0 || mats != nullptr), "%s: %d matrices", what, count);
    D3GS_REQUIRE(cfg->dtype == D3GS_DTYPE_F32 || (cfg->dtype == D3GS_DTYPE_BF16 && !muon), "%s: dtype %d", what, cfg->dtype);
    D3GS_REQUIRE(cfg->steps >= 1 && cfg->steps <= D3GS_NS_MAX_STEPS, "%s: %d steps (1 to %d)", what, cfg->steps,
                 D3GS_NS_MAX_STEPS);
    D3GS_REQUIRE(cfg->eps > 0.0f, "%s: eps must be positive", what);
    for (int32_t i = 0; i < count; ++i) {
        const D3gsOrthoMatrix& m = mats[i];
        const int64_t small = m.rows < m.cols ? m.rows : m.cols, large = m.rows < m.cols ? m.cols : m.rows;
        D3GS_REQUIRE(small >= 0 && small <= kMaxShort && large <= kMaxLong && small * large < (int64_t)1 << 31,
                     "%s: matrix %d is %lld x %lld (short side at most %d, long side at most %d, below 2^31 values)", what, i,
                     (long long)m.rows, (long long)m.cols, kMaxShort, kMaxLong);
        if (m.rows == 0 || m.cols == 0) continue;
        D3GS_REQUIRE(m.src && m.dst && (!muon || m.momentum), "%s: matrix %d has a NULL pointer", what, i);
        D3GS_REQUIRE(m.rows <= 1 || m.src_row_stride >= 0, "%s: matrix %d has a negative stride", what, i);
    }
    return D3GS_OK;
}

int32_t run(const D3gsOrthoMatrix* mats, int32_t count, const D3gsOrthoConfig& cfg, bool muon, void* ws, size_t ws_bytes,
            cudaStream_t st, const char* what) {
    size_t need = 256;
    for (int32_t i = 0; i < count; ++i) need += parts_of(mats[i]).total;
    D3GS_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= need, "%s: workspace missing, unaligned or too small", what);
    char* at = reinterpret_cast<char*>(up256((size_t)(uintptr_t)ws));
    Table t{};
    t.bf16 = cfg.dtype == D3GS_DTYPE_BF16;
    t.eps = cfg.eps;
    t.mu = cfg.momentum;
    t.nesterov = cfg.nesterov;
    t.decay = cfg.decay;
    int32_t i = 0;
    while (i < count) {
        t.count = 0;
        for (; i < count && t.count < kMaxMatrices; ++i) {
            const D3gsOrthoMatrix& d = mats[i];
            if (d.rows == 0 || d.cols == 0) continue;
            const Parts p = parts_of(d);
            Matrix& m = t.mat[t.count++];
            m.src = d.src;
            m.momentum = muon ? d.momentum : nullptr;
            m.dst = d.dst;
            m.src_stride = d.src_row_stride;
            m.rows = (int32_t)d.rows;
            m.cols = (int32_t)d.cols;
            m.m = m.rows < m.cols ? m.rows : m.cols;
            m.n = m.rows < m.cols ? m.cols : m.rows;
            m.rate = d.rate;
            m.x[0] = reinterpret_cast<float*>(at);
            m.x[1] = reinterpret_cast<float*>(at + p.x);
            m.a = reinterpret_cast<float*>(at + 2 * p.x);
            m.b = reinterpret_cast<float*>(at + 2 * p.x + p.a);
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
        auto tiles = [](int64_t v) { return div_up64(v, kTile); };
        auto chunks = [](const Matrix& m) { return div_up64((int64_t)m.rows * m.cols, kNormChunk); };
        t.from = 0;
        unsigned grid = blocks(chunks);
        ns_norm_kernel<<<grid, kThreads, 0, st>>>(t);
        D3GS_LAUNCH_CHECK("ns_norm_kernel");
        ns_load_kernel<<<grid, kThreads, 0, st>>>(t);
        D3GS_LAUNCH_CHECK("ns_load_kernel");
        for (int s = 0; s < cfg.steps; ++s) {
            t.ca = cfg.coefficients[s][0];
            t.cb = cfg.coefficients[s][1];
            t.cc = cfg.coefficients[s][2];
            grid = blocks([&](const Matrix& m) { return tiles(m.m) * tiles(m.m); });
            ns_gemm_kernel<kGram><<<grid, kThreads, 0, st>>>(t);
            D3GS_LAUNCH_CHECK("ns_gemm_kernel");
            ns_gemm_kernel<kSquare><<<grid, kThreads, 0, st>>>(t);
            D3GS_LAUNCH_CHECK("ns_gemm_kernel");
            grid = blocks([&](const Matrix& m) { return tiles(m.m) * tiles(m.n); });
            ns_gemm_kernel<kApply><<<grid, kThreads, 0, st>>>(t);
            D3GS_LAUNCH_CHECK("ns_gemm_kernel");
            t.from ^= 1;
        }
        grid = blocks(chunks);
        ns_store_kernel<<<grid, kThreads, 0, st>>>(t);
        D3GS_LAUNCH_CHECK("ns_store_kernel");
    }
    return D3GS_OK;
}

}  // namespace
}  // namespace d3gs

using namespace d3gs;

extern "C" size_t d3gs_orthogonalize_workspace_bytes(const D3gsOrthoMatrix* matrices, int32_t count,
                                                     const D3gsOrthoConfig* cfg) {
    if (check(matrices, count, cfg, false, "d3gs_orthogonalize_workspace_bytes") != D3GS_OK) return 0;
    size_t need = 256;
    for (int32_t i = 0; i < count; ++i) need += parts_of(matrices[i]).total;
    return need;
}

extern "C" int32_t d3gs_orthogonalize(const D3gsOrthoMatrix* matrices, int32_t count, const D3gsOrthoConfig* cfg,
                                      void* workspace, size_t workspace_bytes, void* stream) {
    if (int32_t rc = check(matrices, count, cfg, false, "d3gs_orthogonalize")) return rc;
    return run(matrices, count, *cfg, false, workspace, workspace_bytes, static_cast<cudaStream_t>(stream), "d3gs_orthogonalize");
}

extern "C" int32_t d3gs_muon_step(const D3gsOrthoMatrix* matrices, int32_t count, const D3gsOrthoConfig* cfg,
                                  void* workspace, size_t workspace_bytes, void* stream) {
    if (int32_t rc = check(matrices, count, cfg, true, "d3gs_muon_step")) return rc;
    return run(matrices, count, *cfg, true, workspace, workspace_bytes, static_cast<cudaStream_t>(stream), "d3gs_muon_step");
}
